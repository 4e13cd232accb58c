"""The operators between a language model's products as a program uses them: a layer's pass over prompts and single tokens, captured steps, two streams,
memory of any contents, the compiled and the Python form of each call, caches of more than 2^32 elements."""
import ctypes as C

import numpy as np
import pytest

import generation_reference as R
from conftest import rel_fro


class Declines:
    def __getattr__(self, name):
        return lambda *args: None


def test_cpu_tensors_are_refused(pkg):
    torch = pytest.importorskip("torch")
    x, positions, f = torch.zeros(2, 2, 64), torch.zeros(2, dtype=torch.int32), torch.zeros(32, dtype=torch.float64)
    cache = pkg.paged_cache(2, 2, 16, 64, device="cpu")
    table, starts, lengths = torch.zeros(1, 1, dtype=torch.int32), torch.tensor([0, 2], dtype=torch.int32), torch.tensor([2], dtype=torch.int32)
    logits, random = torch.zeros(2, 5), torch.zeros(2)
    native = pkg._native()
    assert native.rotary(x, x, positions, f, False, 1.0) is None and native.cache_write(cache, x, x, positions) is None
    assert native.cache_read(cache, table, starts, 2) is None and native.paged_attention(x, cache, table, starts, lengths, 1.0, True, 0, 0) is None
    for call in (lambda: pkg.rotary(x, x, positions, f), lambda: pkg.cache_write(cache, x, x, positions), lambda: pkg.cache_read(cache, table, starts, 2),
                 lambda: pkg.paged_attention(x, cache, table, starts, lengths, 1.0), lambda: pkg.sample(logits, random)):
        with pytest.raises(pkg.InvalidArgumentError):
            call()


class Layer:
    """One layer of a model with a vocabulary, its cache, and what it has written there."""

    def __init__(self, pkg, kind, hidden=64, heads=6, kv=2, size=32, vocabulary=999, page=16, pages=40, batch=3, seed=0):
        import torch
        g = torch.Generator("cuda").manual_seed(seed)
        f = lambda *s: torch.randn(s, device="cuda", generator=g) * s[0] ** -0.5
        self.pkg, self.heads, self.kv, self.size, self.page = pkg, heads, kv, size, page
        self.w_q, self.w_k, self.w_v = f(hidden, heads * size), f(hidden, kv * size), f(hidden, kv * size)
        self.w_o, self.w_vocabulary = f(heads * size, hidden), f(hidden, vocabulary) * 3
        self.embedding = torch.randn(vocabulary, hidden, device="cuda", generator=g)
        frequencies, _ = pkg.rotary_frequencies(size)
        self.frequencies = torch.tensor(frequencies, dtype=torch.float64, device="cuda")
        self.cache = pkg.paged_cache(pages, kv, page, size, torch.int8 if kind == "s8" else torch.float32)
        self.table = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))[:batch * (pages // batch)].reshape(batch, -1).to("cuda", torch.int32)

    def __call__(self, tokens, positions, slots, starts, lengths, random, last, keep=None, max_length=0):
        """tokens .. slots of all rows, some of them padding behind the last sequence; last: the rows that tokens are chosen for."""
        pkg, x = self.pkg, self.embedding[tokens]
        q = pkg.blas_matmul(x, self.w_q).view(-1, self.heads, self.size)
        k = pkg.blas_matmul(x, self.w_k).view(-1, self.kv, self.size)
        v = pkg.blas_matmul(x, self.w_v).view(-1, self.kv, self.size)
        q, k = pkg.rotary(q, k, positions, self.frequencies)
        pkg.cache_write(self.cache, k, v, slots)
        y = pkg.paged_attention(q, self.cache, self.table, starts, lengths, self.size ** -0.5, max_length=max_length)
        logits = pkg.blas_matmul(pkg.blas_matmul(y.view(len(y), -1), self.w_o)[last], self.w_vocabulary)
        if keep is not None:
            keep.update(q=q, k=k, v=v, y=y, logits=logits)
        return pkg.sample(logits, random, top_p=torch_full(len(logits), 0.9), top_k=torch_full(len(logits), 50, np.int32))

    def slots_of(self, i, positions):
        import torch
        positions = torch.as_tensor(positions, device="cuda")
        return self.table[i, positions // self.page].long() * self.page + positions % self.page


def torch_full(n, value, dtype=np.float32):
    import torch
    return torch.from_numpy(np.full(n, value, dtype)).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "s8"])
def test_prompts_then_single_tokens(pkg, T, kind):
    import torch
    rng = np.random.default_rng(5)
    m = Layer(pkg, kind)
    prompts = [rng.integers(0, 999, n) for n in (37, 1, 90)]
    held = [list(p) for p in prompts]
    for step in range(6):
        if step < 2:  # the prompts, the last one's second half in a step of its own
            chunks = [prompts[0], prompts[1], prompts[2][:50]] if step == 0 else [held[0][-1:], held[1][-1:], prompts[2][50:]]
        else:
            chunks = [h[-1:] for h in held]
        counts = [len(c) for c in chunks]
        known = [37, 1, 50] if step == 0 else [len(held[0]), len(held[1]), 90 if step == 1 else len(held[2])]
        pad = 3
        tokens = np.concatenate([*chunks, np.zeros(pad, np.int64)])
        positions = np.concatenate([*(np.arange(n - c, n) for n, c in zip(known, counts)), np.zeros(pad, np.int64)])
        slots = torch.cat([m.slots_of(i, np.arange(n - c, n)) for i, (n, c) in enumerate(zip(known, counts))] + [torch.full((pad,), -1, device="cuda")])
        starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        random, keep = rng.random(3).astype(np.float32), {}
        last = T.t(starts[1:].astype(np.int64) - 1)
        before = [T.n(t).copy() for t in m.cache]
        chosen, odds = m(T.t(tokens), T.t(positions), slots, T.t(starts), T.t(np.array(known, np.int32)), T.t(random), last, keep)
        got = {n: T.n(t) for n, t in keep.items()}
        # what the cache holds now is what it held and the new rows
        cache = [T.n(t) for t in m.cache]
        for i, new in enumerate((got["k"], got["v"])):
            n, scale = R.quantized(new)
            for t, slot in enumerate(T.n(slots)):
                if slot >= 0:
                    before[i][slot // m.page, :, slot % m.page] = n[t] if kind == "s8" else new[t]
                    if kind == "s8":
                        before[2 + i][slot // m.page, :, slot % m.page] = scale[t]
        for a, b in zip(cache, before):
            assert np.array_equal(a, b)
        rows = int(starts[-1])
        want, off = R.attention(got["q"][:rows], cache, T.n(m.table), starts, np.array(known, np.int32), m.size ** -0.5)
        assert (np.abs(got["y"][:rows] - want) <= off).all()
        token, exact, margin = R.sample(got["logits"], random, top_p=np.full(3, 0.9, np.float32), top_k=np.full(3, 50, np.int32))
        assert np.array_equal(T.n(chosen)[margin > 1e-9], token[margin > 1e-9])
        # and the whole pass from the tokens, without pages, in 64 bits: a product over 64 or 192 is off by about K^1.5 2^-24 of its norm, 3e-5 or
        # 1.6e-4, scores of up to about 8 by 8 x 2 x 3e-5, weights by as much; int8 adds half a step of amax / 127 to each of
        # 32 keys and values, about 2.6 / 254 = 1.1% of their norm, and to the scores up to 4% of a weight
        if step != 0:
            for i in range(3):
                known_tokens = np.array(held[i][:known[i]])
                e = T.n(m.embedding).astype(np.float64)[known_tokens]
                q, k, v = (e @ T.n(w).astype(np.float64) for w in (m.w_q, m.w_k, m.w_v))
                f = T.n(m.frequencies)
                q = R.rotary(q.reshape(len(e), m.heads, m.size), np.arange(len(e)), f, False, 1.0)[0]
                k = R.rotary(k.reshape(len(e), m.kv, m.size), np.arange(len(e)), f, False, 1.0)[0]
                v = v.reshape(len(e), m.kv, m.size)
                y = np.zeros((m.heads, m.size))
                for h in range(m.heads):
                    s = k[:, h // 3] @ q[-1, h] * m.size ** -0.5
                    w = np.exp(s - s.max())
                    y[h] = w / w.sum() @ v[:, h // 3]
                logits = y.reshape(-1) @ T.n(m.w_o).astype(np.float64) @ T.n(m.w_vocabulary).astype(np.float64)
                assert rel_fro(got["logits"][i], logits) < (1e-3 if kind == "f32" else 0.08)
        for i, token in enumerate(T.n(chosen)):
            if not (i == 2 and step == 0):  # the middle of a prompt
                held[i].append(int(token))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "s8"])
def test_captured_steps(pkg, T, kind):
    """Two captured steps of different batches (pieces of the keys, workspaces of their own), replayed in turn and at the same time between eager calls."""
    import torch
    rng = np.random.default_rng(6)
    streams = [torch.cuda.Stream() for _ in range(2)]
    models, inputs, graphs, outputs, eager = [], [], [], [], []
    for i in range(2):
        m = Layer(pkg, kind, pages=150, batch=3, seed=i)
        for t in m.cache:
            if t.dtype == torch.int8:
                t.copy_(T.t(rng.integers(-127, 128, t.shape, dtype=np.int8)))
            else:
                t.copy_(T.t((rng.random(t.shape) * 0.03).astype(np.float32)))
        lengths = np.array([300, 790, 51], np.int32)
        state = dict(tokens=T.t(np.zeros(3, np.int64)), positions=T.t(lengths - 1), slots=torch.zeros(3, dtype=torch.int64, device="cuda"),
                     starts=T.t(np.arange(4, dtype=np.int32)), lengths=T.t(lengths), random=T.t(np.zeros(3, np.float32)), last=T.t(np.arange(3)))
        k50, p90 = torch_full(3, 50, np.int32), torch_full(3, 0.9)

        def step(m=m, state=state, k50=k50, p90=p90):
            q = pkg.blas_matmul(m.embedding[state["tokens"]], m.w_q).view(-1, m.heads, m.size)
            k = pkg.blas_matmul(m.embedding[state["tokens"]], m.w_k).view(-1, m.kv, m.size)
            q, k = pkg.rotary(q, k, state["positions"], m.frequencies)
            pkg.cache_write(m.cache, k, k, state["slots"])
            y = pkg.paged_attention(q, m.cache, m.table, state["starts"], state["lengths"], m.size ** -0.5, max_length=1500)
            logits = pkg.blas_matmul(pkg.blas_matmul(y.view(3, -1), m.w_o), m.w_vocabulary)
            return (y, logits, *pkg.sample(logits, state["random"], top_p=p90, top_k=k50))
        with torch.cuda.stream(streams[i]):
            streams[i].wait_stream(torch.cuda.default_stream())
            step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=streams[i]):
            out = step()
        models.append(m), inputs.append(state), graphs.append(graph), outputs.append(out), eager.append(step)
    for turn in range(4):
        for i, (m, state) in enumerate(zip(models, inputs)):
            lengths = np.array([300 + 70 * turn, 790 - turn, 51 + turn], np.int32)
            state["lengths"].copy_(T.t(lengths))
            state["positions"].copy_(T.t(lengths - 1))
            state["tokens"].copy_(T.t(rng.integers(0, 999, 3)))
            state["random"].copy_(T.t(rng.random(3).astype(np.float32)))
            state["slots"].copy_(torch.cat([m.slots_of(j, [n - 1]) for j, n in enumerate(lengths.tolist())]))
        want = [[o.clone() for o in step()] for step in eager]
        for out in outputs:
            for o in out:
                o.fill_(-7)
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for w, out in zip(want, outputs):
            for a, b in zip(w, out):
                assert torch.equal(a, b)


@pytest.mark.gpu
def test_streams_at_the_same_time(pkg, T):
    """The same calls on two streams, each with inputs of its own, one after another: as on one."""
    import torch
    rng = np.random.default_rng(7)
    jobs = []
    for i in range(2):
        cache = pkg.paged_cache(300, 4, 16, 128)
        for t in cache:
            t.copy_(T.t(rng.integers(-127, 128, t.shape, dtype=np.int8)) if t.dtype == torch.int8 else T.t((rng.random(t.shape) * 0.02 + 0.01).astype(np.float32)))
        table = T.t(rng.permutation(300).astype(np.int32).reshape(2, 150))
        lengths, starts = T.t(np.array([2300, 1700], np.int32)), T.t(np.array([0, 1, 9], np.int32))
        q, logits, random = T.t(rng.normal(size=(9, 8, 128)).astype(np.float32)), T.t(rng.normal(size=(9, 50001)).astype(np.float32)), T.t(rng.random(9).astype(np.float32))

        def job(cache=cache, table=table, lengths=lengths, starts=starts, q=q, logits=logits, random=random):
            y = pkg.paged_attention(q, cache, table, starts, lengths, 0.09)
            token, odds = pkg.sample(logits, random)
            return y, token, odds, *pkg.cache_read(cache, table, starts, 9)
        jobs.append(job)
    want = [[t.clone() for t in job()] for job in jobs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for turn in range(5):
        for job, stream in zip(jobs, streams):
            with torch.cuda.stream(stream):
                got.append(job())
    torch.cuda.synchronize()
    for i, outs in enumerate(got):
        for a, b in zip(outs, want[i % 2]):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_same_bits_as_the_python_form(pkg, T, monkeypatch):
    import torch
    rng = np.random.default_rng(8)
    q, k = T.t(rng.normal(size=(21, 8, 64)).astype(np.float32)), T.t(rng.normal(size=(21, 2, 64)).astype(np.float32))
    f = T.t(np.array(pkg.rotary_frequencies(48)[0]))
    positions, logits, random = T.t(rng.integers(0, 5000, 21)), T.t(rng.normal(size=(21, 5001)).astype(np.float32)), T.t(rng.random(21).astype(np.float32))
    slots, table = T.t(np.arange(21, dtype=np.int32)), T.t(np.array([[0, 1, 5], [1, 0, 3]], np.int32))
    starts, lengths = T.t(np.array([0, 20, 21], np.int32)), T.t(np.array([30, 17], np.int32))
    temperature, top_k = torch_full(21, 0.7), torch_full(21, 40, np.int32)
    used = []

    class Counts:
        def __init__(self, real):
            self.real = real

        def __getattr__(self, name):
            def call(*args):
                out = getattr(self.real, name)(*args)
                used.append((name, out is not None))
                return out
            return call

    def everything():
        out = list(pkg.rotary(q, k, positions, f)) + [pkg.rotary(q, None, positions, f, True, 1.5)[0]]
        for kind in (torch.int8, torch.float32):
            cache = pkg.paged_cache(4, 2, 16, 64, kind)
            pkg.cache_write(cache, k, k * 2, slots)
            out += [*cache, *pkg.cache_read(cache, table, starts, 21)]
            out.append(pkg.paged_attention(q, cache, table, starts, lengths, 0.125))
            out.append(pkg.paged_attention(q, cache, table, starts, lengths, 0.125, True, 7, 25))
            out.append(pkg.paged_attention(q, cache, table, starts, lengths, 0.125, False))
        return out + list(pkg.sample(logits, random)) + list(pkg.sample(logits, random, temperature, top_k))

    monkeypatch.setattr(pkg, "_calls", Counts(pkg._native()))
    compiled = everything()
    assert {n for n, done in used if done} >= {"rotary", "cache_write", "cache_read", "paged_attention", "sample"} and all(done for _, done in used)
    monkeypatch.setattr(pkg, "_calls", Declines())
    python = everything()
    assert len(compiled) == len(python)
    for a, b in zip(compiled, python):
        assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b)


@pytest.mark.gpu
def test_workspaces_of_any_contents(pkg, T):
    """Attention in pieces, some of them without keys, and sampling: NaN, infinities and every other bit in the workspace change nothing."""
    import torch
    rng = np.random.default_rng(9)
    lib = pkg.lib()
    cache = pkg.paged_cache(200, 2, 16, 64, torch.float32)
    for t in cache:
        t.copy_(T.t(rng.normal(size=t.shape).astype(np.float32)))
    d = pkg.PagedAttentionDesc()
    d.cache = pkg._cache_desc(cache)
    q, out = T.t(rng.normal(size=(3, 4, 64)).astype(np.float32)), torch.empty(3, 4, 64, device="cuda")
    starts, lengths, table = T.t(np.array([0, 1, 2, 3], np.int32)), T.t(np.array([3200, 40, 0], np.int32)), T.t(np.arange(600, dtype=np.int32).reshape(3, 200) % 200)
    d.q, d.out, d.starts, d.lengths, d.table = (t.data_ptr() for t in (q, out, starts, lengths, table))
    d.q_token_stride = d.out_token_stride = 256
    d.q_head_stride = d.out_head_stride = 64
    d.tokens, d.heads, d.batch, d.table_stride, d.table_width, d.scale, d.causal = 3, 4, 3, 200, 200, 0.125, 1
    needs = lib.tfcc_rocm_paged_attention_workspace(C.byref(d))
    logits, random = T.t(rng.normal(size=(2, 70001)).astype(np.float32)), T.t(rng.random(2).astype(np.float32))
    token, odds = torch.empty(2, dtype=torch.int64, device="cuda"), torch.empty(2, device="cuda")
    s = pkg.SampleDesc()
    s.logits, s.random, s.tokens, s.probabilities = (t.data_ptr() for t in (logits, random, token, odds))
    s.rows, s.length, s.row_stride = 2, 70001, 70001
    needs_too = lib.tfcc_rocm_sample_workspace(2, 70001)
    assert needs > 0 and needs_too > 0
    want = None
    for fill in (0, 0x7fc00000, 0xff800000, 0xffffffff, 0x3f800000, 0x01010101):
        memory = torch.empty(max(needs, needs_too) // 4 + 4, dtype=torch.int32, device="cuda").fill_(fill - (1 << 32) if fill >> 31 else fill)
        d.workspace, d.workspace_bytes = memory.data_ptr(), needs
        pkg.check(lib.tfcc_rocm_paged_attention_f32(torch.cuda.current_stream().cuda_stream, C.byref(d)))
        assert (memory[needs // 4:] == memory[-1]).all()
        memory.fill_(fill - (1 << 32) if fill >> 31 else fill)
        s.workspace, s.workspace_bytes = memory.data_ptr(), needs_too
        pkg.check(lib.tfcc_rocm_sample_f32(torch.cuda.current_stream().cuda_stream, C.byref(s)))
        assert (memory[(needs_too + 3) // 4:] == memory[-1]).all()
        got = [T.n(t).copy() for t in (out, token, odds)]
        want = want or got
        for a, b in zip(got, want):
            assert np.array_equal(a, b)
    assert (want[0][2] == 0).all() and np.isfinite(want[0]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["s8", "f32"])
@pytest.mark.parametrize("heads,chunks", [(4, [1, 40]), (128, [150, 140])])
def test_pages_more_than_32_bits_apart(pkg, T, kind, heads, chunks):
    """A cache of three pages 2^31 + 16 elements apart and more: written, attended over and read back as a small one is."""
    import torch
    rng = np.random.default_rng(10)
    kv, page, size = heads // 2, 160, 64
    dtype, apart = (torch.int8, (1 << 32) + (1 << 24)) if kind == "s8" else (torch.float32, (1 << 31) + (1 << 24))
    memory = torch.empty(2 * apart + 2 * kv * page * size, dtype=dtype, device="cuda")
    far = tuple(torch.as_strided(memory, (3, kv, page, size), (apart, page * size, size, 1), i * kv * page * size) for i in range(2))
    near = pkg.paged_cache(3, kv, page, size, dtype)
    if kind == "s8":
        far += tuple(torch.zeros_like(t) for t in near[2:])
    lengths, starts = np.array([300, 150], np.int32), np.concatenate([[0], np.cumsum(chunks)]).astype(np.int32)
    table = np.array([[2, 1], [0, 0]], np.int32)
    slots = np.concatenate([np.where(np.arange(300) < 160, 2 * page + np.arange(300), page + np.arange(300) - 160), np.arange(150)])
    k, v = (T.t(rng.normal(size=(450, kv, size)).astype(np.float32)) for _ in range(2))
    q = T.t(rng.normal(size=(int(starts[-1]), heads, size)).astype(np.float32))
    outs = []
    for cache in (near, far):
        for t in cache:
            for i in range(3):
                t[i].zero_()
        pkg.cache_write(cache, k, v, T.t(slots))
        y = pkg.paged_attention(q, cache, T.t(table), T.t(starts), T.t(lengths), 0.125)
        outs.append([y, *pkg.cache_read(cache, T.t(table), T.t(np.array([0, 300, 450], np.int32)), 450)])
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    del memory, far
    torch.cuda.empty_cache()
