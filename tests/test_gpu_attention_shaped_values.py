"""Attention with shaped scores at the ends of what its arguments and a float32 cache may hold: caps below float32's smallest number, slopes next to its largest, infinities, NaN
and numbers of 2^80 and more that chunks of many tokens see under a cap, slopes or a prefix."""
import os
import subprocess

import numpy as np
import pytest

import serving_reference as R
from generation_reference import EPS
from test_gpu_attention_shaped import Made

HOST = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "wechat-tfcc_amd", "host")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["s4", "s8", "f32"])
@pytest.mark.parametrize("cap", [1e-45, 1e-46, 1e-60, 5e-324])
def test_caps_below_the_smallest_number(pkg, T, kind, cap):
    """All scores are next to 0, and weights the same: such a cap is not none."""
    import torch
    m = Made(pkg, kind, [300, 45], [2, 45], 4, 2, 64, 16, 3)
    m.check(T, **m.shaped({}, cap=cap))
    m.check(T, **m.shaped({}, cap=cap, slopes=True))
    out = torch.empty(m.q.shape, device="cuda")  # the call's other form
    m.run(T, out=out, cap=cap)
    assert np.array_equal(T.n(out), T.n(m.run(T, cap=cap)))


@pytest.mark.gpu
def test_caps_below_zero_are_refused_however_small(pkg, T):
    import torch
    m = Made(pkg, "f32", [60], [2], 4, 2, 64, 16, 6)
    for cap in (-1e-60, -1e-45, -5e-324):
        for out in (None, torch.empty(m.q.shape, device="cuda")):
            with pytest.raises(pkg.InvalidArgumentError):
                m.run(T, out=out, cap=cap)
    assert np.array_equal(T.n(m.run(T, cap=-0.0)), T.n(m.run(T)))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["s4", "s8", "f32"])
@pytest.mark.parametrize("cap", [0.0, 5.0])
def test_slopes_next_to_the_largest_number(pkg, T, kind, cap):
    """A slope of 2.4e38 and more is finite, though it is not in the units of log2: the key at distance 0 has a bias of 0 and is all there is."""
    m = Made(pkg, kind, [300, 270, 40], [258, 3, 40], 4, 2, 64, 16, 3)
    kw = m.shaped({}, cap=cap)
    kw["slopes"] = np.array([3.4028234e38, 2.4e38, 2.3e38, 1e37], np.float32)
    m.check(T, **kw)


# float32, tiles of 128 and 256 rows, with pages, windows and pieces that end inside a step of 16 keys: lengths, chunks, heads, kv heads, size, page, more, rows of a tile, pieces
FAR = [
    ([300, 270], [258, 260], 64, 32, 64, 16, {}, 128, 1),
    ([310, 270], [258, 260], 64, 32, 40, 20, {"window": 70}, 128, 1),
    ([300, 290], [300, 290], 32, 16, 128, 20, {}, 256, 1),
    ([500, 333], [300, 290], 48, 16, 96, 24, {"causal": False}, 256, 2),
    ([3000, 300], [200, 111], 32, 8, 128, 20, {}, 256, 5),
    ([2700, 2100], [300, 260], 32, 32, 64, 28, {"window": 2300}, 128, 3),
    ([1100, 1030], [400, 410], 12, 12, 64, 32, {}, 128, 4),
    ([400, 200, 90], [260, 280, 90], 48, 48, 96, 16, {}, 256, 1),   # more tokens than are cached
]
SHAPES = [{"cap": 4.0, "slopes": True}, {"cap": 20.0, "prefix": True}, {"slopes": True}, {"slopes": True, "prefix": True}]


def shape_of(m, shape, prefixes):
    return m.shaped({}, shape.get("cap", 0.0), shape.get("slopes", False), prefixes if "prefix" in shape else None)


@pytest.mark.parametrize("case", range(len(FAR)))
def test_planned(case):
    """The tiles and pieces that the cases are about."""
    lengths, chunks, heads, kv, size, page, more, rows, pieces = FAR[case]
    driver = os.path.join(HOST, "build", "paged_attention_plan_print")
    subprocess.check_call(["make", "-s", "-C", HOST, "build/paged_attention_plan_print"])
    most = (max(-(-n // page) for n in lengths) + 1) * page
    line = (sum(chunks), len(lengths), heads // kv, kv, size, most, int(more.get("causal", True)), more.get("window", 0), 128 if size <= 64 else 256, 1)
    got = subprocess.run([driver], input=" ".join(map(str, line)), stdout=subprocess.PIPE, text=True, timeout=60).stdout.split()
    assert (int(got[0]), int(got[2])) == (rows, pieces)


def definition(m, causal=True, window=0, cap=0.0, slopes=None, prefixes=None):
    """(out, how far float32 may be off, rows x keys that are seen) as serving_reference.attention, but with the error of a capped score by the score itself: one far above its
    cap is the cap, however large the sums it comes from.  Of keys that are not finite the error is 0: their scores are infinities or NaN."""
    k, v = R.held(m.cache)
    pages, kv, page_size, size = k.shape
    group = m.q.shape[1] // kv
    out, off = np.full(m.q.shape, np.nan), np.zeros(m.q.shape)
    for i, length in enumerate(m.lengths):
        n = m.starts[i + 1] - m.starts[i]
        at = np.arange(min(int(length), m.table.shape[1] * page_size))
        page = m.table[i][at // page_size]
        there = (page >= 0) & (page < pages)
        page = np.where(there, page, 0)
        position = (int(length) - n + np.arange(n))[:, None]
        seen = np.ones((n, len(at)), bool)
        if causal:
            seen &= at <= position
            if window:
                seen &= at > position - window
            if prefixes is not None:
                seen |= at < prefixes[i]
        seen = np.repeat(seen & there, group, 0)
        far = np.repeat(np.abs(position - at).astype(np.float64), group, 0)
        for h in range(kv):
            x = m.q[m.starts[i]:m.starts[i + 1], h * group:(h + 1) * group].astype(np.float64).reshape(-1, size)
            kk, vv = k[page, h, at % page_size], v[page, h, at % page_size]
            with np.errstate(all="ignore"):
                raw = x @ kk.T * m.scale
                e = (size + 12) * EPS * (np.abs(x) @ np.abs(kk).T) * abs(m.scale)
                bias = 0.0 if slopes is None else np.tile(slopes[h * group:(h + 1) * group].astype(np.float64), n)[:, None] * far
                s = (np.tanh(raw / cap) * cap if cap else raw) - bias
                if cap:
                    e = cap * np.where(np.abs(raw) > e, np.tanh((np.abs(raw) + e) / cap) - np.tanh((np.abs(raw) - e) / cap), np.minimum(2 * e / cap, 2)) + 12 * EPS * np.minimum(np.abs(raw), cap)
                e = np.where(np.isfinite(raw), e, 0) + 4 * EPS * np.abs(np.where(np.isfinite(s), s, 0)) + 4 * EPS * np.abs(bias)
                s = np.where(seen, s, -np.inf)
                top = s.max(-1, keepdims=True)
                w = np.where(seen, np.exp(s - np.where(top == -np.inf, 0, top)), 0)
                p = np.where(seen.any(-1, keepdims=True), w / w.sum(-1, keepdims=True), 0)
                fine = np.where(np.isfinite(vv), vv, 0)
                y, size_of = p @ fine, p @ np.abs(fine)
                for j in np.flatnonzero(~np.isfinite(vv).all(-1)):  # 0 x infinity of a key that a row does not see is nothing
                    y[seen[:, j]] += np.where(np.isfinite(vv[j]), 0, p[seen[:, j], j, None] * vv[j])
                ds = np.where(seen, e, 0).max(-1, keepdims=True)
                # weights below 2^-126 of the largest may be lost
                bound = (2 * ds + 48 * EPS + seen.sum(-1, keepdims=True) * EPS) * size_of + 2.0 ** -126 * (seen @ np.abs(fine)) + 1e-37
            rows = slice(m.starts[i], m.starts[i + 1]), slice(h * group, (h + 1) * group)
            out[rows], off[rows] = y.reshape(n, group, size), bound.reshape(n, group, size)
    return out, off


@pytest.mark.gpu
@pytest.mark.parametrize("value", [np.inf, np.nan, 2.0 ** 90, -3e38])
@pytest.mark.parametrize("case,shape", [(c, s) for c in range(len(FAR)) for s in range(len(SHAPES)) if "prefix" not in SHAPES[s] or not FAR[c][6]])
def test_far_numbers_under_shaped_scores(pkg, T, case, shape, value):
    """Value rows and keys with an infinity, a NaN or a number beyond 2^80, inside the prefix, behind it and on the chunk's own last tokens: rows that see one are those of the
    definition, all others keep every bit."""
    lengths, chunks, heads, kv, size, page, more, _, _ = FAR[case]
    m = Made(pkg, "f32", lengths, chunks, heads, kv, size, page, 71 + case)
    m.table[0, 2] = -1
    prefixes = [n - c // 2 for n, c in zip(lengths, chunks)]  # up to the middle of the chunk: its first tokens see what its later ones are
    kw = dict(more, **shape_of(m, SHAPES[shape], prefixes))
    on = {k: T.t(a) if isinstance(a, np.ndarray) else a for k, a in kw.items()}
    capped = "cap" in SHAPES[shape]
    group = heads // kv
    # (key, cache head, sequence, of keys): within the prefix, the chunk's first and last tokens
    places = [(lengths[0] // 2, 1, 0, False), (lengths[0] - 2, 0, 0, capped), (max(lengths[1] - chunks[1] // 2 - 5, 3), 1, 1, capped), (lengths[1] - 1, kv - 1, 1, False),
              (lengths[1] // 3, kv - 1, 1, False)]
    clean = T.n(m.run(T, **on)).copy()
    mine = np.zeros(clean.shape, bool)
    for at, head, sequence, key in places:
        named, inside = m.table[sequence, at // page], at % page
        if not 0 <= named < len(m.cache[0]):
            continue
        m.cache[0 if key else 1][named, head, inside, 5] = value
        n = chunks[sequence]
        position = lengths[sequence] - n + np.arange(n)
        sees = (at <= position) & (at > position - more.get("window", 10 ** 9)) if more.get("causal", True) else np.ones(n, bool)
        if "prefix" in SHAPES[shape]:
            sees |= at < prefixes[sequence]
        mine[m.starts[sequence]:m.starts[sequence + 1], head * group:(head + 1) * group] |= sees[:, None, None]
    got = T.n(m.run(T, **on)).astype(np.float64)
    assert mine.any() and not mine.all()
    assert np.array_equal(got[~mine], clean[~mine])
    kw.pop("max_length", None)
    want, off = definition(m, **kw)
    same = (got == want) | (np.isnan(got) & np.isnan(want))
    with np.errstate(invalid="ignore"):
        near = np.abs(got - want) <= off
    lost = np.isinf(want) & np.isnan(got)  # a weight below 2^-149 times infinity is NaN in float32 and infinity in 64 bits
    assert (same | near | lost).all(), np.argwhere(~(same | near | lost))[:5].tolist()
    assert not lost[mine].all()


@pytest.mark.gpu
@pytest.mark.parametrize("case", [0, 2, 4, 6])
def test_far_numbers_between_replays_of_shaped_scores(pkg, T, case):
    """A captured call meets infinities that come and go in its cache, and a prefix that moves which rows see them."""
    import torch
    lengths, chunks, heads, kv, size, page = FAR[case][:6]
    m = Made(pkg, "f32", lengths, chunks, heads, kv, size, page, 91)
    kw = m.shaped({}, cap=10.0, slopes=True, prefixes=[0] * len(lengths))
    cache, q, table, starts, held = m.on(T), T.t(m.q), T.t(m.table), T.t(m.starts), T.t(m.lengths)
    slopes, prefixes = T.t(kw["slopes"]), T.t(kw["prefixes"])
    call = lambda: pkg.paged_attention(q, cache, table, starts, held, m.scale, cap=10.0, slopes=slopes, prefixes=prefixes)
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    at = lengths[0] - 3
    named, inside = m.table[0, at // page], at % page
    before = cache[1][named, 0, inside, 3].item()
    group = heads // kv
    for prefix in (0, at, at + 1):
        prefixes.fill_(prefix)
        for value in (before, float("inf"), 2.0 ** 90, float("nan"), before):
            cache[1][named, 0, inside, 3] = value
            eager = call()
            for _ in range(2):
                out.zero_()
                graph.replay()
                torch.cuda.synchronize()
                assert torch.equal(out.isnan(), eager.isnan()) and torch.equal(out.nan_to_num(0.0), eager.nan_to_num(0.0))
            if value != value:
                rows = eager[:chunks[0], :group, 3].isnan().all(-1)
                assert int(rows.sum()) == (chunks[0] if prefix > at else 3)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["s4", "s8"])
@pytest.mark.parametrize("lengths,chunks,heads,kv,page", [([60], [2], 4, 2, 16), ([90], [1], 4, 2, 32), ([70], [1], 4, 2, 24), ([30], [2], 4, 2, 8), ([260, 270], [260, 270], 128, 64, 256)])
def test_pages_more_than_32_bits_of_bytes_apart(pkg, T, kind, lengths, chunks, heads, kv, page):
    """Every page but the first starts behind 2^32 bytes: rings for pages of each kind, keys one by one, wide tiles."""
    import torch
    m = Made(pkg, kind, lengths, chunks, heads, kv, 128, page, 6, spare=0)
    shaped = m.shaped({}, cap=5.0, slopes=True, prefixes=[7] * len(lengths))
    on = {k: T.t(v) if isinstance(v, np.ndarray) else v for k, v in shaped.items()}
    want = [T.n(m.run(T)), T.n(m.run(T, **on))]
    far = (1 << 32) + 4096
    assert m.table[0, 0] > 0 or m.table[0, 1] > 0
    cache = []
    for t in m.on(T):
        if t.dim() == 4:
            memory = torch.empty((far * (t.shape[0] - 1) + t[0].numel(),), dtype=t.dtype, device="cuda")
            v = torch.as_strided(memory, t.shape, (far, *t.stride()[1:]))
            v.copy_(t)
            t = v
        cache.append(t)
    assert np.array_equal(T.n(m.run(T, tuple(cache))), want[0]) and np.array_equal(T.n(m.run(T, tuple(cache), **on)), want[1])
