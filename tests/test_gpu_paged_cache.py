"""Writing a paged cache and reading it back: integers and scales bit for bit those of the definition (the quotient in 64 bits), and
nothing else touched."""
import ctypes as C

import numpy as np
import pytest

import generation_reference as R


def test_refused_without_a_device(pkg):
    lib, c = pkg.lib(), pkg.PagedCache()
    write = lambda **k: lib.tfcc_rocm_cache_write(None, C.byref(c), k.get("keys", 64), 0, 0, 64, 0, 0, k.get("tokens", 1), 64, k.get("type", pkg.S32))
    read = lambda: lib.tfcc_rocm_cache_read(None, C.byref(c), 64, 0, 1, 1, 64, 1, 64, 64)
    assert lib.tfcc_rocm_cache_write(None, None, 64, 0, 0, 64, 0, 0, 1, 64, pkg.S32) == 1
    c.keys = c.values = c.key_scales = c.value_scales = 4096
    c.type, c.pages, c.heads, c.page_size, c.size = pkg.S8, 2, 2, 16, 64
    assert write(tokens=0) == 0 and write(keys=None) == 1 and write(type=pkg.F32) == 1
    for name, value in (("type", pkg.U8), ("pages", 0), ("heads", 0), ("page_size", 0), ("size", 0), ("size", 12), ("size", 264),
                        ("page_stride", 4), ("row_stride", 7), ("keys", 4100), ("key_scales", None), ("values", None), ("heads", 65536)):
        before = getattr(c, name)
        setattr(c, name, value)
        assert write() == 1 and read() == 1, (name, value)
        setattr(c, name, before)
    c.type, c.size, c.row_stride = pkg.F32, 60, 2
    assert write() == 1


CASES = [
    # type, heads, page, size, tokens, pages
    ("s8", 1, 1, 8, 1, 3),
    ("s8", 2, 16, 64, 5, 4),
    ("s8", 8, 32, 128, 77, 5),
    ("s8", 3, 24, 80, 40, 3),
    ("s8", 5, 7, 200, 33, 6),
    ("s8", 1, 16, 256, 9, 2),
    ("f32", 4, 16, 64, 21, 3),
    ("f32", 3, 10, 100, 17, 4),
    ("f32", 2, 5, 256, 11, 4),
]


def cache_of(pkg, kind, pages, heads, page, size):
    """A cache whose memory is marked."""
    import torch
    cache = pkg.paged_cache(pages, heads, page, size, torch.int8 if kind == "s8" else torch.float32)
    for i, t in enumerate(cache):
        t.fill_(77 if i < 2 else 7.75)
    return cache


@pytest.mark.gpu
@pytest.mark.parametrize("kind,heads,page,size,tokens,pages", CASES)
def test_written_bit_for_bit(pkg, T, kind, heads, page, size, tokens, pages):
    import torch
    rng = np.random.default_rng(size * 100 + tokens)
    x = [rng.normal(size=(tokens, heads, size)).astype(np.float32) * np.exp(rng.normal(size=(tokens, heads, 1)) * 6).astype(np.float32) for _ in range(2)]
    x[0][0, 0] = 0.0  # a row of zeros has scale 0
    if tokens > 3:
        # quotients on the borders: multiples of half a step of a scale of 2^-k, which are ties
        x[1][1, 0] = (rng.integers(-253, 254, size) * 0.5 * 0.25).astype(np.float32)
        x[1][1, 0, 0] = 127 * 0.25
        x[0][2, 0] *= np.float32(1e-43) / np.abs(x[0][2, 0]).max()  # subnormal, with a scale of one or two units
        x[1][2, 0] = np.float32(3e38)
        x[0][3, 0, 1] = np.nan
        x[1][3, 0, 2] = -np.inf
    slots = rng.permutation(pages * page)[:tokens]
    if tokens > 8:
        slots[4:8] = [-1, pages * page, -7, pages * page + 1000]  # skipped
    cache = cache_of(pkg, kind, pages, heads, page, size)
    want = [T.n(t).copy() for t in cache]
    for i, new in enumerate(x):
        n, scale = R.quantized(new)
        for t, slot in enumerate(slots):
            if 0 <= slot < pages * page:
                want[i][slot // page, :, slot % page] = n[t] if kind == "s8" else new[t]
                if kind == "s8":
                    want[2 + i][slot // page, :, slot % page] = scale[t]
    for dtype in (np.int64, np.int32):
        cache = cache_of(pkg, kind, pages, heads, page, size)
        pkg.cache_write(cache, T.t(x[0]), T.t(x[1]), T.t(slots.astype(dtype)))
        for g, w in zip(cache, want):
            assert np.array_equal(T.n(g), w, equal_nan=w.dtype != np.int8)


@pytest.mark.gpu
def test_every_integer_is_the_true_quotients(pkg, T):
    """Values next to every border between two integers, for scales of all mantissas."""
    import torch
    rng = np.random.default_rng(1)
    scale = np.float32(1) + rng.integers(0, 2 ** 23, 4096).astype(np.float32) * np.float32(2.0 ** -23)
    top = scale * np.float32(127)
    scale = top * np.float32(1 / 127)
    border = ((np.arange(63) * 2 - 62.0) + 0.5)[None] * scale[:, None].astype(np.float64)
    rows = np.zeros((4096, 64), np.float32)
    rows[:, 0] = top
    rows[:, 1:] = np.nextafter(border.astype(np.float32), np.float32(np.inf) * rng.choice([-1, 1], border.shape).astype(np.float32))
    half = rng.random(border.shape) < 0.5
    rows[:, 1:] = np.where(half, border.astype(np.float32), rows[:, 1:])
    cache = pkg.paged_cache(64, 1, 64, 64)
    pkg.cache_write(cache, T.t(rows[:, None]), T.t(-rows[:, None]), T.t(np.arange(4096, dtype=np.int32)))
    n, s = R.quantized(rows)
    assert np.array_equal(T.n(cache[2]).reshape(-1), s)
    assert np.array_equal(T.n(cache[0]).reshape(4096, 64), n)
    assert np.array_equal(T.n(cache[1]).reshape(4096, 64), R.quantized(-rows)[0])


def strided(cache):
    """The same contents with rows before heads, in memory that is wider than the head."""
    import torch
    out = []
    for t in cache:
        if t.dim() == 4:
            wide = torch.zeros((t.shape[0], t.shape[2], t.shape[1], t.shape[3] + 16), dtype=t.dtype, device=t.device)
            view = wide[..., :t.shape[3]].transpose(1, 2)
        else:
            view = torch.zeros((t.shape[0], t.shape[2], t.shape[1]), dtype=t.dtype, device=t.device).transpose(1, 2)
        view.copy_(t)
        out.append(view)
    return tuple(out)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,heads,page,size,tokens,pages", CASES)
def test_read_back(pkg, T, kind, heads, page, size, tokens, pages):
    import torch
    rng = np.random.default_rng(size + tokens)
    cache = pkg.paged_cache(pages, heads, page, size, torch.int8 if kind == "s8" else torch.float32)
    if kind == "s8":
        for t in cache[:2]:
            t.copy_(T.t(rng.integers(-127, 128, t.shape, dtype=np.int8)))
        for t in cache[2:]:
            t.copy_(T.t(rng.random(t.shape).astype(np.float32)))
    else:
        for t in cache:
            t.copy_(T.t(rng.normal(size=t.shape).astype(np.float32)))
    lengths = [min(page * pages, n) for n in (0, page + 1, 1, 0, 2 * page, page - 1)]
    table = np.stack([rng.permutation(pages) for _ in lengths]).astype(np.int32)
    starts = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    table[1, 0], total = pages, int(starts[-1]) + 3
    if pages > 1:
        table[4, 1] = -1
    flat = [t.astype(np.float32) * s[..., None] for t, s in zip(map(T.n, cache[:2]), map(T.n, cache[2:]))] if kind == "s8" else [T.n(t) for t in cache]
    for held in (cache, strided(cache)):
        d = pkg._cache_desc(held)
        out = [torch.full((total, heads, size), 5.5, device="cuda") for _ in range(2)]
        on, begin = T.t(table), T.t(starts)
        pkg.check(pkg.lib().tfcc_rocm_cache_read(pkg._stream(), C.byref(d), on.data_ptr(), pages, pages, len(lengths), begin.data_ptr(),
                                                 total, out[0].data_ptr(), out[1].data_ptr()))
        again = pkg.cache_read(held, T.t(table), T.t(starts), total)
        for x, y, f in zip(out, again, flat):
            want = np.full((total, heads, size), 5.5, np.float32)
            for i, n in enumerate(lengths):
                at = np.arange(n)
                named = table[i][at // page]
                there = (named >= 0) & (named < pages)
                want[starts[i]:starts[i + 1]] = np.where(there[:, None, None], f[np.where(there, named, 0), :, at % page], 0)
            assert np.array_equal(T.n(x), want)
            assert np.array_equal(T.n(y)[:starts[-1]], want[:starts[-1]])


@pytest.mark.gpu
def test_strided_writes(pkg, T):
    import torch
    rng = np.random.default_rng(3)
    x = [T.t(rng.normal(size=(6, 4, 64)).astype(np.float32)) for _ in range(2)]
    slots = T.t(np.array([3, 0, 17, 31, 8, 16], np.int64))
    for dtype in (torch.int8, torch.float32):
        cache = pkg.paged_cache(2, 4, 16, 64, dtype)
        other = strided(cache)
        pkg.cache_write(cache, *x, slots)
        wide = torch.zeros((6, 3, 4, 65), device="cuda")
        views = [wide[:, i, :, 1:] for i in (0, 2)]
        for v, t in zip(views, x):
            v.copy_(t)
        pkg.cache_write(other, *views, slots)
        for a, b in zip(cache, other):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_refused(pkg, T):
    import torch
    cache = pkg.paged_cache(2, 4, 16, 64)
    x, slots = torch.zeros((6, 4, 64), device="cuda"), torch.zeros(6, dtype=torch.int32, device="cuda")
    starts, table = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros((1, 2), dtype=torch.int32, device="cuda")
    for args in ((cache[:3], x, x, slots), (cache[:2], x, x, slots), (cache, x[:, :3], x[:, :3], slots), (cache, x, x[:5], slots),
                 (cache, x.half(), x, slots), (cache, x, x, slots[:5]), (cache, x, x, slots.float()), (cache, x, x, slots.cpu()),
                 ((cache[0], cache[1][:1], *cache[2:]), x, x, slots), ((*cache[:3], cache[3][:1]), x, x, slots)):
        with pytest.raises(pkg.InvalidArgumentError):
            pkg.cache_write(*args)
    for args in ((cache, table.long(), starts, 3), (cache, table, starts[:1], 3), (cache, table, starts, -1)):
        with pytest.raises(pkg.InvalidArgumentError):
            pkg.cache_read(*args)
    with pytest.raises(pkg.TfccRocmError):
        pkg.cache_write(pkg.paged_cache(2, 4, 16, 12), torch.zeros((6, 4, 12), device="cuda"), torch.zeros((6, 4, 12), device="cuda"), slots)
    with pytest.raises(pkg.InvalidArgumentError):
        pkg.paged_cache(1, 1, 1, 8, torch.float16)
    assert pkg.cache_read(cache, table, starts, 0)[0].shape == (0, 4, 64)
    pkg.cache_write(cache, x[:0], x[:0], slots[:0])
