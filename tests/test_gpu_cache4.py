"""A paged cache of 4-bit integers written and read, and runs of rows copied inside caches of all types, against the definitions."""
import ctypes as C

import numpy as np
import pytest

import serving_reference as R


def dtype_of(kind):
    import torch
    return {"s4": torch.uint8, "s8": torch.int8, "f32": torch.float32}[kind]


def described(pkg, kind):
    c = pkg.PagedCache()
    c.keys = c.values = c.key_scales = c.value_scales = 4096
    c.type, c.pages, c.heads, c.page_size, c.size = kind, 2, 3, 16, 64
    width = 32 if kind == pkg.S4 else 64
    c.row_stride, c.head_stride, c.page_stride = width, 16 * width, 3 * 16 * width
    c.scale_row_stride, c.scale_head_stride, c.scale_page_stride = 1, 16, 48
    return c


def test_refused_without_a_device(pkg):
    lib, c = pkg.lib(), described(pkg, pkg.S4)
    write = lambda keys=64: lib.tfcc_rocm_cache_write(None, C.byref(c), keys, 0, 0, 64, 0, 0, 1, 64, pkg.S32)
    read = lambda table=64: lib.tfcc_rocm_cache_read(None, C.byref(c), table, 0, 1, 1, 64, 1, 64, 64)
    copy = lambda sources=64, kind=pkg.S32, runs=1: lib.tfcc_rocm_cache_copy(None, C.byref(c), sources, 64, kind, None, runs)
    assert lib.tfcc_rocm_cache_copy(None, None, 64, 64, pkg.S32, None, 1) == 1
    assert copy(runs=0) == 0 and copy(kind=pkg.F32) == 1 and copy(kind=pkg.S4) == 1
    for call in (write, read, copy):
        assert call(None) == 1 and b"null argument" in lib.tfcc_rocm_last_error_string()
    for name, value in (("type", pkg.U8), ("pages", 0), ("heads", 0), ("page_size", 0), ("size", 0), ("size", 8), ("size", 40), ("size", 272),
                        ("page_stride", 4), ("row_stride", 12), ("keys", 4100), ("key_scales", None), ("values", None), ("heads", 65536)):
        before = getattr(c, name)
        setattr(c, name, value)
        assert write() == 1 and read() == 1 and copy() == 1, (name, value)
        setattr(c, name, before)


@pytest.mark.parametrize("name,dimension", [("page_stride", "pages"), ("head_stride", "heads"), ("row_stride", "page_size"), ("scale_page_stride", "pages"),
                                            ("scale_head_stride", "heads"), ("scale_row_stride", "page_size")])
def test_shared_memory_is_not_written(pkg, name, dimension):
    lib = pkg.lib()
    for kind in (pkg.S4, pkg.S8, pkg.F32):
        c = described(pkg, kind)
        copy = lambda: lib.tfcc_rocm_cache_copy(None, C.byref(c), None, 64, pkg.S32, None, 1)
        assert copy() == 1 and b"null" in lib.tfcc_rocm_last_error_string()
        setattr(c, name, 0)
        assert copy() == 1
        assert (b"stride of 0" in lib.tfcc_rocm_last_error_string()) == (kind != pkg.F32 or not name.startswith("scale"))
        setattr(c, dimension, 1)
        assert copy() == 1 and b"null" in lib.tfcc_rocm_last_error_string()


def test_copies_of_more_than_one_launch(pkg):
    lib, c = pkg.lib(), described(pkg, pkg.S4)
    said = lambda runs: (lib.tfcc_rocm_cache_copy(None, C.byref(c), None, 64, pkg.S32, None, runs), lib.tfcc_rocm_last_error_string())
    # 3 heads of 16 rows of 32 bytes: a workgroup for the rows, one for the scales
    assert b"null" in said((1 << 22) - 1)[1] and b"runs of" in said(1 << 22)[1] and b"runs of" in said(0xffffffff)[1]
    c.heads, c.page_size, c.size = 65535, 1 << 24, 256
    assert b"runs of" in said(1)[1]


WRITTEN = [(1, 16, 16, 1, 2), (2, 16, 64, 40, 4), (3, 24, 48, 30, 3), (1, 7, 80, 20, 5), (8, 32, 128, 33, 2), (2, 64, 256, 100, 3), (5, 1, 144, 3, 9)]


@pytest.mark.gpu
@pytest.mark.parametrize("heads,page,size,tokens,pages", WRITTEN)
def test_written_bit_for_bit(pkg, T, heads, page, size, tokens, pages):
    import torch
    rng = np.random.default_rng(size * 100 + tokens)
    x = [rng.normal(size=(tokens, heads, size)).astype(np.float32) * np.exp(rng.normal(size=(tokens, heads, 1)) * 6).astype(np.float32) for _ in range(2)]
    x[0][0, 0] = 0.0  # a row of zeros has scale 0
    if tokens > 3:
        x[1][1, 0] = (rng.integers(-13, 14, size) * 0.5 * 0.25).astype(np.float32)  # ties
        x[1][1, 0, 0] = 7 * 0.25
        x[0][2, 0] *= np.float32(1e-44) / np.abs(x[0][2, 0]).max()  # subnormal, with a scale of a unit or none
        x[1][2, 0] = np.float32(3e38)
        x[0][3, 0, 1] = np.nan
        x[1][3, 0, 2] = -np.inf
    slots = rng.permutation(pages * page)[:tokens]
    if tokens > 8:
        slots[[4, 6]] = [-1, pages * page]  # skipped
    for kind in (np.int32, np.int64):
        cache = pkg.paged_cache(pages, heads, page, size, torch.uint8)
        before = [rng.integers(0, 256, tuple(t.shape)).astype(np.uint8) if t.dtype == torch.uint8 else rng.random(tuple(t.shape)).astype(np.float32) for t in cache]
        for t, b in zip(cache, before):
            t.copy_(T.t(b))
        pkg.cache_write(cache, T.t(x[0]), T.t(x[1]), T.t(slots.astype(kind)))
        want = [b.copy() for b in before]
        for i, s in enumerate(slots):
            if 0 <= s < pages * page:
                for held in (0, 1):
                    n, scale = R.quantized4(x[held][i])
                    want[held][s // page, :, s % page], want[2 + held][s // page, :, s % page] = R.pack(n), scale
        for got, w in zip(cache, want):
            assert np.array_equal(T.n(got), w, equal_nan=w.dtype == np.float32)


@pytest.mark.gpu
def test_every_integer_is_the_true_quotients(pkg, T):
    """Values next to every border between two integers, for scales of all mantissas."""
    import torch
    rng = np.random.default_rng(1)
    top = (np.float32(1) + rng.integers(0, 2 ** 23, 4096).astype(np.float32) * np.float32(2.0 ** -23)) * np.float32(7)
    scale = top * np.float32(1 / 7)
    border = (rng.integers(-7, 7, (4096, 63)) + 0.5) * scale[:, None].astype(np.float64)
    rows = np.zeros((4096, 64), np.float32)
    rows[:, 0] = top
    rows[:, 1:] = np.nextafter(border.astype(np.float32), np.float32(np.inf) * rng.choice([-1, 1], border.shape).astype(np.float32))
    rows[:, 1:] = np.where(rng.random(border.shape) < 0.5, border.astype(np.float32), rows[:, 1:])
    cache = pkg.paged_cache(64, 1, 64, 64, torch.uint8)
    pkg.cache_write(cache, T.t(rows[:, None]), T.t(-rows[:, None]), T.t(np.arange(4096, dtype=np.int32)))
    n, s = R.quantized4(rows)
    for i, sign in ((0, 1), (1, -1)):
        assert np.array_equal(T.n(cache[i]).reshape(4096, 32), R.pack(sign * n)) and np.array_equal(T.n(cache[2 + i]).reshape(-1), s)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,most", [("uint8", 7), ("int8", 127)])
@pytest.mark.parametrize("size", [32, 128, 256])
def test_scales_of_all_exponents(pkg, T, kind, most, size):
    """From subnormal ones to float32's largest, with values on the borders between two integers, next to them and elsewhere."""
    import torch
    rng = np.random.default_rng(size)
    top = np.ldexp(1 + rng.random(1024), rng.permutation(np.arange(1024) % 276) - 148).astype(np.float32)
    top[:2] = np.float32(3.4028234e38), np.float32(2.0 ** -149)
    scale = top * np.float32(1 / most)
    border = (rng.integers(-most, most, (1024, size)) + 0.5) * scale[:, None].astype(np.float64)
    with np.errstate(over="ignore", under="ignore"):
        rows = border.astype(np.float32)
        near = np.nextafter(rows, np.float32(np.inf) * rng.choice([-1, 1], rows.shape).astype(np.float32))
        rows = np.where(rng.random(rows.shape) < 0.4, near, rows)
        rows = np.where(rng.random(rows.shape) < 0.3, (rng.uniform(-1, 1, rows.shape) * top[:, None].astype(np.float64)).astype(np.float32), rows)
    rows = np.clip(rows, -top[:, None], top[:, None])
    rows[:, size - 1] = top
    cache = pkg.paged_cache(64, 1, 16, size, getattr(torch, kind))
    pkg.cache_write(cache, T.t(rows[:, None]), T.t(-rows[:, None]), T.t(np.arange(1024, dtype=np.int32)))
    good = scale > 0
    n = np.rint(rows.astype(np.float64) / np.where(good, scale, 1).astype(np.float64)[:, None])
    n = np.where(good[:, None], np.clip(n, -most, most), 0).astype(np.int8)
    for i, sign in ((0, 1), (1, -1)):
        want = R.pack(sign * n) if kind == "uint8" else sign * n
        assert np.array_equal(T.n(cache[i]).reshape(1024, -1), want) and np.array_equal(T.n(cache[2 + i]).reshape(-1), scale)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,page,size,tokens,pages", WRITTEN)
def test_read_back(pkg, T, heads, page, size, tokens, pages):
    import torch
    rng = np.random.default_rng(size + tokens)
    cache = pkg.paged_cache(pages, heads, page, size, torch.uint8)
    for t in cache[:2]:
        t.copy_(T.t(rng.integers(0, 256, tuple(t.shape)).astype(np.uint8)))  # all integers, -8 among them
    for t in cache[2:]:
        t.copy_(T.t(rng.random(tuple(t.shape)).astype(np.float32)))
    lengths = [min(page * pages, n) for n in (0, page + 1, 1, 0, 2 * page, page - 1)]
    table = np.stack([rng.permutation(pages) for _ in lengths]).astype(np.int32)
    table[4, -1] = pages  # outside
    starts = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    keys, values = pkg.cache_read(cache, T.t(table), T.t(starts), int(starts[-1]))
    for held, got in ((0, T.n(keys)), (1, T.n(values))):
        n, s = R.unpack(T.n(cache[held])), T.n(cache[2 + held])
        want = []
        for i, length in enumerate(lengths):
            for at in range(length):
                p = table[i, at // page]
                want.append(n[p, :, at % page].astype(np.float32) * s[p, :, at % page][:, None] if p < pages else np.zeros((heads, size), np.float32))
        assert np.array_equal(got, np.array(want))


def filled(pkg, T, kind, pages, heads, page, size, seed):
    rng = np.random.default_rng(seed)
    cache = pkg.paged_cache(pages, heads, page, size, dtype_of(kind))
    for t in cache:
        b = rng.integers(0, 256, tuple(t.shape)).astype(np.uint8)
        t.copy_(T.t(rng.normal(size=tuple(t.shape)).astype(np.float32) if t.is_floating_point() else b.view(np.int8) if kind == "s8" else b))
    return cache


COPIED = [(1, 16, 64, 6), (8, 32, 128, 20), (3, 24, 80, 9), (5, 7, 48, 12), (2, 1, 16, 30), (12, 200, 256, 7), (4, 64, 208, 40),
          (1, 16, 256, 600), (3, 24, 80, 512), (8, 16, 128, 510), (8, 100, 128, 530), (1, 1, 16, 700)]  # more runs and fewer than scales go apart for


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["s4", "s8", "f32"])
@pytest.mark.parametrize("heads,page,size,pages", COPIED)
def test_copies(pkg, T, kind, heads, page, size, pages):
    """Whole pages, parts of pages at other rows, several copies of one, and runs that are skipped or cut at a page's end."""
    rng = np.random.default_rng(pages)
    order = rng.permutation(pages)
    runs = pages // 2
    for rows in (None, rng.integers(-1, page + 3, runs).astype(np.int32)):
        for slots in (np.int32, np.int64):
            cache = filled(pkg, T, kind, pages, heads, page, size, pages)
            before = [T.n(t).copy() for t in cache]
            sources = order[rng.integers(0, runs, runs)] * page + rng.integers(0, page, runs) * (rng.random(runs) < 0.5)
            destinations = order[runs:2 * runs] * page + rng.integers(0, page, runs) * (rng.random(runs) < 0.5)
            if runs > 4:
                sources[1], destinations[2], sources[3] = -1, pages * page, pages * page + 5
            pkg.cache_copy(cache, T.t(sources.astype(slots)), T.t(destinations.astype(slots)), None if rows is None else T.t(rows))
            for got, want in zip(cache, R.copied(before, sources, destinations, rows)):
                assert np.array_equal(T.n(got), want)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["s4", "s8", "f32"])
def test_copies_and_writes_of_strided_caches(pkg, T, kind):
    """Keys and values of one allocation, rows with gaps, heads inside rows: other memory stays as it was."""
    import torch
    heads, page, size, pages = 4, 16, 64, 6
    cache = filled(pkg, T, kind, pages, heads, page, size, 0)
    rng = np.random.default_rng(1)
    x = [T.t(rng.normal(size=(5, heads, size)).astype(np.float32)) for _ in range(2)]
    slots, sources, destinations = (T.t(np.array(v, np.int64)) for v in ([3, 90, 17, 31, 64], [0, 20, 33], [80, 68, 50]))
    width = cache[0].shape[3]
    memory = torch.full((pages, page, heads, 2, width + 16), 77, dtype=cache[0].dtype, device="cuda")
    views = [memory[:, :, :, i, 8 if kind != "f32" else 16:][..., :width].permute(0, 2, 1, 3) for i in (0, 1)]
    if kind != "f32":
        scales = torch.full((pages, page, 2, heads + 3), 5.0, device="cuda")
        views += [scales[:, :, i, 1:1 + heads].permute(0, 2, 1) for i in (0, 1)]
    for v, t in zip(views, cache):
        v.copy_(t)
    for c in (cache, tuple(views)):
        pkg.cache_write(c, *x, slots)
        pkg.cache_copy(c, sources, destinations, T.t(np.array([16, 9, 40], np.int32)))
    for v, t in zip(views, cache):
        assert torch.equal(v, t)
        v.fill_(77 if v.dim() == 4 else 5)
    assert (memory == 77).all() and (kind == "f32" or (scales == 5).all())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["s4", "f32"])
def test_copies_beyond_32_bits(pkg, T, kind):
    """Pages further apart than 2^32 elements."""
    import torch
    heads, page, size = 2, 16, 64
    width = size // 2 if kind == "s4" else size
    far = (1 << 32) + 4096 if kind == "s4" else (1 << 31) + 4096
    memory = [torch.empty((far + 8192,), dtype=dtype_of(kind), device="cuda") for _ in range(2)]
    cache = tuple(torch.as_strided(m, (2, heads, page, width), (far, page * width, width, 1)) for m in memory)
    if kind == "s4":
        cache += tuple(torch.zeros((2, heads, page), device="cuda") for _ in range(2))
    x = [T.t(np.random.default_rng(i).normal(size=(3, heads, size)).astype(np.float32)) for i in range(2)]
    pkg.cache_write(cache, *x, T.t(np.array([1, 2, 3], np.int32)))
    pkg.cache_copy(cache, T.t(np.array([1], np.int32)), T.t(np.array([page + 5], np.int32)), T.t(np.array([3], np.int32)))
    for t in cache:
        assert torch.equal(t[0, :, 1:4], t[1, :, 5:8]) and t[0, :, 1:4].any()


@pytest.mark.gpu
def test_captured_copies(pkg, T):
    """What the slots hold is read when the graph runs."""
    import torch
    cache = filled(pkg, T, "s4", 8, 2, 16, 64, 3)
    sources, destinations, rows = (T.t(np.array(v, np.int32)) for v in ([0, 16], [64, 80], [16, 5]))
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        with torch.cuda.graph(graph, stream=stream):
            pkg.cache_copy(cache, sources, destinations, rows)
    for a, b, n in (([0, 16], [64, 80], [16, 5]), ([33, 16], [112, 96], [3, 16]), ([-1, 0], [5, 97], [4, 4])):
        fresh = filled(pkg, T, "s4", 8, 2, 16, 64, n[0])
        before = [T.n(t).copy() for t in fresh]
        for t, f in zip(cache, fresh):
            t.copy_(f)
        for t, v in ((sources, a), (destinations, b), (rows, n)):
            t.copy_(T.t(np.array(v, np.int32)))
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(cache, R.copied(before, a, b, n)):
            assert np.array_equal(T.n(got), want)


@pytest.mark.gpu
def test_refused(pkg, T):
    import torch
    cache = pkg.paged_cache(2, 4, 16, 64, torch.uint8)
    x, slots = torch.zeros((6, 4, 64), device="cuda"), torch.zeros(6, dtype=torch.int32, device="cuda")
    for args in ((cache[:2], x, x, slots), (cache, x[..., :32].contiguous(), x[..., :32].contiguous(), slots), ((cache[0].view(torch.int8), *cache[1:]), x, x, slots)):
        with pytest.raises(pkg.InvalidArgumentError):
            pkg.cache_write(*args)
    for args in ((cache, slots, slots[:5]), (cache, slots, slots.long()), (cache, slots.float(), slots.float()), (cache, slots, slots, slots[:3]), (cache, slots, slots, slots.long()),
                 (cache, slots.cpu(), slots), (cache, slots[None], slots[None]), (cache[:3], slots, slots)):
        with pytest.raises(pkg.InvalidArgumentError):
            pkg.cache_copy(*args)
    for size in (8, 40, 272):
        odd = pkg.paged_cache(2, 4, 16, size, torch.uint8)
        with pytest.raises(pkg.TfccRocmError):
            pkg.cache_copy(odd, slots[:1], slots[:1])
    with pytest.raises(pkg.InvalidArgumentError):
        pkg.paged_cache(2, 4, 16, 63, torch.uint8)
    pkg.cache_copy(cache, slots[:0], slots[:0])
