"""A cache whose rows share memory can be read but not written."""
import ctypes as C

import numpy as np
import pytest

import generation_reference as R


def cache_of(pkg, kind):
    c = pkg.PagedCache()
    c.keys = c.values = c.key_scales = c.value_scales = 4096
    c.type, c.pages, c.heads, c.page_size, c.size = kind, 2, 3, 16, 64
    c.row_stride, c.head_stride, c.page_stride = 64, 16 * 64, 3 * 16 * 64
    c.scale_row_stride, c.scale_head_stride, c.scale_page_stride = 1, 16, 48
    return c


@pytest.mark.parametrize("name,dimension", [("page_stride", "pages"), ("head_stride", "heads"), ("row_stride", "page_size"), ("scale_page_stride", "pages"),
                                            ("scale_head_stride", "heads"), ("scale_row_stride", "page_size")])
def test_writes_refused_without_a_device(pkg, name, dimension):
    lib = pkg.lib()
    for kind in (pkg.S8, pkg.F32):
        c = cache_of(pkg, kind)
        write = lambda keys=None: lib.tfcc_rocm_cache_write(None, C.byref(c), keys, 0, 0, 64, 0, 0, 1, 64, pkg.S32)
        assert write() == 1 and b"null" in lib.tfcc_rocm_last_error_string()  # all else is in order
        setattr(c, name, 0)
        assert write() == 1
        refused = b"stride of 0" in lib.tfcc_rocm_last_error_string()
        assert refused == (kind == pkg.S8 or not name.startswith("scale"))  # float32 has no scales
        setattr(c, dimension, 1)
        assert write() == 1 and b"null" in lib.tfcc_rocm_last_error_string()  # a single one needs no stride


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["s8", "f32"])
def test_shared_memory_is_read_and_not_written(pkg, T, kind):
    import torch
    rng = np.random.default_rng(4)
    cache = pkg.paged_cache(1, 1, 16, 64, torch.int8 if kind == "s8" else torch.float32)
    x = T.t(rng.normal(size=(16, 1, 64)).astype(np.float32))
    pkg.cache_write(cache, x, x, T.t(np.arange(16, dtype=np.int32)))
    shared = tuple(t.expand(3, 2, *t.shape[2:]) for t in cache)
    before = [t.clone() for t in cache]
    two = T.t(rng.normal(size=(4, 2, 64)).astype(np.float32))
    with pytest.raises(pkg.TfccRocmError):
        pkg.cache_write(shared, two, two, T.t(np.array([0, 16, 32, 5], np.int32)))
    assert all(torch.equal(a, b) for a, b in zip(cache, before))
    table, starts = T.t(np.array([[2, 0]], np.int32)), T.t(np.array([0, 20], np.int32))
    keys, _ = pkg.cache_read(shared, table, starts, 20)
    one, _ = pkg.cache_read(cache, T.t(np.array([[0, 0]], np.int32)), starts, 20)
    assert torch.equal(keys, one.expand(20, 2, 64))
    q = T.t(rng.normal(size=(1, 4, 64)).astype(np.float32))
    lengths, starts = T.t(np.array([20], np.int32)), T.t(np.array([0, 1], np.int32))
    dense = tuple(t.contiguous() for t in shared)
    assert torch.equal(pkg.paged_attention(q, shared, table, starts, lengths, 0.125), pkg.paged_attention(q, dense, table, starts, lengths, 0.125))
