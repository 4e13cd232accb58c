"""Counts beyond 32 bits in the Python forms of the generation calls: refused, or as good as the largest that 32 bits hold."""
import numpy as np
import pytest


@pytest.mark.gpu
def test_bounds_and_windows_beyond_32_bits(pkg, T):
    """A bound of 2^32 + 100 is not one of 100."""
    import generation_reference as R
    from test_gpu_paged_attention import Made
    m = Made(pkg, "s8", [700, 90], [3, 20], 4, 2, 64, 16, 3)
    want = T.n(m.run(T))
    for most in (2 ** 31 - 1, 2 ** 31, 2 ** 32 - 1, 2 ** 32 + 100, 2 ** 70):
        assert np.array_equal(T.n(m.run(T, max_length=most)), want), most
        assert np.array_equal(T.n(m.run(T, window=most)), want), most
    assert not np.array_equal(T.n(m.run(T, max_length=100)), want) and not np.array_equal(T.n(m.run(T, window=100)), want)


@pytest.mark.gpu
def test_tensors_beyond_32_bits_are_refused(pkg, T):
    """Dimensions that only a stride of 0 makes, before anything of that size is allocated."""
    import torch
    m, far = 2 ** 32 + 1, 2 ** 31
    x = torch.zeros((1, 1, 16), device="cuda")
    cache = pkg.paged_cache(1, 1, 16, 16)
    i32 = torch.zeros(2, dtype=torch.int32, device="cuda")
    f = torch.ones(8, dtype=torch.float64, device="cuda")
    for n in (m, far):
        wide = x.expand(n, 1, 16)
        for call in (lambda: pkg.rotary(wide, None, i32, f), lambda: pkg.rotary(x.expand(1, n, 16), None, i32[:1], f),
                     lambda: pkg.cache_write(cache, wide, wide, i32), lambda: pkg.cache_read(cache, i32[None], i32, n),
                     lambda: pkg.cache_write(tuple(t.expand(n, *t.shape[1:]) for t in cache), x, x, i32[:1]),
                     lambda: pkg.cache_read(tuple(t.expand(n, *t.shape[1:]) for t in cache), i32[None], i32, 1),
                     lambda: pkg.cache_read(cache, i32[:1, None].expand(1, n), i32, 1), lambda: pkg.paged_attention(wide, cache, i32[None], i32, i32[:1], 1.0),
                     lambda: pkg.sample(torch.zeros((1, 1), device="cuda").expand(n, 1), torch.zeros(1, device="cuda")),
                     lambda: pkg.sample(torch.zeros((1, 1), device="cuda").expand(1, n), torch.zeros(1, device="cuda"))):
            with pytest.raises(pkg.InvalidArgumentError):
                call()
    with pytest.raises(pkg.InvalidArgumentError):
        pkg.cache_read(cache, i32[None], i32, -1)
