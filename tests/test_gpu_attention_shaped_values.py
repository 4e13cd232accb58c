"""Attention with shaped scores at the ends of what its arguments may hold: caps below float32's smallest number, slopes next to its largest."""
import numpy as np
import pytest

from test_gpu_attention_shaped import Made


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
