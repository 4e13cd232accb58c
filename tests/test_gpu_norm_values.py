"""The norm's float32 result and its integers asked for in one call: neither changes the other, whatever the rows and the weight hold."""
import ctypes as C

import numpy as np
import pytest

import serving_reference as R
from generation_reference import EPS
from test_gpu_norm import desc


def both(pkg, T, x, w, eps=1e-6):
    """(out, steps, scales, sums) of one call."""
    import torch
    rows, width = x.shape
    x, w = T.t(x), T.t(w)
    out, steps = torch.empty((rows, width), device="cuda"), torch.empty((rows, width), dtype=torch.uint8, device="cuda")
    scales, sums = torch.empty(rows, device="cuda"), torch.empty(rows, dtype=torch.int32, device="cuda")
    d = desc(pkg, rows=rows, width=width, eps=eps, x=x.data_ptr(), weight=w.data_ptr(), out=out.data_ptr(), steps=steps.data_ptr(), scales=scales.data_ptr(),
             sums=sums.data_ptr(), x_row_stride=width, out_row_stride=width, steps_row_stride=width)
    pkg.check(pkg.lib().tfcc_rocm_rms_norm_f32(pkg._stream(), C.byref(d)))
    return tuple(T.n(t) for t in (out, steps, scales, sums))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,width", [(6, 40), (6, 100), (6, 700), (300, 700), (6, 3000), (300, 2000), (6, 9000), (6, 17000)])
@pytest.mark.parametrize("weight", [1.0, np.inf, -np.inf, np.nan, 0.0])
def test_out_beside_steps_of_rows_that_are_not_finite(pkg, T, rows, width, weight):
    """An infinity or a NaN of a row, or of the weight, concerns in `out` what the formula says, with steps or without: an infinite value brings the others to 0, a
    weight of infinity its own column alone."""
    rng = np.random.default_rng(width)
    x, w = rng.normal(size=(rows, width)).astype(np.float32), (rng.random(width) + 0.5).astype(np.float32)
    x[1, 3], x[3, width - 1], x[4, 0] = np.inf, np.nan, -np.inf
    if weight != 1.0:
        w[5] = weight
    with np.errstate(invalid="ignore"):
        _, y, t, _ = R.norm(x, w, np.float64(np.float32(1e-6)))
    out, steps, scales, sums = both(pkg, T, x, w)
    alone = T.n(pkg.rms_norm(T.t(x), T.t(w), 1e-6)[0])
    for got in (out, alone):
        got = got.astype(np.float64)
        assert np.array_equal(np.isnan(got), np.isnan(y)) and np.array_equal(got[np.isinf(y)], y[np.isinf(y)])
        fine = np.isfinite(y)
        assert (np.abs(got[fine] - y[fine]) <= (EPS + 2.0 ** -40) * np.abs(y[fine]) + 2.0 ** -149).all()  # float32's last rounding, and 2^-40 for all before it
    bad = ~np.isfinite(t).all(-1)
    assert np.array_equal(np.isnan(scales), bad) and (steps[bad] == 128).all() and (sums[bad] == 128 * width).all()
    want = [T.n(v) for v in pkg.rms_norm_quantized(T.t(x), T.t(w), 1e-6)[:3]]
    assert np.array_equal(steps, want[0]) and np.array_equal(scales, want[1], equal_nan=True) and np.array_equal(sums, want[2])
    if not bad.all():
        t = t[~bad][:2]
        assert np.array_equal(steps[~bad][:2], 128 + R.norm_steps(t, np.abs(t).max(-1, keepdims=True)))


@pytest.mark.gpu
@pytest.mark.parametrize("eps", [1e-46, 1e-60, 5e-324, 2.0 ** -150, -1e-60])
def test_an_eps_that_float32_does_not_hold(pkg, T, eps):
    """Rounded to float32 it would be 0, and a row of zeros 0 / 0."""
    x, w = T.t(np.zeros((2, 8), np.float32)), T.t(np.ones(8, np.float32))
    for call in (pkg.rms_norm, pkg.rms_norm_quantized):
        with pytest.raises(pkg.InvalidArgumentError):
            call(x, w, eps)
    assert (T.n(pkg.rms_norm(x, w, 2.0 ** -149)[0]) == 0).all() and np.isnan(T.n(pkg.rms_norm(x, w, 0.0)[0])).all()
