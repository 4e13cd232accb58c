"""Root-mean-square norm as float32 and as 8-bit integers, and rows of integers back to float32, against the definitions in 64 bits."""
import ctypes as C

import numpy as np
import pytest

import serving_reference as R
from generation_reference import EPS


def desc(pkg, **given):
    d = pkg.RmsNormDesc()
    d.x = d.weight = d.out = 4096
    d.rows, d.width, d.eps = 2, 8, 1e-6
    d.x_row_stride = d.residual_row_stride = d.sum_row_stride = d.out_row_stride = d.steps_row_stride = 8
    for k, v in given.items():
        setattr(d, k, v)
    return d


def test_refused_without_a_device(pkg):
    lib = pkg.lib()
    call = lambda **k: lib.tfcc_rocm_rms_norm_f32(None, C.byref(desc(pkg, **k)))
    assert lib.tfcc_rocm_rms_norm_f32(None, None) == 1
    assert call(rows=0) == 0 and call(rows=0, out=None) == 0
    for given in ({"width": 0}, {"width": 1 << 24}, {"eps": -1.0}, {"eps": float("nan")}, {"eps": float("inf")}, {"out": None}, {"x": None}, {"weight": None},
                  {"steps": 8192}, {"scales": 8192}, {"sums": 8192}, {"sum": 4096}, {"sum": 4096, "out": 8192, "sum_row_stride": 16}, {"x_row_stride": 16},
                  {"residual": 8192, "sum": 8192, "sum_row_stride": 9}, {"residual": 4096}, {"out_row_stride": 0, "x": 8192}, {"out_row_stride": 7, "x": 8192},
                  {"sum": 8192, "sum_row_stride": 0}, {"steps": 8192, "scales": 1 << 20, "steps_row_stride": 7, "out": None}):
        assert call(**given) == 1, given
    for width, most in ((8, (1 << 26) - 4), (1024, (1 << 26) - 4), (1025, (1 << 24) - 1), (4096, (1 << 24) - 1), (4097, (1 << 22) - 1)):
        strides = {n: width for n in ("x_row_stride", "out_row_stride")}
        for rows, fits in ((most, True), (most + 1, False)):
            assert call(width=width, rows=rows, weight=None, **strides) == 1
            assert (b"null" if fits else b"rows") in lib.tfcc_rocm_last_error_string()
    rows = lambda *a: lib.tfcc_rocm_dequantize_rows(None, *a)
    assert rows(None, pkg.U8, 0, 8, 0, None, None, None) == 0 and rows(None, pkg.U8, 8, 0, 0, None, None, None) == 0
    for a in ((64, pkg.F32, 1, 1, 0, 64, None, 64), (64, pkg.S4, 1, 1, 0, 64, None, 64), (64, pkg.S16, 1, 1, 0, 64, None, 64), (None, pkg.U8, 1, 1, 0, 64, None, 64),
              (64, pkg.U8, 1, 1, 0, None, None, 64), (64, pkg.U8, 1, 1, 0, 64, None, None), (64, pkg.U8, 1 << 16, 1 << 15, 0, 64, None, 64)):
        assert rows(*a) == 1, a


def test_whole_number_steps_of_the_reference():
    """The reference's own rounding: ties, and quotients that are none."""
    t = np.array([[127.0, 0.5, 1.5, -2.5, 126.5, -0.5, 3.0, 0.0]])
    assert R.norm_steps(t, np.abs(t).max(-1, keepdims=True)).tolist() == [[127, 0, 2, -2, 126, 0, 3, 0]]
    t = np.array([[3.0, 1.0, -2.0, 1e-30, 0.0]])
    assert R.norm_steps(t, np.abs(t).max(-1, keepdims=True)).tolist() == [[127, 42, -85, 0, 0]]


WIDTHS = [1, 2, 3, 4, 5, 63, 64, 255, 768, 1003, 1024, 1025, 4095, 4096, 4097, 5000, 11008, 16384, 16385, 20001]


def check(T, pkg, x, w, eps, residual):
    """Both forms against the definition."""
    with np.errstate(over="ignore"):
        h, y, t, top = R.norm(x, w, np.float64(np.float32(eps)), residual)
    t_ = lambda a: None if a is None else T.t(a)
    out, held = pkg.rms_norm(t_(x), t_(w), eps, residual=t_(residual))
    assert (held is None) == (residual is None) and (held is None or np.array_equal(T.n(held), h))
    # 64-bit sums and products: float32's last rounding, and 2^-40 for all before it
    got = T.n(out).astype(np.float64)
    assert (np.abs(got - y) <= (EPS + 2.0 ** -40) * np.abs(y) + 2.0 ** -149).all()
    steps, scales, sums, held = pkg.rms_norm_quantized(t_(x), t_(w), eps, residual=t_(residual))
    assert steps.dtype.is_floating_point is False and (held is None or np.array_equal(T.n(held), h))
    n = T.n(steps).astype(np.int64)
    assert np.array_equal(n, 128 + R.norm_steps(t, top).reshape(n.shape))
    assert np.array_equal(T.n(sums), n.sum(-1))
    most = np.abs(y).max(-1)
    assert (np.abs(T.n(scales) - most / 127) <= (EPS + 2.0 ** -40) * most / 127 + 2.0 ** -149).all()
    back = T.n(pkg.dequantize_rows(steps, scales, offset=128))
    assert np.array_equal(back, (n - 128).astype(np.float32) * T.n(scales)[..., None])


@pytest.mark.gpu
@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("residual", [False, True])
def test_against_the_definition(pkg, T, width, residual):
    rng = np.random.default_rng(width)
    rows = 5 if width < 8000 else 2
    x = (rng.normal(size=(rows, width)) * np.exp(rng.normal(size=(rows, 1)) * 4)).astype(np.float32)
    w = (rng.random(width) + 0.5).astype(np.float32) * rng.choice([-1, 1], width).astype(np.float32)
    check(T, pkg, x, w, 1e-6, rng.normal(size=x.shape).astype(np.float32) if residual else None)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,width", [(1, 64), (33, 64), (1001, 63), (35, 128), (1003, 97), (300, 129), (301, 256), (299, 300), (257, 512), (600, 1030), (256, 1023), (257, 1023), (256, 2050), (257, 2050), (600, 4096), (300, 5001), (300, 9537)])
def test_few_rows_and_many(pkg, T, rows, width):
    rng = np.random.default_rng(rows + width)
    x = (rng.normal(size=(rows, width)) * np.exp(rng.normal(size=(rows, 1)) * 4)).astype(np.float32)
    check(T, pkg, x, (rng.random(width) + 0.5).astype(np.float32), 1e-6, rng.normal(size=x.shape).astype(np.float32))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 1, 16), (0, 8), (3, 0, 8), (2, 3, 5, 20), (300, 256), (16,)])
def test_shapes(pkg, T, shape):
    rng = np.random.default_rng(1)
    x, w = rng.normal(size=shape).astype(np.float32), np.ones(shape[-1], np.float32)
    if x.size:
        check(T, pkg, x, w, 1e-5, x[::-1].copy())
    out, held = pkg.rms_norm(T.t(x), T.t(w), 1e-5)
    steps, scales, sums, none = pkg.rms_norm_quantized(T.t(x), T.t(w), 1e-5)
    assert tuple(out.shape) == tuple(steps.shape) == shape and tuple(scales.shape) == tuple(sums.shape) == shape[:-1] and held is None and none is None


@pytest.mark.gpu
@pytest.mark.parametrize("width", [64, 1500, 5000])
def test_every_step_is_the_true_quotients(pkg, T, width):
    """Values next to the borders between two integers and on them, which no 32-bit quotient tells apart."""
    rng = np.random.default_rng(width)
    rows = 16
    top = (1 + rng.random(rows) * 2).astype(np.float32)
    top[:6] = 127 * 2.0 ** np.arange(-3, 3)  # ties that are exact
    border = (rng.integers(-126, 126, (rows, width)) + 0.5) * top[:, None].astype(np.float64) / 127
    x = np.nextafter(border.astype(np.float32), np.float32(np.inf) * rng.choice([-1, 1], border.shape).astype(np.float32))
    x = np.where(rng.random(border.shape) < 0.6, border.astype(np.float32), x)
    x[:, width // 2] = top
    check(T, pkg, x, np.full(width, 0.75, np.float32), 1e-6, None)
    w = (1 + rng.integers(0, 2 ** 23, width) * 2.0 ** -23).astype(np.float32)  # products of 48 bits
    check(T, pkg, (x / w).astype(np.float32), w, 0.0, None)


@pytest.mark.gpu
@pytest.mark.parametrize("width", [40, 3000, 9000, 17000])
def test_numbers_of_all_sizes(pkg, T, width):
    rng = np.random.default_rng(width)
    x = rng.normal(size=(6, width)).astype(np.float32)
    x[0] *= np.float32(1e38) / np.abs(x[0]).max()      # squares beyond float32
    x[1] *= np.float32(1e-42)                           # subnormal
    x[2] = 0
    x[3, 1:] *= np.float32(1e-30)
    x[4] *= np.float32(1e-25)                           # squares below float32
    check(T, pkg, x, np.ones(width, np.float32), 1e-6, None)
    check(T, pkg, x[[0, 1, 3, 4, 5]], np.full(width, 3, np.float32), 0.0, None)


@pytest.mark.gpu
@pytest.mark.parametrize("width", [40, 3000, 9000, 17000])
def test_rows_that_are_not_finite(pkg, T, width):
    rng = np.random.default_rng(width)
    x = rng.normal(size=(6, width)).astype(np.float32)
    x[1, 3], x[3, width - 1], x[4, 0] = np.inf, np.nan, -np.inf
    w = np.ones(width, np.float32)
    with np.errstate(invalid="ignore"):
        _, y, _, _ = R.norm(x, w, 1e-6)
    out = T.n(pkg.rms_norm(T.t(x), T.t(w), 1e-6)[0])
    assert np.array_equal(np.isnan(out), np.isnan(y)) and (out[[1, 4]][~np.isnan(y[[1, 4]])] == 0).all()
    steps, scales, sums, _ = (None if t is None else T.n(t) for t in pkg.rms_norm_quantized(T.t(x), T.t(w), 1e-6))
    bad = np.array([False, True, False, True, True, False])
    assert np.array_equal(np.isnan(scales), bad) and (steps[bad] == 128).all() and (sums[bad] == 128 * width).all()
    assert np.isnan(T.n(pkg.dequantize_rows(T.t(steps), T.t(scales), 128))[bad]).all()
    w[5] = np.inf  # a weight concerns all rows
    steps, scales, _, _ = pkg.rms_norm_quantized(T.t(x), T.t(w), 1e-6)
    assert np.isnan(T.n(scales)).all() and (T.n(steps) == 128).all()


@pytest.mark.gpu
@pytest.mark.parametrize("width", [37, 1003, 4097, 16400])
def test_in_place_and_strides(pkg, T, width):
    """The residual stream in its own memory, the result in the input's, rows further apart than they are wide, and what lies between them."""
    import torch
    rng = np.random.default_rng(width)
    x, r = (rng.normal(size=(3, width)).astype(np.float32) for _ in range(2))
    w = (rng.random(width) + 0.5).astype(np.float32)
    want, held = (T.n(t) for t in pkg.rms_norm(T.t(x), T.t(w), 1e-6, residual=T.t(r)))
    steps, scales, sums, _ = (T.n(t) for t in pkg.rms_norm_quantized(T.t(x), T.t(w), 1e-6, residual=T.t(r)))
    wide = width + 5
    memory = torch.full((3, 3, wide), 7.0, device="cuda")
    a, b, c = memory[0], memory[1], memory[2]
    a[:, :width].copy_(T.t(x))
    b[:, :width].copy_(T.t(r))
    held_steps = torch.full((3, wide), 9, dtype=torch.uint8, device="cuda")
    s, n = torch.empty(3, device="cuda"), torch.empty(3, dtype=torch.int32, device="cuda")
    weight = T.t(w)
    d = desc(pkg, rows=3, width=width, x=a.data_ptr(), residual=b.data_ptr(), sum=b.data_ptr(), out=a.data_ptr(), weight=weight.data_ptr(), steps=held_steps.data_ptr(),
             scales=s.data_ptr(), sums=n.data_ptr(), x_row_stride=wide, residual_row_stride=wide, sum_row_stride=wide, out_row_stride=wide, steps_row_stride=wide)
    pkg.check(pkg.lib().tfcc_rocm_rms_norm_f32(pkg._stream(), C.byref(d)))
    assert np.array_equal(T.n(a)[:, :width], want) and np.array_equal(T.n(b)[:, :width], held)
    assert np.array_equal(T.n(held_steps)[:, :width], steps) and np.array_equal(T.n(s), scales) and np.array_equal(T.n(n), sums)
    assert (T.n(memory)[:, :, width:] == 7).all() and (T.n(held_steps)[:, width:] == 9).all() and (T.n(c) == 7).all()
    # views of other strides, through the Python form
    view = torch.zeros((3, 2, wide), device="cuda")[:, 1, 2:2 + width]
    view.copy_(T.t(x))
    turned = T.t(np.ascontiguousarray(r.T)).T
    got = pkg.rms_norm(view, weight, 1e-6, residual=turned)
    assert np.array_equal(T.n(got[0]), want) and np.array_equal(T.n(got[1]), held)


@pytest.mark.gpu
def test_row_starts_beyond_32_bits(pkg, T):
    """Rows 2^31 values apart."""
    import torch
    far = (1 << 31) + 64
    memory = torch.empty((far + 64,), device="cuda")
    x = torch.as_strided(memory, (2, 40), (far, 1))
    rng = np.random.default_rng(0)
    a, w = rng.normal(size=(2, 40)).astype(np.float32), np.ones(40, np.float32)
    x.copy_(T.t(a))
    assert np.array_equal(T.n(pkg.rms_norm(x, T.t(w), 1e-6)[0]), T.n(pkg.rms_norm(T.t(a), T.t(w), 1e-6)[0]))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,width", [(1, 1), (5, 1), (7, 3), (1, 4099), (33, 130), (3, 5000), (257, 64)])
@pytest.mark.parametrize("kind", [np.int32, np.int8, np.uint8])
@pytest.mark.parametrize("offset", [0, 128, -3])
def test_rows_of_integers(pkg, T, rows, width, kind, offset):
    rng = np.random.default_rng(rows * width)
    info = np.iinfo(kind)
    a = rng.integers(info.min, info.max, (rows, width), endpoint=True).astype(kind)
    a.reshape(-1)[0] = info.min
    scales, columns = (rng.normal(size=n).astype(np.float32) for n in (rows, width))
    first = (a.astype(np.int64) - offset).astype(np.float32) * scales[:, None]  # each product rounded to float32
    assert np.array_equal(T.n(pkg.dequantize_rows(T.t(a), T.t(scales), offset)), first)
    assert np.array_equal(T.n(pkg.dequantize_rows(T.t(a), T.t(scales), offset, T.t(columns))), first * columns)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1, 64, 96), (5, 300, 1003), (200, 768, 768)])
def test_norm_product_and_back(pkg, T, m, n, k):
    """The norm's integers and sums are what the integer product takes."""
    rng = np.random.default_rng(m)
    x, r = (rng.normal(size=(m, k)).astype(np.float32) for _ in range(2))
    w = (rng.random(k) + 0.5).astype(np.float32)
    b, columns = rng.integers(-127, 128, (k, n), dtype=np.int8), (rng.random(n) * 0.01).astype(np.float32)
    steps, scales, sums, _ = pkg.rms_norm_quantized(T.t(x), T.t(w), 1e-6, residual=T.t(r))
    product = pkg.quantization_matmul_offsets(steps, sums, T.t(b), pkg.reduce_sum(T.t(b), False), -128, 0)
    got = T.n(pkg.dequantize_rows(product, scales, column_scales=T.t(columns)))
    whole = (T.n(steps).astype(np.int64) - 128) @ b.astype(np.int64)
    assert np.array_equal(T.n(product), whole) and np.array_equal(T.n(sums), T.n(pkg.reduce_sum(steps, True)))
    assert np.array_equal(got, whole.astype(np.float32) * T.n(scales)[:, None] * columns)
    # against the product in 64 bits: half a step of the row for each term
    _, y, _, _ = R.norm(x, w, np.float64(np.float32(1e-6)), r)
    want = y @ (b * columns.astype(np.float64))
    assert (np.abs(got - want) <= 0.5001 * T.n(scales)[:, None] * np.abs(b * columns.astype(np.float64)).sum(0) + 4 * EPS * np.abs(want)).all()


@pytest.mark.gpu
def test_captured_and_on_other_streams(pkg, T):
    import torch
    rng = np.random.default_rng(5)
    x, r, w = (T.t(rng.normal(size=s).astype(np.float32)) for s in ((9, 2000), (9, 2000), (2000,)))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        pkg.rms_norm_quantized(x, w, 1e-6, residual=r)
        with torch.cuda.graph(graph, stream=stream):
            steps, scales, sums, held = pkg.rms_norm_quantized(x, w, 1e-6, residual=r)
            back = pkg.dequantize_rows(steps, scales, 128)
            out, _ = pkg.rms_norm(held, w, 1e-6)
    for seed in range(4):
        x.copy_(T.t(np.random.default_rng(seed).normal(size=(9, 2000)).astype(np.float32)))
        graph.replay()
        torch.cuda.synchronize()
        want = pkg.rms_norm_quantized(x, w, 1e-6, residual=r)
        assert all(torch.equal(a, b) for a, b in zip((steps, scales, sums, held), want))
        assert torch.equal(back, pkg.dequantize_rows(want[0], want[1], 128)) and torch.equal(out, pkg.rms_norm(want[3], w, 1e-6)[0])


@pytest.mark.gpu
def test_refused(pkg, T):
    import torch
    x, w = torch.zeros((4, 8), device="cuda"), torch.ones(8, device="cuda")
    for args, kw in (((x.half(), w, 1e-6), {}), ((x, w[:7], 1e-6), {}), ((x, w.double(), 1e-6), {}), ((x, w, -1.0), {}), ((x, w, float("nan")), {}),
                     ((x, w, 1e-6), {"residual": x[:3]}), ((x, w, 1e-6), {"residual": x.double()}), ((x[:, :0], w[:0], 1e-6), {}), ((x[0, 0], w, 1e-6), {}),
                     ((x.cpu(), w, 1e-6), {}), ((x, w.cpu(), 1e-6), {}), ((x, w, 1e-6), {"residual": x.cpu()})):
        for call in (pkg.rms_norm, pkg.rms_norm_quantized):
            with pytest.raises(pkg.InvalidArgumentError):
                call(*args, **kw)
    a, s = torch.zeros((4, 8), dtype=torch.int32, device="cuda"), torch.ones(4, device="cuda")
    for args in ((x, s), (a.short(), s), (a, s[:3]), (a, s.double()), (a, s, 0, w[:7]), (a, s, 1 << 31), (a, s, 0, w.double()), (a.cpu(), s), (a, s.cpu()), (a[0, 0], s)):
        with pytest.raises(pkg.InvalidArgumentError):
            pkg.dequantize_rows(*args)
