"""Rotary positions against the definition in 64 bits: layouts, parts of heads, odd sizes, strides, far positions, in place."""
import math

import numpy as np
import pytest

import generation_reference as R


def off(size):
    """The cosine's argument, half a turn at most, is rounded to float32 (2 pi 2^-26 < 0.79 * 2^-23), sine and cosine are within two
    units of the last place (2^-23), the magnitude, the products and their sum round once each (2^-24 of |a| + |b|)."""
    return (0.79 + 1.0 + 1.5) * 2.0 ** -23 * size + 1e-37


def test_frequencies(pkg):
    plain, magnitude = pkg.rotary_frequencies(64, base=10000.0)
    want = 10000.0 ** (-np.arange(32) / 32.0)
    assert magnitude == 1.0 and np.allclose(plain, want, rtol=1e-14)
    assert np.allclose(pkg.rotary_frequencies(64, scaling="linear", factor=4.0)[0], want / 4, rtol=1e-14)
    f = pkg.rotary_frequencies(64, scaling="base", factor=8.0)[0]
    assert f[0] == 1.0 and math.isclose(f[-1], want[-1] / 8, rel_tol=1e-12)
    turns = 8192 * want / (2 * math.pi)
    r = np.clip((turns - 1) / 3, 0, 1)
    f = pkg.rotary_frequencies(64, scaling="turns", factor=8.0, original_length=8192, low=1, high=4)[0]
    assert np.allclose(f, want * (r + (1 - r) / 8), rtol=1e-13) and f[0] == 1.0 and math.isclose(f[-1], want[-1] / 8, rel_tol=1e-13)
    f, magnitude = pkg.rotary_frequencies(64, scaling="index", factor=8.0, original_length=4096, low=1, high=32)
    place = lambda n: 64 * math.log(4096 / (n * 2 * math.pi)) / (2 * math.log(10000.0))
    ramp = np.clip((np.arange(32) - math.floor(place(32))) / (math.ceil(place(1)) - math.floor(place(32))), 0, 1)
    assert np.allclose(f, want * (1 - ramp) + want / 8 * ramp, rtol=1e-13)
    assert math.isclose(magnitude, 0.1 * math.log(8.0) + 1, rel_tol=1e-7)


@pytest.mark.parametrize("kw", [dict(part=7), dict(part=0), dict(part=2048), dict(base=0.0), dict(base=math.inf), dict(scaling="linear", factor=0.0),
                                dict(scaling="turns", factor=2.0), dict(scaling="index", factor=2.0, original_length=10, low=4, high=4),
                                dict(scaling="base", part=2, factor=2.0), dict(scaling="steps"),
                                dict(scaling="index", base=1.0, factor=2.0, original_length=64)])
def test_frequencies_refused(pkg, kw):
    with pytest.raises(pkg.InvalidArgumentError):
        pkg.rotary_frequencies(**{"part": 64, **kw})


def test_refused_without_a_device(pkg):
    import ctypes as C
    lib, d = pkg.lib(), pkg.RotaryDesc()
    call = lambda: lib.tfcc_rocm_rotary_f32(None, C.byref(d))
    assert lib.tfcc_rocm_rotary_f32(None, None) == 1
    d.size, d.part, d.tokens, d.position_type = 64, 64, 1, pkg.S32
    d.heads[0] = 1
    assert call() == 1 and b"null" in lib.tfcc_rocm_last_error_string()
    d.in_[0] = d.out[0] = d.positions = d.frequencies = 4096
    for name, value in (("size", 0), ("size", 1025), ("part", 66), ("part", 3), ("part", 0), ("position_type", pkg.F32), ("tokens", 1 << 31)):
        before = getattr(d, name)
        setattr(d, name, value)
        assert call() == 1, (name, value)
        setattr(d, name, before)
    d.heads[0] = 0
    assert call() == 1
    d.heads[0] = 1
    d.out_head_stride[0] = 5  # in place with other strides
    assert call() == 1
    d.out_head_stride[0] = 0
    d.out[1] = 4096
    assert call() == 1
    d.out[1] = None
    d.tokens = 0
    assert call() == 0  # nothing to do


CASES = [
    # tokens, heads, kv heads, size, part, interleaved, positions up to
    (1, 1, 1, 2, 2, False, 10),
    (1, 32, 8, 128, 128, False, 4096),
    (3, 5, 0, 64, 64, True, 100),
    (7, 12, 12, 64, 32, True, 2048),
    (5, 3, 2, 80, 20, False, 1000),    # halves of ten values: one at a time
    (5, 3, 2, 77, 18, True, 1000),     # an odd head
    (5, 3, 2, 77, 18, False, 1000),
    (600, 4, 1, 96, 96, False, 1 << 20),
    (2, 2, 2, 1024, 1024, True, 2 ** 31 - 1),
    (1030, 20, 5, 80, 80, False, 131072),
]


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,heads,kv,size,part,interleaved,far", CASES)
def test_against_the_definition(pkg, T, tokens, heads, kv, size, part, interleaved, far):
    import torch
    rng = np.random.default_rng(tokens + size)
    q = rng.normal(size=(tokens, heads, size)).astype(np.float32)
    k = rng.normal(size=(tokens, kv, size)).astype(np.float32) if kv else None
    positions = rng.integers(0, far, tokens, endpoint=True)
    positions[0] = far
    f, _ = pkg.rotary_frequencies(part)
    tf = torch.tensor(f, dtype=torch.float64, device="cuda")
    for dtype in (np.int32, np.int64):
        if far > 2 ** 31 - 1 and dtype == np.int32:
            continue
        got = pkg.rotary(T.t(q), None if k is None else T.t(k), T.t(positions.astype(dtype)), tf, interleaved=interleaved, magnitude=1.25)
        for g, x in zip(got, (q, k)):
            if x is None:
                assert g is None
                continue
            want, size_of = R.rotary(x, positions, f, interleaved, 1.25)
            g = T.n(g).astype(np.float64)
            assert np.array_equal(g[..., part:], want[..., part:])
            assert (np.abs(g - want) <= off(size_of)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_strides_and_in_place(pkg, T, interleaved):
    import torch
    rng = np.random.default_rng(5)
    qkv = rng.normal(size=(9, 12 * 64 + 5)).astype(np.float32)
    positions = np.arange(9, dtype=np.int32) * 1000 - 4000  # negative ones among them
    f, _ = pkg.rotary_frequencies(48)
    tf, tp = torch.tensor(f, dtype=torch.float64, device="cuda"), T.t(positions)
    whole = T.t(qkv)
    q, k = (whole[:, i * 256 + 1:(i + 1) * 256 + 1].unflatten(1, (4, 64)) for i in (0, 1))  # off by one float, odd row stride
    wq, sq = R.rotary(qkv[:, 1:257].reshape(9, 4, 64), positions, f, interleaved)
    wk, sk = R.rotary(qkv[:, 257:513].reshape(9, 4, 64), positions, f, interleaved)
    oq, ok = pkg.rotary(q, k, tp, tf, interleaved=interleaved)
    assert (np.abs(T.n(oq) - wq) <= off(sq)).all() and (np.abs(T.n(ok) - wk) <= off(sk)).all()
    back = pkg.rotary(q, k, tp, tf, interleaved=interleaved, out=(q, k))
    assert back[0] is q and torch.equal(q, oq) and torch.equal(k, ok)
    want = qkv.copy()
    want[:, 1:257], want[:, 257:513] = T.n(oq).reshape(9, 256), T.n(ok).reshape(9, 256)
    assert np.array_equal(T.n(whole), want)  # nothing beside them
    assert torch.equal(pkg.rotary(q.transpose(0, 2).contiguous().transpose(0, 2), None, tp, tf)[0], pkg.rotary(q.contiguous(), None, tp, tf)[0])


@pytest.mark.gpu
def test_empty_and_refused(pkg, T):
    import torch
    f = torch.tensor(pkg.rotary_frequencies(16)[0], dtype=torch.float64, device="cuda")
    q, p = torch.zeros((3, 2, 16), device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    out, none = pkg.rotary(q[:0], None, p[:0], f)
    assert out.shape == (0, 2, 16) and none is None
    for args in ((q.double(), None, p, f), (q, q[:2], p, f), (q, None, p[:2], f), (q, None, p.float(), f), (q, None, p, f.float()),
                 (q[..., :8], None, p, f), (q, None, p.cpu(), f), (q[0], None, p, f)):
        with pytest.raises(pkg.InvalidArgumentError):
            pkg.rotary(*args)
    with pytest.raises(pkg.InvalidArgumentError):
        pkg.rotary(q, None, p, f, out=(q[:2], None))
