"""Sampling against the definition in 64 bits: the same token wherever the choice is not nearer to another one than 64-bit sums can
tell, and its probability to float32."""
import ctypes as C

import numpy as np
import pytest

import generation_reference as R


def test_refused_without_a_device(pkg):
    lib, d = pkg.lib(), pkg.SampleDesc()
    call = lambda: lib.tfcc_rocm_sample_f32(None, C.byref(d))
    assert lib.tfcc_rocm_sample_f32(None, None) == 1
    d.rows, d.length = 1, 0
    assert call() == 1
    d.length = (1 << 20) + 1
    assert call() == 1
    d.length = 10
    assert call() == 1 and b"null" in lib.tfcc_rocm_last_error_string()
    d.rows = 0
    assert call() == 0


def check(pkg, T, logits, random, most_near=0.05, **kw):
    got, odds = pkg.sample(T.t(logits), T.t(random), **{k: None if v is None else T.t(v) for k, v in kw.items()})
    got, odds = T.n(got), T.n(odds)
    want, exact, margin = R.sample(logits, random, **kw)
    near = margin < 1e-9
    assert near.mean() <= most_near
    assert np.array_equal(got[~near], want[~near]), (got, want, margin)
    # a weight in 64 bits over a sum of integers of 2^-43 each, rounded to float32 once
    assert (np.abs(odds - exact) <= 2.0 ** -24 * exact + logits.shape[1] * 2.0 ** -43 * exact + 1e-45)[~near].all()
    return got


def f32(*v):
    return np.array(v, np.float32)


def parameters(rng, rows):
    return dict(temperature=(rng.random(rows) * 1.5 + 0.2).astype(np.float32), top_k=rng.integers(1, 60, rows).astype(np.int32),
                top_p=(rng.random(rows) * 0.5 + 0.5).astype(np.float32), min_p=(rng.random(rows) * 0.1).astype(np.float32))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,length", [(1, 1), (3, 2), (5, 63), (4, 64), (4, 65), (7, 1000), (2, 4097), (33, 32000), (3, 100003), (1, 200001), (300, 517)])
@pytest.mark.parametrize("filters", ["", "k", "p", "m", "kp", "kpm", "tkpm"])
def test_against_the_definition(pkg, T, rows, length, filters):
    rng = np.random.default_rng(rows * 7 + length)
    logits = (rng.normal(size=(rows, length)) * 3).astype(np.float32)
    p = parameters(rng, rows)
    kw = {name: p[name] if key in filters else None for name, key in (("temperature", "t"), ("top_k", "k"), ("top_p", "p"), ("min_p", "m"))}
    check(pkg, T, logits, rng.random(rows).astype(np.float32), **kw)


@pytest.mark.gpu
def test_ends_of_the_parameters(pkg, T):
    rng = np.random.default_rng(2)
    logits = (rng.normal(size=(12, 777)) * 2).astype(np.float32)
    u = rng.random(12).astype(np.float32)
    for kw in (dict(temperature=np.zeros(12, np.float32)), dict(temperature=np.full(12, -1, np.float32)), dict(temperature=np.full(12, 1e-30, np.float32)),
               dict(temperature=np.full(12, 1e30, np.float32)), dict(top_k=np.zeros(12, np.int32)), dict(top_k=np.full(12, -3, np.int32)),
               dict(top_k=np.full(12, 777, np.int32)), dict(top_k=np.full(12, 10 ** 9, np.int32)), dict(top_k=np.ones(12, np.int32)),
               dict(top_p=np.zeros(12, np.float32)), dict(top_p=np.full(12, -1, np.float32)), dict(top_p=np.ones(12, np.float32)),
               dict(top_p=np.full(12, 1e-9, np.float32)), dict(top_p=np.full(12, 0.99999994, np.float32)), dict(min_p=np.ones(12, np.float32)),
               dict(min_p=np.full(12, 2, np.float32)), dict(min_p=np.full(12, -1, np.float32)), dict(min_p=np.full(12, 1e-30, np.float32))):
        check(pkg, T, logits, u, **kw)
    check(pkg, T, logits, np.zeros(12, np.float32))
    check(pkg, T, logits, np.full(12, 0.99999994, np.float32))
    check(pkg, T, logits, np.ones(12, np.float32))  # outside the interval: the last token


@pytest.mark.gpu
@pytest.mark.parametrize("length", [100, 5000, 70001])
def test_equal_logits(pkg, T, length):
    """Ties are taken in the order of their positions, among a few values and all over."""
    rng = np.random.default_rng(length)
    logits = rng.integers(-2, 3, (20, length)).astype(np.float32)
    logits[:5] = 1.0
    logits[5, ::2], logits[5, 1::2] = 0.0, -0.0  # one and the same
    logits[6] = -1e30
    u = rng.random(20).astype(np.float32)
    p = parameters(rng, 20)
    p["top_k"] = rng.integers(1, length, 20).astype(np.int32)
    check(pkg, T, logits, u, top_k=p["top_k"])
    check(pkg, T, logits, u, top_p=p["top_p"])
    check(pkg, T, logits, u, min_p=p["min_p"])
    check(pkg, T, logits, u, **p)


@pytest.mark.gpu
@pytest.mark.parametrize("length", [10, 3000, 60001])
def test_logits_that_are_no_numbers(pkg, T, length):
    rng = np.random.default_rng(length)
    logits = (rng.normal(size=(10, length)) * 3).astype(np.float32)
    logits[0] = -np.inf
    logits[1] = np.nan
    logits[2, :] = -np.inf
    logits[2, length // 2] = -3e38
    logits[3, ::2] = np.nan
    logits[4, 1::3] = -np.inf
    logits[5, [1, length - 2]] = np.inf
    logits[6] = np.finfo(np.float32).min
    logits[7, 3:] = np.finfo(np.float32).min
    logits[8, :-1], logits[8, -1] = -np.inf, np.nan
    u = rng.random(10).astype(np.float32)
    p = parameters(rng, 10)
    got = check(pkg, T, logits, u)
    assert got[0] == got[1] == got[8] == -1 and got[2] == length // 2 and got[5] in (1, length - 2)
    check(pkg, T, logits, u, **p)
    check(pkg, T, logits, u, top_k=np.full(10, 7, np.int32), temperature=np.zeros(10, np.float32))


@pytest.mark.gpu
def test_far_tails(pkg, T):
    """A likely token among a million unlikely ones: the sum of their weights counts."""
    rng = np.random.default_rng(4)
    logits = rng.normal(size=(6, 1 << 20)).astype(np.float32)
    logits[:, 12345] = [10, 14, 18, 25, 40, 100]
    check(pkg, T, logits, rng.random(6).astype(np.float32))
    check(pkg, T, logits, rng.random(6).astype(np.float32), top_p=np.full(6, 0.95, np.float32))


@pytest.mark.gpu
def test_every_share_of_the_interval(pkg, T):
    """Random numbers all over [0, 1) choose tokens in proportion to their weights."""
    import torch
    p = np.array([0.05, 0.0, 0.25, 0.1, 0.6])
    with np.errstate(divide="ignore"):
        logits = np.log(p).astype(np.float32)
    u = (np.arange(2000) + 0.5) / 2000
    got, _ = pkg.sample(T.t(np.tile(logits, (2000, 1))), T.t(u.astype(np.float32)))
    assert np.abs(np.bincount(T.n(got), minlength=5) / 2000 - p).max() <= 1 / 2000


@pytest.mark.gpu
def test_strides_and_refusals(pkg, T):
    import torch
    rng = np.random.default_rng(5)
    wide = T.t(rng.normal(size=(6, 1003)).astype(np.float32))
    u = T.t(rng.random(6).astype(np.float32))
    assert torch.equal(pkg.sample(wide[:, 1:1001], u)[0], pkg.sample(wide[:, 1:1001].contiguous(), u)[0])
    assert torch.equal(pkg.sample(wide.t().contiguous().t(), u)[0], pkg.sample(wide, u)[0])
    assert pkg.sample(wide[:0], u[:0])[0].shape == (0,)
    for args, kw in (((wide[0], u), {}), ((wide.double(), u), {}), ((wide, u[:5]), {}), ((wide, None), {}), ((wide, u), dict(top_k=u)),
                     ((wide, u), dict(top_p=u.double())), ((wide, u.cpu()), {}), ((wide[:, :0], u), {})):
        with pytest.raises(pkg.InvalidArgumentError):
            pkg.sample(*args, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("size,offset", [(1.0, 0.0), (1e-3, 1e4), (100.0, -1e6), (1e4, 1e8), (1e30, 1e37), (1e-30, 0.0)])
@pytest.mark.parametrize("least", [1.0, 0.5, 1e-3, 1e-30])
def test_least_weights_at_all_sizes(pkg, T, size, offset, least):
    """Logits far from zero, close together and far apart, with temperatures that fit them and others that do not."""
    rng = np.random.default_rng(12)
    logits = (rng.normal(size=(6, 5003)) * size + offset).astype(np.float32)
    temperature = (np.array([1.0, 0.3, 3.0, 1e-3, 1e3, 1e6]) * size).astype(np.float32)
    # margins are in units of the largest weight: where the least kept one is below 1e-9 of it, every row with a weight that small is called near
    near = 1.0 if least < 1e-9 else 0.05
    for top_p in (None, np.full(6, 0.97, np.float32)):
        check(pkg, T, logits, rng.random(6).astype(np.float32), near, temperature=temperature, min_p=np.full(6, least, np.float32), top_p=top_p)
