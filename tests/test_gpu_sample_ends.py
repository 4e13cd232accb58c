"""Sampling where a temperature is far below the distance of one float to the next, so that only the largest logits have weights."""
import numpy as np
import pytest

from test_gpu_sample import check


@pytest.mark.gpu
@pytest.mark.parametrize("filters", [(), ("top_p",), ("top_k",), ("min_p",), ("top_k", "top_p", "min_p")])
@pytest.mark.parametrize("top", [100.0, 1.0, -3.0, 1e-30, -1e30])
def test_temperatures_below_a_float_of_the_top(pkg, T, filters, top):
    """All logits but the largest, the next float below it and below that among them, have weights of 0."""
    rng = np.random.default_rng(21)
    rows, length = 64, 300
    top = np.float32(top)
    below = np.nextafter(top, np.float32(-np.inf))
    step = float(top) - float(below)
    logits = (float(top) - np.abs(rng.normal(size=(rows, length))) * abs(float(top)) - step).astype(np.float32)
    logits[:, [7, 100, 250]] = [below, top, np.nextafter(below, np.float32(-np.inf))]
    # the next float below lies 2^6 to 2^52 e-foldings down and beyond, in steps that hit every remainder of 2^32 / 32
    temperature = (step / 2.0 ** np.linspace(6, 52, rows)).astype(np.float32)
    if top == 100:
        temperature[0] = np.float32(8.20077174e-14)
    keep = temperature > 0
    kw = dict(temperature=temperature, top_k=np.full(rows, 40, np.int32), top_p=np.full(rows, 0.9, np.float32), min_p=np.full(rows, 1e-3, np.float32))
    kw = {k: v[keep] for k, v in kw.items() if k == "temperature" or k in filters}
    got = check(pkg, T, logits[keep], np.full(int(keep.sum()), 0.05, np.float32), **kw)
    assert (got == 100).all()


@pytest.mark.gpu
@pytest.mark.parametrize("filters", [(), ("top_p",), ("top_k",), ("min_p",)])
def test_infinite_logits_at_all_temperatures(pkg, T, filters):
    """Those of +infinity share the weight, whatever the temperature is."""
    rng = np.random.default_rng(22)
    rows, length = 40, 2000
    logits = rng.normal(size=(rows, length)).astype(np.float32)
    logits[:, [11, 1500]] = np.inf
    temperature = np.resize(np.array([1e-45, 1e-30, 1.0, 3e38, np.inf], np.float32), rows)
    kw = dict(top_k=np.full(rows, 30, np.int32), top_p=np.full(rows, 0.99, np.float32), min_p=np.full(rows, 0.5, np.float32))
    got, odds = pkg.sample(T.t(logits), T.t(np.linspace(0, 0.999, rows, dtype=np.float32)), temperature=T.t(temperature), **{k: T.t(kw[k]) for k in filters})
    assert np.array_equal(T.n(got), np.where(np.arange(rows) < rows / 2, 11, 1500)) and (T.n(odds) == 0.5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("least", [1e-3, 1e-7, 1e-12, 1e-30, 1e-44])
@pytest.mark.parametrize("size", [1.0, 100.0, 1e30, 1e-30])
def test_small_least_weights(pkg, T, least, size):
    """How near a row comes to another choice is measured against the least weight itself, so that rows are compared however small that is."""
    rng = np.random.default_rng(23)
    rows, length = 12, 5003
    least = np.float32(least)
    logits = (rng.normal(size=(rows, length)) * size * 3).astype(np.float32)
    temperature = (np.linspace(0.05, 3.0, rows) * size).astype(np.float32)
    random = rng.random(rows).astype(np.float32)
    got, odds = (T.n(t) for t in pkg.sample(T.t(logits), T.t(random), temperature=T.t(temperature), min_p=T.t(np.full(rows, least))))
    compared = 0
    for r in range(rows):
        x = logits[r].astype(np.float64)
        w = np.exp((x - x.max()) / float(temperature[r]))
        kept = np.where(w >= float(least), w, 0)
        sums = kept.cumsum()
        goal = float(random[r]) * sums[-1]
        # weights in 64 bits are off by 2^-48 and less; sums of integers of 2^-51 of the largest by 5003 halves of those
        if (np.abs(w - float(least)) < 1e-10 * float(least)).any() or (np.abs(sums - goal) < 1e-9 * sums[-1]).any():
            continue
        compared += 1
        at = int((sums <= goal).sum())
        assert got[r] == at and abs(odds[r] - kept[at] / sums[-1]) <= 2.0 ** -23 * kept[at] / sums[-1]
    assert compared >= rows - 1
