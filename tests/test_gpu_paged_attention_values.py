"""Attention over a paged cache with queries, keys and values of all sizes, the same throughout a row: float32 accuracy over a float32 cache and over an
int8 one with scales from 2^-100 to 2^96."""
import numpy as np
import pytest

import generation_reference as R
from conftest import rel_fro
from test_gpu_paged_attention import Made

SHAPES = [
    # lengths, chunks, heads, kv heads, size, page
    ([300, 45], [2, 45], 4, 2, 128, 16),
    ([300, 45], [2, 45], 4, 2, 64, 7),
    ([3000], [1], 4, 2, 64, 16),
    ([300, 270], [258, 260], 64, 32, 64, 16),   # tiles of 128 rows
    ([300, 290], [300, 290], 32, 16, 128, 20),  # float32: of 256, int8: of 16
    ([3000], [300], 32, 16, 128, 16),           # pieces
]
SIZES = [
    # values, keys, queries
    (1e-26, 1, 1), (1e-28, 1, 1), (2e-30, 1, 1), (2e23, 1, 1), (1e26, 1, 1), (1e29, 1, 1),
    (1, 1e-29, 1e29), (1, 1e29, 1e-29), (1e-28, 1e-29, 1e29), (1, 2e23, 5e-24),
]


def largest_products(m):
    """[tokens, heads, 1] of the largest weight times 127 scales of its value, and how many keys are seen."""
    v = m.cache[3].astype(np.float64) * 127
    k = R.held(m.cache)[0]
    heads, group = k.shape[1], m.q.shape[1] // k.shape[1]
    most, seen_of = np.zeros(m.q.shape[:2] + (1,)), np.zeros((m.q.shape[0], 1, 1))
    for i, length in enumerate(m.lengths):
        at, rows = np.arange(length), slice(m.starts[i], m.starts[i + 1])
        n = rows.stop - rows.start
        seen = at <= (length - n + np.arange(n))[:, None]
        seen_of[rows] = seen.sum(-1)[:, None, None]
        page, inside = m.table[i][at // m.page], at % m.page
        for h in range(m.q.shape[1]):
            s = np.where(seen, m.q[rows, h].astype(np.float64) @ k[page, h // group, inside].T * m.scale, -np.inf)
            p = np.exp(s - s.max(-1, keepdims=True))
            most[rows, h, 0] = (p / p.sum(-1, keepdims=True) * v[page, h // group, inside]).max(-1)
    assert heads * group == m.q.shape[1]
    return most, seen_of


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["s8", "f32"])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
@pytest.mark.parametrize("values,keys,queries", SIZES)
def test_one_size_throughout(pkg, T, kind, shape, values, keys, queries):
    m = Made(pkg, kind, *SHAPES[shape], 31 + shape)
    of = (lambda c: m.cache[c]) if kind == "f32" else (lambda c: m.cache[c + 2])
    of(0)[:] *= np.float32(keys)
    of(1)[:] *= np.float32(values * (1 if kind == "f32" else 40))  # int8: scales of 8e-31 and more, above 2^-100
    m.q *= np.float32(queries)
    got = T.n(m.run(T)).astype(np.float64)
    want, off = R.attention(m.q, m.cache, m.table, m.starts, m.lengths, m.scale)
    if kind == "s8" and values < 2.0 ** -80:
        # the frame takes scales for 2^-90 at least: a row's largest weight times scale lies at 2^-2 or above, and the pieces of such a product leave 2^-25,
        # 2^-23 of the largest for each key
        most, seen = largest_products(m)
        off = off + seen * 2.0 ** -23 * most
    assert (np.abs(got - want) <= off).all(), (np.abs(got - want) / off).max()
    assert rel_fro(got / values, want / values) <= 3e-6


@pytest.mark.gpu
@pytest.mark.parametrize("shape", range(len(SHAPES)))
@pytest.mark.parametrize("values,keys,queries", [(1e32, 1, 1), (1e34, 1, 1), (1, 1e32, 1e-32), (1, 1e34, 1e-30)])
def test_float32_above_the_range(pkg, T, shape, values, keys, queries):
    """Beyond 2^80 nothing is lost as long as sums of weights times values and of products stay below infinity."""
    m = Made(pkg, "f32", *SHAPES[shape], 51 + shape)
    m.cache[0] *= np.float32(keys)
    m.cache[1] *= np.float32(values)
    m.q *= np.float32(queries)
    got = T.n(m.run(T)).astype(np.float64)
    want, off = R.attention(m.q, m.cache, m.table, m.starts, m.lengths, m.scale)
    assert (np.abs(got - want) <= off).all(), (np.abs(got - want) / off).max()
    if keys * queries <= 1:  # scores of 2^14 are multiples of 2^-9 in float32: weights are off by 2^-10 of themselves, whoever works them out
        assert rel_fro(got / values, want / values) <= 3e-6


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [3, 4, 5])
def test_one_large_row_among_others(pkg, T, shape):
    """A value row of 10^33, a key of 10^33 that queries of ordinary size make the only one that counts or the one that never does: rows that do not
    see it keep every bit."""
    m = Made(pkg, "f32", *SHAPES[shape], 61)
    clean = T.n(m.run(T)).copy()
    length, chunk = m.lengths[0], m.starts[1]
    at = length - chunk // 2
    page, inside = m.table[0, at // m.page], at % m.page
    later = np.zeros(len(m.q), bool)
    later[:chunk] = np.arange(length - chunk, length) >= at
    group = m.q.shape[1] // m.cache[0].shape[1]
    mine = np.zeros(clean.shape, bool)
    mine[:, group:2 * group] = later[:, None, None]
    for c in (1, 0):
        before = m.cache[c][page, 1, inside].copy()
        m.cache[c][page, 1, inside] *= np.float32(1e33)
        got = T.n(m.run(T))
        assert np.array_equal(got[~mine], clean[~mine])
        want, off = R.attention(m.q, m.cache, m.table, m.starts, m.lengths, m.scale)
        if c == 0:  # scores of 10^33: one key is all there is, exactly, or is not there
            off = 60 * R.EPS * np.abs(want) + (length + 60) * R.EPS * 8
        assert (np.abs(got - want) <= off)[mine].all()
        m.cache[c][page, 1, inside] = before


# float32, tiles of 128 and 256 rows; rows, windows and pages that end inside a step of 16 keys
FAR = [
    ([300, 270], [258, 260], 64, 32, 64, 16, {}),
    ([310, 270], [258, 260], 64, 32, 40, 20, {"window": 70}),
    ([300, 290], [300, 290], 32, 16, 128, 20, {"window": 100}),
    ([500, 333], [300, 290], 48, 16, 96, 24, {"causal": False}),
    ([3000, 300], [200, 111], 32, 8, 128, 20, {}),          # pieces
    ([2700, 2100], [300, 260], 32, 32, 64, 28, {"window": 2300}),
    ([400, 200, 90], [260, 280, 90], 48, 48, 96, 16, {}),   # more tokens than are cached
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(FAR)))
@pytest.mark.parametrize("value", [np.inf, np.nan, 1e30, -3e38])
def test_far_numbers_here_and_there(pkg, T, case, value):
    """Some value rows and keys with an infinity, a NaN or a number beyond 2^80, pages that are nowhere: rows that see one are those of the definition, all
    others keep every bit."""
    lengths, chunks, heads, kv, size, page, more = FAR[case]
    m = Made(pkg, "f32", lengths, chunks, heads, kv, size, page, 71 + case)
    m.table[0, 2] = -1
    m.table[0, -2] = len(m.cache[0])
    clean = T.n(m.run(T, **more)).copy()
    group = heads // kv
    mine = np.zeros(clean.shape, bool)
    for i, (at, head) in enumerate([(lengths[0] // 2, 1), (lengths[0] - 2, 0), (lengths[1] - 70, 1), (lengths[1] // 2 + 3, kv - 1), (lengths[0] // 3, kv - 1)]):
        sequence = 1 if i in (2, 3) else 0
        named, inside = m.table[sequence, at // page], at % page
        if not 0 <= named < len(m.cache[0]):
            continue
        # a key takes part as a zero times that number: nothing of it is in a score, but it is there
        c = 0 if i == 1 and np.isfinite(value) else 1
        m.cache[c][named, head, inside, 5] = value
        if c == 0:
            m.q[:, :, 5] = 0
            clean = None
        n = chunks[sequence]
        position = lengths[sequence] - n + np.arange(n)
        sees = (at <= position) & (at > position - more.get("window", 10 ** 9)) if more.get("causal", True) else np.ones(n, bool)
        mine[m.starts[sequence]:m.starts[sequence + 1], head * group:(head + 1) * group] |= sees[:, None, None]
    got = T.n(m.run(T, **more)).astype(np.float64)
    if clean is not None:
        assert np.array_equal(got[~mine], clean[~mine])
    want, off = R.attention(m.q, m.cache, m.table, m.starts, m.lengths, m.scale, **more)
    off = np.where(np.isfinite(want), off, 0)
    same = (got == want) | (np.isnan(got) & np.isnan(want))
    with np.errstate(invalid="ignore"):
        near = np.abs(got - want) <= off
    # a weight below 2^-149 times infinity is NaN in float32 and infinity in 64 bits
    lost = np.isinf(want) & np.isnan(got)
    assert (same | near | lost).all() and not lost.all()
    assert mine.any()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [3, 4, 5])
def test_far_numbers_between_replays(pkg, T, shape):
    """A captured call meets infinities that come and go in its cache."""
    import torch
    m = Made(pkg, "f32", *SHAPES[shape], 91)
    cache, q, table, starts, lengths = m.on(T), T.t(m.q), T.t(m.table), T.t(m.starts), T.t(m.lengths)
    call = lambda: pkg.paged_attention(q, cache, table, starts, lengths, m.scale)
    clean = call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    at = int(m.lengths[0]) // 2
    named, inside = m.table[0, at // m.page], at % m.page
    for value in (None, float("inf"), None, 1e33, float("nan"), None):
        held = cache[1][named, 0, inside, 3].item()
        if value is not None:
            cache[1][named, 0, inside, 3] = value
        eager = call()
        for _ in range(2):
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out.isnan(), eager.isnan()) and torch.equal(out.nan_to_num(0.0), eager.nan_to_num(0.0))
        assert torch.equal(eager.nan_to_num(0.0), clean.nan_to_num(0.0)) == (value is None)
        cache[1][named, 0, inside, 3] = held


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["s8", "f32"])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
@pytest.mark.parametrize("scale", [-0.125, 0.0, -0.0])
def test_scales_of_scores_below_and_at_zero(pkg, T, kind, shape, scale):
    m = Made(pkg, kind, *SHAPES[shape], 93 + shape)
    m.scale = scale
    m.check(T)
