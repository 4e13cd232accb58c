"""Attention over a paged cache against the definition in 64 bits, within what float32 sums may be off by."""
import ctypes as C

import numpy as np
import pytest

import generation_reference as R
from conftest import rel_fro


def test_refused_without_a_device(pkg):
    lib, d = pkg.lib(), pkg.PagedAttentionDesc()
    call = lambda: lib.tfcc_rocm_paged_attention_f32(None, C.byref(d))
    size = lambda: lib.tfcc_rocm_paged_attention_workspace(C.byref(d))
    assert lib.tfcc_rocm_paged_attention_f32(None, None) == 1 and lib.tfcc_rocm_paged_attention_workspace(None) == 0
    c = d.cache
    c.keys = c.values = c.key_scales = c.value_scales = 4096
    c.type, c.pages, c.heads, c.page_size, c.size = pkg.S8, 200, 2, 16, 64
    d.heads, d.tokens, d.batch, d.table_width, d.causal = 8, 1, 1, 200, 1
    assert call() == 1 and b"null" in lib.tfcc_rocm_last_error_string()
    d.q = d.out = d.starts = d.lengths = d.table = 4096
    needs = size()
    assert needs > 0 and call() == 1 and b"workspace" in lib.tfcc_rocm_last_error_string()
    d.workspace, d.workspace_bytes = 4096, needs - 1
    assert call() == 1
    d.workspace, d.workspace_bytes = 4097, needs
    assert call() == 1
    d.workspace = 4096
    for name, value in (("heads", 0), ("heads", 7), ("tokens", 1 << 31), ("q", 4100), ("out", 4104), ("q_token_stride", 6), ("out_head_stride", 5),
                        ("table_width", 1 << 30)):
        before = getattr(d, name)
        setattr(d, name, value)
        assert call() == 1 and size() == 0, (name, value)
        setattr(d, name, before)
    d.causal, d.window = 0, 5
    assert call() == 1 and size() == 0
    d.window, d.tokens = 0, 0
    assert call() == 0 and size() == 0


class Made:
    """A cache with the pages of its sequences mixed up, and a chunk of queries for each."""

    def __init__(self, pkg, kind, lengths, chunks, heads, kv, size, page, seed, spare=2):
        import torch
        rng = self.rng = np.random.default_rng(seed)
        each = [max(1, -(-n // page)) for n in lengths]
        pages = sum(each) + spare
        order = rng.permutation(pages).astype(np.int32)
        self.table = rng.integers(-5, pages + 5, (len(lengths), max(each) + 1)).astype(np.int32)  # what lies behind is anything
        at = 0
        for i, n in enumerate(each):
            self.table[i, :n] = order[at:at + n]
            at += n
        shape = (pages, kv, page, size)
        if kind == "s8":
            self.cache = [rng.integers(-127, 128, shape, dtype=np.int8) for _ in range(2)]
            self.cache += [(rng.random(shape[:3]) * 0.02 + 0.01).astype(np.float32) for _ in range(2)]
        else:
            self.cache = [rng.normal(size=shape).astype(np.float32) for _ in range(2)]
        self.lengths, self.page = np.array(lengths, np.int32), page
        self.starts = np.concatenate([[0], np.cumsum(chunks)]).astype(np.int32)
        self.q = rng.normal(size=(int(self.starts[-1]), heads, size)).astype(np.float32)
        self.scale = float(size ** -0.5)
        self.pkg = pkg

    def on(self, T):
        return tuple(T.t(c) for c in self.cache)

    def run(self, T, cache=None, out=None, **kw):
        return self.pkg.paged_attention(T.t(self.q), cache or self.on(T), T.t(self.table), T.t(self.starts), T.t(self.lengths), self.scale, out=out, **kw)

    def check(self, T, got=None, cache=None, **kw):
        got = T.n(self.run(T, cache, **kw) if got is None else got).astype(np.float64)
        most = kw.pop("max_length", None)
        want, off = R.attention(self.q, self.cache, self.table, self.starts, self.lengths, self.scale, most=most, **kw)
        assert np.array_equal(np.isnan(got), np.isnan(want))
        fine = ~np.isnan(want)
        same = got == want  # infinities among them
        with np.errstate(invalid="ignore"):
            assert (same | (np.abs(got - want) <= off))[fine].all(), np.nanmax((np.abs(got - want) / off)[fine & ~same])
        finite = np.isfinite(want)
        assert rel_fro(got[finite], want[finite]) <= 1e-5


CASES = [
    # kind, lengths, chunks, heads, kv heads, size, page, more
    ("s8", [1], [1], 1, 1, 64, 16, {}),
    ("f32", [1], [1], 1, 1, 64, 16, {}),
    ("s8", [777], [1], 12, 12, 64, 16, {}),
    ("s8", [33, 0, 200, 1, 517], [1, 1, 1, 1, 1], 8, 2, 128, 32, {}),         # one has nothing cached
    ("f32", [33, 0, 200, 1, 517], [1, 1, 1, 1, 1], 8, 2, 128, 32, {}),
    ("s8", [40, 300, 90], [40, 7, 0], 6, 2, 128, 16, {}),                      # a whole prompt, a chunk, a sequence without one
    ("f32", [40, 300, 90], [40, 7, 0], 6, 2, 64, 16, {}),
    ("s8", [3, 70], [5, 66], 4, 4, 64, 16, {}),                                # more tokens than cached: the first see nothing
    ("f32", [3, 70], [5, 66], 4, 4, 64, 16, {}),
    ("s8", [257, 65], [1, 3], 20, 5, 80, 24, {}),                              # pages that end inside a tile
    ("f32", [257, 65], [1, 3], 20, 5, 80, 24, {}),
    ("s8", [130, 61], [30, 2], 3, 1, 40, 7, {}),                               # rows of 8 bytes, odd pages, groups of three
    ("f32", [130, 61], [30, 2], 3, 1, 36, 7, {}),
    ("s8", [129], [9], 33, 1, 200, 1, {}),                                     # pages of one row, more heads than a tile has rows
    ("f32", [129], [9], 33, 1, 252, 16, {}),
    ("s8", [500, 90], [64, 1], 4, 2, 256, 64, {}),
    ("f32", [500, 90], [64, 1], 4, 2, 192, 64, {}),
    ("s8", [700, 100], [3, 100], 8, 8, 64, 16, {"window": 1}),
    ("f32", [700, 100], [3, 100], 8, 8, 64, 16, {"window": 37}),
    ("s8", [1500, 600], [1, 130], 8, 1, 128, 32, {"window": 300}),
    ("s8", [90, 300], [20, 3], 4, 4, 96, 16, {"causal": False}),
    ("f32", [90, 300], [20, 3], 4, 4, 96, 16, {"causal": False}),
    ("s8", [900, 60], [2, 2], 4, 1, 64, 16, {"max_length": 512}),              # keys behind the bound are not seen
    ("s8", [3000, 1, 2048, 129], [1, 1, 1, 1], 32, 8, 128, 128, {}),           # many pieces
    ("f32", [3000, 1, 2048, 129], [1, 1, 1, 1], 32, 8, 128, 128, {}),
    # chunks of more tokens
    ("s8", [64], [64], 1, 1, 64, 16, {}),
    ("s8", [300, 129, 70], [300, 33, 70], 2, 2, 64, 16, {}),
    ("s8", [1000, 257], [130, 257], 8, 2, 128, 32, {}),
    ("s8", [513, 90], [200, 90], 5, 1, 80, 48, {}),
    ("s8", [200, 40, 0, 77], [100, 60, 0, 77], 4, 4, 96, 16, {}),              # the second has more tokens than are cached
    ("s8", [400, 300], [160, 1], 3, 1, 192, 16, {}),
    ("s8", [333], [333], 2, 1, 144, 16, {}),
    ("s8", [290, 100], [290, 100], 4, 2, 256, 16, {}),
    ("s8", [1500, 600], [200, 600], 2, 2, 64, 32, {"window": 1}),
    ("s8", [1500, 600], [200, 600], 4, 2, 128, 32, {"window": 150}),
    ("s8", [300, 500], [100, 120], 4, 2, 128, 16, {"causal": False}),
    ("s8", [6000], [70], 8, 2, 128, 64, {}),                                   # few tiles of a long context: pieces
    ("s8", [2500, 700], [90, 90], 8, 2, 128, 16, {"max_length": 2100}),
    ("f32", [300, 129, 70], [300, 33, 70], 2, 2, 64, 16, {}),
    ("f32", [513, 90], [200, 90], 5, 1, 80, 48, {"window": 100}),
    ("f32", [1000, 257], [130, 257], 8, 2, 128, 32, {}),
    ("f32", [290, 100], [290, 100], 4, 2, 256, 16, {}),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(CASES)))
def test_against_the_definition(pkg, T, case):
    kind, lengths, chunks, heads, kv, size, page, more = CASES[case]
    Made(pkg, kind, lengths, chunks, heads, kv, size, page, case).check(T, **more)


# Chunks of many tokens; most of them go over the keys together, 128 or 256 rows in a workgroup.
TILES = [
    ([600, 300, 257, 700], [300, 300, 257, 290], 32, 32, 64, 16, {}),
    ([300, 290, 0, 1100, 260, 257], [70, 97, 0, 90, 64, 65], 64, 16, 128, 32, {}),
    ([513, 400], [260, 300], 64, 64, 80, 48, {}),                              # heads that do not fill their tiles
    ([400, 200, 90], [260, 280, 90], 48, 48, 96, 16, {}),                      # more tokens than are cached
    ([400, 300], [260, 270], 64, 64, 192, 16, {}),
    ([290, 280], [290, 270], 64, 64, 144, 16, {}),
    ([290, 300], [290, 258], 64, 64, 256, 16, {}),
    ([700, 600], [300, 290], 64, 64, 64, 32, {"window": 1}),
    ([700, 600], [128, 140], 128, 64, 128, 32, {"window": 150}),
    ([300, 400], [260, 270], 64, 64, 128, 16, {"causal": False}),
    ([1500, 1200], [128, 128], 128, 64, 128, 64, {}),                          # contexts of more than 1024 keys
    ([1500, 700, 300], [258, 257, 259], 32, 32, 64, 16, {"max_length": 1280}),
    ([5000], [257], 128, 128, 64, 16, {"window": 4000}),
    ([3000, 2500, 100], [160, 140, 100], 32, 8, 128, 16, {}),                  # float32: pieces of a long context, some without keys
    ([2900, 2300], [300, 260], 32, 32, 64, 20, {}),
    ([4000, 700], [140, 200], 32, 8, 80, 64, {"max_length": 2500}),
    ([150, 140, 133, 100] * 4, [100, 99, 70, 65] * 4, 12, 6, 40, 16, {}),      # chunks that fill half of their tiles
]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["s8", "f32"])
@pytest.mark.parametrize("case", range(len(TILES)))
def test_chunks_against_the_definition(pkg, T, kind, case):
    lengths, chunks, heads, kv, size, page, more = TILES[case]
    Made(pkg, kind, lengths, chunks, heads, kv, size, page, 100 + case).check(T, **more)


# Pages that end inside a step's keys: 16 rows and more, and fewer, a page for each key.
ENDS = [(kind, page, size, chunks, heads) for page in (17, 20, 24, 31, 40, 100, 5) for kind in ("s8", "f32")
        for size, chunks, heads in ((64, [1, 1, 1], 4), (128, [1, 33, 7], 4), (256, [1, 1, 1], 4), (64, [300, 270, 260], 64))]


@pytest.mark.gpu
@pytest.mark.parametrize("kind,page,size,chunks,heads", ENDS)
def test_pages_that_end_inside_a_step(pkg, T, kind, page, size, chunks, heads):
    m = Made(pkg, kind, [700, 333, 290], chunks, heads, heads // 2 if heads == 4 else heads, size, page, page)
    m.check(T)
    m.table[0, ::3] = -1
    m.table[1, 1::2] = len(m.cache[0])
    m.check(T)
    m.check(T, window=37)


@pytest.mark.gpu
def test_many_sequences(pkg, T):
    """More sequences than a wavefront has lanes, some without tokens."""
    rng = np.random.default_rng(9)
    chunks = rng.integers(0, 4, 150)
    chunks[:70] = 0
    lengths = chunks + rng.integers(0, 60, 150)
    for kind in ("s8", "f32"):
        Made(pkg, kind, lengths, chunks, 4, 2, 64, 16, 3).check(T)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["s8", "f32"])
@pytest.mark.parametrize("chunks,heads", [([1, 30, 64], 4), ([150, 90, 64], 4), ([300, 300, 300], 64)])
def test_pages_outside_the_cache(pkg, T, kind, chunks, heads):
    m = Made(pkg, kind, [200, 90, 64] if heads == 4 else [320, 310, 300], chunks, heads, heads // 2 if heads == 4 else heads, 64, 16, 4)
    m.table[0, [0, 5]] = [-1, 10 ** 6]
    m.table[1, 3] = len(m.cache[0])
    m.table[2] = -1  # nothing is there at all
    m.check(T)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["s8", "f32"])
@pytest.mark.parametrize("chunks,heads", [([1, 1], 6), ([40, 21], 6), ([120, 70], 6), ([258, 260], 128)])
def test_what_a_row_does_not_see_may_be_anything(pkg, T, kind, chunks, heads):
    import torch
    m = Made(pkg, kind, [150, 70] if heads == 6 else [290, 270], chunks, heads, heads // 3 if heads == 6 else heads // 2, 64, 16, 5)
    group = heads // m.cache[0].shape[1]
    clean = T.n(m.run(T)).copy()
    rows = np.ones((m.cache[0].shape[0], 16), bool)  # slots of no sequence
    for i, n in enumerate(m.lengths):
        at = np.arange(n)
        rows[m.table[i][at // 16], at % 16] = False
    for c in m.cache[:2] if kind == "f32" else m.cache[2:]:
        c.swapaxes(1, 2)[rows] = np.nan
    assert np.array_equal(T.n(m.run(T)), clean)
    # the last token's own key and value are not finite: the rows before it do not see them
    last = m.lengths[0] - 1
    page, inside = m.table[0, last // 16], last % 16
    if kind == "s8":
        m.cache[3][page, 1, inside] = np.inf
    else:
        m.cache[1][page, 1, inside, 5] = np.inf
        m.cache[1][page, 1, inside, 40] = np.nan
    got = T.n(m.run(T))
    mine = np.zeros(got.shape, bool)
    mine[m.starts[1] - 1, group:2 * group] = True
    assert np.array_equal(got[~mine], clean[~mine])
    if kind == "f32":
        assert np.isposinf(got[m.starts[1] - 1, group:2 * group, 5]).all() and np.isnan(got[m.starts[1] - 1, group:2 * group, 40]).all()
        m.check(T)
    else:
        assert np.isnan(got[m.starts[1] - 1, group:2 * group]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind,page", [("s8", 16), ("s8", 24), ("s8", 7), ("f32", 16), ("f32", 24), ("f32", 7)])
@pytest.mark.parametrize("lengths,chunks,heads", [([200, 64], [30, 1], 6), ([4000, 64], [1, 1], 2), ([290, 270], [258, 260], 128), ([3000, 100], [300, 100], 64)])
def test_queries_that_are_not_finite(pkg, T, kind, page, lengths, chunks, heads):
    """Their rows are NaN, not the zeros of a row that sees nothing; the others keep every bit."""
    m = Made(pkg, kind, lengths, chunks, heads, heads // 2, 64, page, 19)
    clean = T.n(m.run(T)).copy()
    for value in (np.nan, np.inf, -np.inf):
        token = chunks[0] - 1
        m.q[token, 1, 5] = value
        got = T.n(m.run(T))
        mine = np.zeros(got.shape, bool)
        mine[token, 1] = True
        assert np.isnan(got[mine]).all() and np.array_equal(got[~mine], clean[~mine])


@pytest.mark.gpu
@pytest.mark.parametrize("length,chunk,heads,size", [(200, 30, 6, 64), (290, 258, 64, 64), (300, 290, 64, 128), (3000, 300, 32, 128)])
def test_keys_that_are_not_finite(pkg, T, length, chunk, heads, size):
    """A score of infinity or NaN makes a row NaN, one of -infinity takes the key out; rows that do not see the key keep every bit."""
    m = Made(pkg, "f32", [length, 64], [chunk, 30], heads, heads // 2, size, 16, 18)
    clean = T.n(m.run(T)).copy()
    at = length - chunk // 2
    page, inside = m.table[0, at // 16], at % 16
    later = np.arange(length - chunk, length) >= at
    m.cache[0][page, 1, inside, 3] = np.nan
    got = T.n(m.run(T))
    assert np.isnan(got[:chunk, 2:4][later]).all() and np.array_equal(got[:chunk, 2:4][~later], clean[:chunk, 2:4][~later])
    m.cache[0][page, 1, inside, 3] = np.inf
    got = T.n(m.run(T)).astype(np.float64)
    mine = np.zeros(got.shape, bool)
    mine[:chunk, 2:4] = later[:, None, None]
    assert np.array_equal(got[~mine], clean[~mine])
    x = m.q[:chunk, 2:4, 3]
    assert np.isnan(got[:chunk, 2:4][later][x[later] > 0]).all()
    out = later[:, None] & (x < 0)
    want = np.zeros((chunk, 2, size))
    pages = m.table[0][np.arange(length) // 16]
    k, v = m.cache[0][pages, 1, np.arange(length) % 16].astype(np.float64), m.cache[1][pages, 1, np.arange(length) % 16].astype(np.float64)
    for t, h in zip(*np.nonzero(out)):
        seen = np.arange(length) <= length - chunk + t
        seen[at] = False
        s = k[seen] @ m.q[t, 2 + h].astype(np.float64) * m.scale
        w = np.exp(s - s.max())
        want[t, h] = w / w.sum() @ v[seen]
    assert out.any() and rel_fro(got[:chunk, 2:4][out], want[out]) < 1e-5


@pytest.mark.gpu
@pytest.mark.parametrize("chunks,heads,kv", [([2, 45], 4, 2), ([200, 45], 4, 2), ([257, 270], 64, 64)])
def test_scales_of_all_sizes(pkg, T, chunks, heads, kv):
    """Rows of values from 10^-20 to 10^20, zeros among them, and queries likewise."""
    m = Made(pkg, "s8", [300, 45 if kv == 2 else 270], chunks, heads, kv, 128, 16, 6)
    m.cache[3][:] = np.exp(m.rng.normal(size=m.cache[3].shape) * 15).astype(np.float32)
    m.cache[3][m.rng.random(m.cache[3].shape) < 0.2] = 0
    m.cache[2][m.rng.random(m.cache[2].shape) < 0.2] = 0
    m.q[1] *= 1e-25
    m.q[2] = 0
    m.check(T)
    for c in m.cache[3:]:
        c[:] = 0
    assert not T.n(m.run(T)).any()


@pytest.mark.gpu
@pytest.mark.parametrize("length,chunk,kv", [(4000, 1, 2), (300, 20, 2), (1100, 128, 128)])
@pytest.mark.parametrize("order", [1, -1])
def test_scales_further_apart_than_float32_exponents(pkg, T, length, chunk, kv, order):
    """The weights of keys whose values are small beside the others' count in full, whichever come first."""
    m = Made(pkg, "s8", [length], [chunk], kv, kv, 64, 16, 17)
    at = np.arange(m.lengths[0])
    scales = np.where((at < length * 3 // 4)[::order], np.float32(1e-25), np.float32(1e25)).astype(np.float32)
    m.cache[3][m.table[0][at // 16], :, at % 16] = scales[:, None]
    m.check(T)


@pytest.mark.gpu
@pytest.mark.parametrize("chunks,heads,kv", [([3, 30], 4, 2), ([250, 30], 4, 2), ([257, 270], 64, 64)])
def test_large_scores(pkg, T, chunks, heads, kv):
    """Weights that all fall on one key or underflow."""
    for kind in ("s8", "f32"):
        m = Made(pkg, kind, [400, 30 if kv == 2 else 300], chunks, heads, kv, 64, 16, 7)
        m.scale *= 100
        m.check(T)


@pytest.mark.gpu
@pytest.mark.parametrize("chunk,kv", [(1, 1), (64, 1), (128, 128)])
def test_rows_whose_scores_rise_beside_rows_whose_do_not(pkg, T, chunk, kv):
    """The largest score of one row moves with every key, that of the other stays: neither loses what it has."""
    m = Made(pkg, "s8", [5000 if kv == 1 else 1500], [chunk], 2 * kv, kv, 64, 16, 13)
    m.cache[0][:] = m.cache[0][0, 0, 0]
    at = np.arange(m.lengths[0])
    m.cache[2][m.table[0][at // 16], :, at % 16] = np.linspace(0.001, 0.02, len(at), dtype=np.float32)[:, None]
    m.q[:, 0::2] = m.cache[0][0, 0, 0] / np.float32(100)
    m.q[:, 1::2] = -m.q[:, 0::2]
    got = m.run(T)
    m.check(T, got)
    want, _ = R.attention(m.q, m.cache, m.table, m.starts, m.lengths, m.scale)
    assert rel_fro(T.n(got), want) <= 1.5e-6  # scores up to 20: 20 x 2^-24 each


@pytest.mark.gpu
@pytest.mark.parametrize("kind,size", [("s8", 64), ("f32", 64), ("s8", 72), ("f32", 100)])
def test_strides(pkg, T, kind, size):
    import torch
    from test_gpu_paged_cache import strided
    m = Made(pkg, kind, [300, 45], [1, 20], 4, 2, size, 16, 8)
    plain = m.run(T)
    assert torch.equal(m.run(T, cache=strided(m.on(T))), plain)
    wide = torch.full((21, 3, 4, size + 4), 9.0, device="cuda")
    q, out = wide[:, 0, :, 4:], wide[:, 2, :, 4:]
    q.copy_(T.t(m.q))
    before = wide.clone()
    got = pkg.paged_attention(q, m.on(T), T.t(np.concatenate([m.table, m.table], 1))[:, :m.table.shape[1]], T.t(m.starts), T.t(m.lengths), m.scale, out=out)
    assert got is out and torch.equal(out, plain)
    before[:, 2, :, 4:] = plain
    assert torch.equal(wide, before)
    # a query that does not begin at 16 bytes
    with pytest.raises(pkg.TfccRocmError):
        pkg.paged_attention(torch.zeros((21, 4, size + 1), device="cuda")[..., 1:], m.on(T), T.t(m.table), T.t(m.starts), T.t(m.lengths), m.scale)


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,chunks", [([2000, 1, 700], [1, 1, 1]), ([90, 200], [60, 3])])
def test_rows_behind_the_last_sequence_stay(pkg, T, lengths, chunks):
    import torch
    m = Made(pkg, "s8", lengths, chunks, 8, 2, 64, 16, 10)
    n = int(m.starts[-1])
    want = m.run(T)
    m.q = np.concatenate([m.q, m.q[:2], m.q[:1] * np.nan])
    out = torch.full(m.q.shape, 3.25, device="cuda")
    m.run(T, out=out)
    assert torch.allclose(out[:n], want, rtol=1e-5, atol=1e-6) and bool((out[n:] == 3.25).all())


@pytest.mark.gpu
def test_offsets_past_32_bits(pkg, T):
    """Pages that lie more than 2^32 elements into the cache."""
    import torch
    pages, page, size = 2 ** 20 + 64, 64, 72
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("not enough memory")
    cache = pkg.paged_cache(pages, 1, page, size)
    m = Made(pkg, "s8", [200, 77], [1, 20], 4, 1, size, page, 11)
    there = pages - 1 - np.arange(m.cache[0].shape[0])
    for big, small in zip(cache, m.cache):
        big[torch.from_numpy(there).cuda()] = T.t(small)
    small = m.on(T)
    want = m.run(T, cache=small)
    table = m.table
    m.table = np.where((table >= 0) & (table < len(there)), there[np.clip(table, 0, len(there) - 1)], -1).astype(np.int32)
    assert torch.equal(m.run(T, cache=cache), want)
    back = pkg.cache_read(cache, T.t(m.table), T.t(np.array([0, 200, 277], np.int32)), 277)
    near = pkg.cache_read(small, T.t(table), T.t(np.array([0, 200, 277], np.int32)), 277)
    assert torch.equal(back[0], near[0]) and torch.equal(back[1], near[1])
    x = T.t(m.rng.normal(size=(2, 1, size)).astype(np.float32))
    slots = np.array([pages * page - 1, (pages - 3) * page + 5])
    pkg.cache_write(cache, x, x, T.t(slots))
    n, s = R.quantized(T.n(x))
    assert np.array_equal(T.n(cache[0][-1, :, -1]), n[0]) and np.array_equal(T.n(cache[3][-3, :, 5]), s[1])


@pytest.mark.gpu
def test_refused(pkg, T):
    import torch
    m = Made(pkg, "s8", [30], [2], 4, 2, 64, 16, 12)
    cache, q, table, starts, lengths = m.on(T), T.t(m.q), T.t(m.table), T.t(m.starts), T.t(m.lengths)
    for args in ((q[:, :3], cache, table, starts, lengths), (q[..., :32], cache, table, starts, lengths), (q, cache, table.long(), starts, lengths),
                 (q, cache, table, starts[:1], lengths), (q, cache, table, starts, lengths.long()), (q.double(), cache, table, starts, lengths),
                 (q, cache[:2], table, starts, lengths), (q, cache, table.cpu(), starts, lengths), (q, cache, torch.cat([table, table]), starts, lengths)):
        with pytest.raises(pkg.InvalidArgumentError):
            pkg.paged_attention(*args, 0.125)
    for kw in (dict(window=-1), dict(window=3, causal=False), dict(max_length=-1), dict(out=q[:1]), dict(out=q.double())):
        with pytest.raises(pkg.InvalidArgumentError):
            pkg.paged_attention(q, cache, table, starts, lengths, 0.125, **kw)
    assert pkg.paged_attention(q[:0], cache, table, torch.zeros_like(starts), lengths, 0.125).shape == (0, 4, 64)
