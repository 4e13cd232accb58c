"""Attention over a paged cache of 4-bit integers, and with capped scores, distance biases and prefixes over caches of all types, against the
definition in 64 bits, within what float32 sums may be off by."""
import ctypes as C

import numpy as np
import pytest

import serving_reference as R
from conftest import rel_fro
from test_gpu_paged_attention import Made as Plain


class Made(Plain):
    """As for plain scores, with a cache of any type."""

    def __init__(self, pkg, kind, lengths, chunks, heads, kv, size, page, seed, spare=2):
        super().__init__(pkg, "s8" if kind == "s4" else kind, lengths, chunks, heads, kv, size, page, seed, spare)
        if kind == "s4":
            self.cache[:2] = [R.pack(self.rng.integers(-8, 8, c.shape)) for c in self.cache[:2]]
            self.cache[2:] = [c * np.float32(16) for c in self.cache[2:]]

    def shaped(self, kw, cap=0.0, slopes=False, prefixes=None):
        """The arguments of a call with a shape of its scores."""
        heads = self.q.shape[1]
        kw = dict(kw)
        if cap:
            kw["cap"] = cap
        if slopes:
            kw["slopes"] = (2.0 ** (-8.0 * (1 + np.arange(heads)) / heads)).astype(np.float32) * self.rng.choice([1, 1, 1, -0.01], heads).astype(np.float32)
        if prefixes is not None:
            kw["prefixes"] = np.array(prefixes, np.int32)
        return kw

    def off(self, **kw):
        """How far two kernels may be from each other: each may be so far from the definition."""
        return 2 * R.attention(self.q, self.cache, self.table, self.starts, self.lengths, self.scale, **kw)[1]

    def check(self, T, got=None, cache=None, **kw):
        given = {k: T.t(v) if isinstance(v, np.ndarray) else v for k, v in kw.items()}
        got = T.n(self.run(T, cache, **given) if got is None else got).astype(np.float64)
        want, off = R.attention(self.q, self.cache, self.table, self.starts, self.lengths, self.scale, most=kw.pop("max_length", None), **kw)
        assert np.array_equal(np.isnan(got), np.isnan(want))
        fine = np.isfinite(want)
        assert (np.abs(got - want) <= off)[fine].all(), np.nanmax((np.abs(got - want) / off)[fine])
        assert rel_fro(got[fine], want[fine]) <= 1e-5


def test_refused_without_a_device(pkg):
    lib, d, s = pkg.lib(), pkg.PagedAttentionDesc(), pkg.AttentionScores()
    call = lambda: lib.tfcc_rocm_paged_attention_scores_f32(None, C.byref(d), C.byref(s))
    assert lib.tfcc_rocm_paged_attention_scores_f32(None, None, C.byref(s)) == 1 and lib.tfcc_rocm_paged_attention_scores_f32(None, C.byref(d), None) == 1
    c = d.cache
    c.keys = c.values = c.key_scales = c.value_scales = 4096
    c.type, c.pages, c.heads, c.page_size, c.size = pkg.S4, 200, 2, 16, 64
    d.heads, d.tokens, d.batch, d.table_width, d.causal = 8, 1, 1, 200, 1
    for s.cap, fits in ((0.0, True), (30.0, True), (-1.0, False), (float("nan"), False), (float("inf"), False)):
        assert call() == 1 and (b"null" in lib.tfcc_rocm_last_error_string()) == fits
    s.cap, s.prefixes = 0.0, 4096
    assert call() == 1 and b"null" in lib.tfcc_rocm_last_error_string()
    d.window = 3
    assert call() == 1 and b"prefix" in lib.tfcc_rocm_last_error_string()
    d.window, d.causal = 0, 0
    assert call() == 1 and b"prefix" in lib.tfcc_rocm_last_error_string()
    s.prefixes, s.slopes, s.cap = None, 4096, 5.0
    assert call() == 1 and b"null" in lib.tfcc_rocm_last_error_string()
    for c.size in (8, 24, 40, 72, 272):
        assert call() == 1 and b"heads of" in lib.tfcc_rocm_last_error_string()
    c.size, d.tokens = 64, 0
    assert call() == 0


def test_tanh():
    """What the kernels form below 0.55 and above, in float32: half a step and the rounding of the last sums below; above, the difference of 1 and a number
    below 1 whose parts are a few steps off."""
    x = np.concatenate([np.linspace(1e-6, 0.55, 200001), np.geomspace(1e-30, 1e-3, 20001)]).astype(np.float32)
    f = np.float32
    y = x * x
    r = np.full_like(x, f(-0.00627424))
    for c in (0.02107168, -0.05385231, 0.13332586, -0.33333318):
        r = (r.astype(np.float64) * y + f(c)).astype(f)
    got = ((x * y).astype(np.float64) * r + x).astype(f)
    want = np.tanh(x.astype(np.float64))
    assert (np.abs(got - want) <= 2.0 ** -23 * want).all()
    x = np.linspace(0.55, 20, 200001).astype(f)
    e = np.exp2((x * f(2.88539008)).astype(f).astype(np.float64)).astype(f)
    got = 1 - 2 * (1 / (e + f(1))).astype(f).astype(np.float64)
    want = np.tanh(x.astype(np.float64))
    assert (np.abs(got - want) <= 6 * 2.0 ** -24 * want).all()


CASES = [
    # lengths, chunks, heads, kv heads, size, page, more
    ([1], [1], 1, 1, 64, 16, {}),
    ([777], [1], 12, 12, 64, 16, {}),
    ([33, 0, 200, 1, 517], [1, 1, 1, 1, 1], 8, 2, 128, 32, {}),         # one has nothing cached
    ([40, 300, 90], [40, 7, 0], 6, 2, 128, 16, {}),                      # a whole prompt, a chunk, a sequence without one
    ([3, 70], [5, 66], 4, 4, 64, 16, {}),                                # more tokens than cached: the first see nothing
    ([257, 65], [1, 3], 20, 5, 80, 24, {}),                              # rows of 40 bytes, pages that end inside a tile
    ([130, 61], [30, 2], 3, 1, 48, 7, {}),                               # odd pages, groups of three
    ([129], [9], 33, 1, 208, 1, {}),                                     # pages of one row, more heads than a tile has rows
    ([300, 41], [2, 5], 2, 2, 16, 16, {}),                               # rows of 8 bytes
    ([300, 41], [2, 5], 2, 2, 32, 20, {}),
    ([500, 90], [64, 1], 4, 2, 256, 64, {}),
    ([500, 90], [4, 1], 4, 2, 192, 24, {}),
    ([700, 100], [3, 100], 8, 8, 64, 16, {"window": 1}),
    ([1500, 600], [1, 130], 8, 1, 128, 32, {"window": 300}),
    ([90, 300], [20, 3], 4, 4, 96, 16, {"causal": False}),
    ([900, 60], [2, 2], 4, 1, 64, 16, {"max_length": 512}),              # keys behind the bound are not seen
    ([3000, 1, 2048, 129], [1, 1, 1, 1], 32, 8, 128, 128, {}),           # many pieces
    ([6000], [70], 8, 2, 128, 64, {}),
    ([2500, 700], [90, 90], 8, 2, 128, 16, {"max_length": 2100}),
    ([1000, 257], [130, 257], 8, 2, 128, 32, {}),
    ([290, 100], [290, 100], 4, 2, 256, 16, {}),
]
SHAPES = [{"cap": 5.0}, {"slopes": True}, {"cap": 2.0, "slopes": True}, {"prefix": True}, {"cap": 30.0, "slopes": True, "prefix": True}]


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(CASES)))
def test_4_bits_against_the_definition(pkg, T, case):
    lengths, chunks, heads, kv, size, page, more = CASES[case]
    Made(pkg, "s4", lengths, chunks, heads, kv, size, page, case).check(T, **more)


def fits(shape, more):
    """A prefix has neither a window nor all keys."""
    return "prefix" not in shape or not (more.get("window") or not more.get("causal", True))


def shape_of(m, shape, more):
    if "prefix" not in shape:
        return m.shaped(more, **shape)
    return m.shaped(more, shape.get("cap", 0.0), shape.get("slopes", False), m.rng.integers(-3, m.lengths + 40))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["s4", "s8", "f32"])
@pytest.mark.parametrize("case,shape", [(c, s) for c in range(len(CASES)) for s in range(len(SHAPES)) if fits(SHAPES[s], CASES[c][-1])])
def test_shaped_against_the_definition(pkg, T, kind, shape, case):
    lengths, chunks, heads, kv, size, page, more = CASES[case]
    m = Made(pkg, kind, lengths, chunks, heads, kv, size, page, 100 + case)
    m.q *= np.float32(1 + case % 4)  # scores on both sides of what the cap bends
    m.check(T, **shape_of(m, SHAPES[shape], more))


# Chunks of many tokens, most of which go over the keys together, 128 or 256 rows in a workgroup.
TILES = [
    ([600, 300, 257, 700], [300, 300, 257, 290], 32, 32, 64, 16, {}),
    ([300, 290, 0, 1100, 260, 257], [70, 97, 0, 90, 64, 65], 64, 16, 128, 32, {}),
    ([400, 200, 90], [260, 280, 90], 48, 48, 96, 16, {}),                      # more tokens than are cached
    ([290, 280], [290, 270], 64, 64, 160, 16, {}),
    ([290, 300], [290, 258], 64, 64, 256, 16, {}),
    ([700, 600], [300, 290], 64, 64, 64, 32, {"window": 1}),
    ([700, 600], [128, 140], 128, 64, 128, 32, {"window": 150}),
    ([300, 400], [260, 270], 64, 64, 128, 16, {"causal": False}),
    ([1500, 700, 300], [258, 257, 259], 32, 32, 64, 16, {"max_length": 1280}),
    ([3000, 2500, 100], [160, 140, 100], 32, 8, 128, 16, {}),
    ([2900, 2300], [300, 260], 32, 32, 64, 20, {}),                            # pages that end inside a step
    ([150, 140, 133, 100] * 4, [100, 99, 70, 65] * 4, 12, 6, 32, 16, {}),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(TILES)))
def test_chunks_of_4_bits_against_the_definition(pkg, T, case):
    lengths, chunks, heads, kv, size, page, more = TILES[case]
    Made(pkg, "s4", lengths, chunks, heads, kv, size, page, case).check(T, **more)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["s4", "s8", "f32"])
@pytest.mark.parametrize("case,shape", [(c, s) for c in range(len(TILES)) for s in (2, 4) if fits(SHAPES[s], TILES[c][-1])])
def test_shaped_chunks_against_the_definition(pkg, T, kind, shape, case):
    lengths, chunks, heads, kv, size, page, more = TILES[case]
    m = Made(pkg, kind, lengths, chunks, heads, kv, size, page, 50 + case)
    m.check(T, **shape_of(m, SHAPES[shape], more))


# Wide tiles of 4-bit integers: chunks that fill half of them, and 450 workgroups, or 280 over up to 512 keys; heads of 80 have rows of 40 bytes.
WIDE = [
    ([600, 400, 300], [260, 270, 290], 128, 64, 128, 32, {}),
    ([300, 290, 0, 500, 260], [70, 97, 0, 90, 64], 128, 64, 128, 16, {}),
    ([700, 600, 90], [300, 200, 90], 128, 64, 96, 20, {}),
    ([513, 600, 90], [260, 300, 90], 128, 64, 80, 48, {}),
    ([513, 600], [260, 300], 128, 64, 112, 20, {"window": 100}),
    ([700, 600], [128, 140], 256, 64, 128, 32, {"window": 1}),
    ([300, 400], [260, 270], 128, 64, 128, 16, {"causal": False}),
    ([1500, 700, 300], [258, 257, 259], 64, 64, 128, 64, {"max_length": 1280}),
    ([400, 200, 90], [260, 280, 90], 96, 48, 128, 24, {}),                     # more tokens than are cached
    ([3000, 2500], [200, 160], 256, 64, 128, 32, {}),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(WIDE)))
def test_wide_tiles_of_4_bits(pkg, T, case):
    lengths, chunks, heads, kv, size, page, more = WIDE[case]
    there = [n for n in chunks if n]
    each = -(-(-(-sum(there) // len(chunks)) * heads // kv) // 128)
    assert len(chunks) * each * kv >= (280 if max(lengths) <= 512 else 450)
    m = Made(pkg, "s4", lengths, chunks, heads, kv, size, page, case)
    m.check(T, **more)
    m.check(T, **m.shaped(more, cap=4.0, slopes=True, prefixes=None if more.get("window") or "causal" in more else [100] * len(lengths)))
    if case in (0, 3):
        m.table[0, 0], m.table[1, 2], m.table[2, -1] = -1, m.cache[0].shape[0], 2 ** 31 - 1
        m.check(T)
        # what no row sees, and what only the last rows see, may be anything
        before = T.n(m.run(T))
        for i, (n, chunk) in enumerate(zip(lengths, chunks)):
            for s in m.cache[2:]:
                s[m.table[i][(n - 1) // page], :, (n - 1) % page] = np.nan
        got, last = T.n(m.run(T)), m.starts[1:] - 1
        rest = np.setdiff1d(np.arange(len(m.q)), last)
        assert np.isnan(got[last]).all() and np.array_equal(got[rest], before[rest])


@pytest.mark.gpu
@pytest.mark.parametrize("batch,longest,chunk,heads,kv,size,page", [(70, 900, 1, 16, 8, 64, 16), (150, 300, 3, 12, 4, 32, 32), (64, 1300, 1, 8, 8, 128, 64), (130, 40, 1, 4, 4, 48, 24),
                                                                    (40, 700, 2, 8, 8, 256, 32), (65, 3000, 1, 24, 4, 96, 16), (20, 1500, 9, 66, 2, 64, 20)])
def test_many_sequences_of_all_lengths(pkg, T, batch, longest, chunk, heads, kv, size, page):
    """More workgroups than run at once, taken by falling length: lengths of zero, equal ones, sequences without a chunk."""
    rng = np.random.default_rng(batch)
    lengths = rng.integers(0, longest + 1, batch)
    lengths[::7], lengths[3::9] = longest, 0
    chunks = np.where(rng.random(batch) < 0.15, 0, rng.integers(1, chunk + 1, batch))
    m = Made(pkg, "s4", lengths.tolist(), chunks.tolist(), heads, kv, size, page, batch)
    m.check(T)
    m.check(T, max_length=longest // 2)
    m.check(T, **m.shaped({}, cap=3.0, slopes=True))


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,heads,kv,size,page", [([5000, 3000, 1100] * 11, 8, 4, 128, 32), ([4100] * 40, 12, 6, 64, 16), ([2500, 1] * 50, 4, 2, 256, 64),
                                                        ([4000, 900] * 16, 8, 8, 32, 20), ([9000], 64, 32, 128, 64)])
def test_workgroups_of_many_wavefronts(pkg, T, lengths, heads, kv, size, page):
    m = Made(pkg, "s4", lengths, [1] * len(lengths), heads, kv, size, page, len(lengths))
    m.check(T)
    m.check(T, window=1500)
    m.check(T, **m.shaped({}, cap=3.0, slopes=True, prefixes=[40] * len(lengths)))


PIECES = [
    # kind, lengths, chunks, heads, kv heads, size, page of calls whose keys come in 3 to 137 pieces, some in one, and in 2 and 3 with wide tiles
    ("s4", [1000], [1], 64, 64, 64, 16),
    ("s8", [1500, 90], [2, 1], 60, 60, 64, 16),
    ("f32", [1000, 300], [1, 3], 24, 24, 64, 16),
    ("s8", [1790], [1], 32, 8, 128, 32),
    ("f32", [1000, 300], [1, 3], 12, 12, 64, 16),
    ("s4", [2300, 40], [1, 1], 8, 2, 128, 32),
    ("f32", [9000], [1], 8, 1, 256, 16),
    ("s8", [70000], [1], 4, 1, 80, 64),
    ("s4", [33000], [2], 2, 1, 32, 32),
    ("f32", [1000, 20, 640], [512, 20, 600], 12, 12, 64, 16),
    ("f32", [1500, 1100], [160, 120], 32, 8, 128, 16),
    ("s8", [2100, 40], [1060, 40], 32, 8, 128, 16),
]


@pytest.mark.gpu
@pytest.mark.parametrize("rising", [1, -1])
@pytest.mark.parametrize("case", range(len(PIECES)))
def test_pieces_joined(pkg, T, case, rising):
    """Scores that rise or fall by 60 over the keys, so that the largest is in one piece and the others' sums shrink to it; prefixes, by which pieces are
    empty for some rows and not for others; and rows that see nothing."""
    kind, lengths, chunks, heads, kv, size, page = PIECES[case]
    m = Made(pkg, kind, lengths, chunks, heads, kv, size, page, 100 + case)
    m.check(T)
    slopes = np.full(heads, rising * 60.0 / max(lengths), np.float32)
    m.check(T, slopes=slopes)
    m.check(T, slopes=-slopes / 6, cap=3.0, prefixes=np.array([n // 3 for n in lengths], np.int32))
    m.lengths[-1] = 0
    m.check(T, slopes=slopes)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["s4", "s8", "f32"])
@pytest.mark.parametrize("lengths,chunks,heads,kv", [([400, 90], [3, 1], 8, 2), ([700, 300], [300, 290], 64, 64)])
def test_prefixes(pkg, T, kind, lengths, chunks, heads, kv):
    """Of nothing, of all, of more than is cached, and up to the middle of the chunk; a sequence whose tokens are all before it."""
    for prefixes in ([0, 0], [-7, 1], [lengths[0], lengths[1]], [1 << 30, 2 ** 31 - 1], [lengths[0] - 1, lengths[1] - chunks[1]], [17, lengths[1] - 5]):
        m = Made(pkg, kind, lengths, chunks, heads, kv, 64, 16, 7)
        m.check(T, **m.shaped({}, prefixes=prefixes))
    # more tokens than are cached: those before the first key see the prefix alone
    m = Made(pkg, kind, [30, 20], [40, 3], 4, 4, 64, 16, 8)
    m.check(T, **m.shaped({}, slopes=True, prefixes=[7, 0]))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["s4", "s8", "f32"])
@pytest.mark.parametrize("lengths,chunks,heads,kv", [([400, 90], [3, 1], 8, 2), ([5000], [1], 2, 2), ([700, 300], [300, 290], 64, 64)])
def test_caps_of_all_sizes(pkg, T, kind, lengths, chunks, heads, kv):
    """Scores far above their cap and far below, and scores that overflow: they are those of an infinity."""
    for cap, times in ((50.0, 0.01), (50.0, 30.0), (1e-3, 1.0), (1e30, 1.0), (8.0, 1e3), (3e38, 1.0)):
        m = Made(pkg, kind, lengths, chunks, heads, kv, 64, 16, 3)
        m.q *= np.float32(times)
        m.check(T, **m.shaped({}, cap=cap))
    m = Made(pkg, kind, lengths, chunks, heads, kv, 64, 16, 3)
    m.q = np.sign(m.q) * np.float32(3e38)
    m.q[..., 1:] = 0
    m.scale = 1e4  # scores beyond float32 where the first values are not 0
    m.check(T, **m.shaped({}, cap=20.0))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["s4", "s8", "f32"])
def test_no_shape_is_the_plain_call(pkg, T, kind):
    m = Made(pkg, kind, [700, 90], [3, 20], 4, 2, 64, 16, 3)
    plain = T.n(m.run(T))
    for kw in ({"cap": 0.0}, {"cap": 0}, {"slopes": T.t(np.zeros(4, np.float32))}, {"prefixes": T.t(np.zeros(2, np.int32))}):
        assert (np.abs(T.n(m.run(T, **kw)).astype(np.float64) - plain) <= m.off()).all()
    assert np.array_equal(T.n(m.run(T, cap=0)), plain)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["s4", "s8", "f32"])
def test_far_positions(pkg, T, kind):
    """Positions far behind all keys that a bound lets a row see: the bias is that of the differences."""
    m = Made(pkg, kind, [300], [2], 4, 2, 64, 16, 3)
    m.lengths = np.array([1 << 30], np.int32)
    kw = m.shaped({"max_length": 300}, slopes=True)
    got = T.n(m.run(T, max_length=300, slopes=T.t(kw["slopes"])))
    shifted = Made(pkg, kind, [300], [2], 4, 2, 64, 16, 3)
    shifted.lengths = np.array([302], np.int32)  # two positions behind the last key
    near = T.n(shifted.run(T, max_length=300, slopes=T.t(kw["slopes"])))
    assert np.isfinite(got).all() and np.array_equal(got, near)


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,chunks,heads", [([1, 30, 64], [1, 30, 64], 4), ([300, 300, 300], [300, 300, 300], 64), ([3000, 40, 9], [1, 1, 1], 4)])
@pytest.mark.parametrize("page", [16, 24, 8])
def test_pages_outside_the_cache(pkg, T, lengths, chunks, heads, page):
    for kind in ("s4", "s8", "f32"):
        m = Made(pkg, kind, lengths, chunks, heads, heads, 64, page, 5)
        m.table[0, 0], m.table[1, 1], m.table[2, -1] = -1, m.cache[0].shape[0], 2 ** 31 - 1
        m.check(T, **m.shaped({}, cap=4.0, slopes=True, prefixes=[0, 20, 200]))
        if kind == "s4":
            m.check(T)


@pytest.mark.gpu
@pytest.mark.parametrize("chunks,heads", [([1, 1], 6), ([40, 21], 6), ([258, 260], 128)])
def test_what_a_row_does_not_see_may_be_anything(pkg, T, chunks, heads):
    """Scales of NaN and infinity behind the sequences' ends, on other pages, and among what only later tokens see."""
    lengths = [290, 270]
    m = Made(pkg, "s4", lengths, chunks, heads, heads // 2, 64, 16, 9)
    before = T.n(m.run(T))
    shaped = m.shaped({}, cap=3.0, slopes=True)
    on = {k: T.t(v) if isinstance(v, np.ndarray) else v for k, v in shaped.items()}
    shaped_before = T.n(m.run(T, **on))
    used = np.zeros(m.cache[2].shape, bool)
    for i, n in enumerate(lengths):
        at = np.arange(n)
        used[m.table[i][at // 16], :, at % 16] = True
    for s in m.cache[2:]:
        s[~used] = np.where(m.rng.random(s.shape) < 0.5, np.nan, np.inf)[~used]
    assert np.array_equal(T.n(m.run(T)), before) and np.array_equal(T.n(m.run(T, **on)), shaped_before)
    # the last key of each sequence concerns the last token alone
    for i, n in enumerate(lengths):
        for s in m.cache[2:]:
            s[m.table[i][(n - 1) // 16], :, (n - 1) % 16] = np.nan
    last = m.starts[1:] - 1
    rest = np.setdiff1d(np.arange(len(m.q)), last)
    for kw, want in (({}, before), (on, shaped_before)):
        got = T.n(m.run(T, **kw))
        assert np.isnan(got[last]).all() and np.array_equal(got[rest], want[rest])


@pytest.mark.gpu
@pytest.mark.parametrize("length,chunk,kv", [(4000, 1, 2), (300, 20, 2), (1100, 128, 128)])
@pytest.mark.parametrize("order", [1, -1])
def test_scales_further_apart_than_float32_exponents(pkg, T, length, chunk, kv, order):
    m = Made(pkg, "s4", [length], [chunk], 2 * kv, kv, 64, 16, 2)
    at = np.arange(length)
    m.cache[3][m.table[0][at // 16], :, at % 16] = np.exp2(np.linspace(-90, 90, length)[::order])[:, None].astype(np.float32)
    m.check(T)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["s4", "s8", "f32"])
@pytest.mark.parametrize("size", [64, 96, 80])
def test_strides(pkg, T, kind, size):
    """A cache of other strides and queries among other heads, prefixes and slopes from views."""
    import torch
    m = Made(pkg, kind, [200, 64, 33], [30, 1, 2], 6, 2, size, 16, 4)
    shaped = m.shaped({}, cap=6.0, slopes=True, prefixes=[20, 0, 33])
    on = {k: T.t(v) if isinstance(v, np.ndarray) else v for k, v in shaped.items()}
    want = T.n(m.run(T, **on))
    cache = m.on(T)
    pages, kv, page, width = cache[0].shape
    memory = torch.zeros((pages, page, kv, 2, width + 16), dtype=cache[0].dtype, device="cuda")
    views = [memory[:, :, :, i, 16:].permute(0, 2, 1, 3) for i in (0, 1)]
    if kind != "f32":
        scales = torch.zeros((pages, page, 2, kv + 3), device="cuda")
        views += [scales[:, :, i, 1:1 + kv].permute(0, 2, 1) for i in (0, 1)]
    for v, t in zip(views, cache):
        v.copy_(t)
    wide = torch.zeros((m.q.shape[0], 3, 6, size + 4), device="cuda")
    q = wide[:, 1, :, 4:]
    q.copy_(T.t(m.q))
    out = torch.zeros((m.q.shape[0], 6, 2 * size), device="cuda")[..., :size]
    slopes = torch.zeros((6, 2), device="cuda")
    slopes[:, 1] = on["slopes"]
    got = m.pkg.paged_attention(q, tuple(views), T.t(m.table), T.t(m.starts), T.t(m.lengths), m.scale, out=out, cap=6.0, slopes=slopes[:, 1], prefixes=on["prefixes"])
    assert got is out
    assert (np.abs(T.n(out).astype(np.float64) - want) <= m.off(**shaped)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,chunks", [([2000, 1, 700], [1, 1, 1]), ([90, 200], [60, 3])])
def test_rows_behind_the_last_sequence_stay(pkg, T, lengths, chunks):
    import torch
    for kind in ("s4", "f32"):
        m = Made(pkg, kind, lengths, chunks, 4, 2, 64, 16, 6)
        tokens = m.q.shape[0]
        m.q = np.concatenate([m.q, np.ones((5, 4, 64), np.float32)])
        out = torch.full(m.q.shape, 9.0, device="cuda")
        m.run(T, out=out, cap=5.0)
        assert (T.n(out)[tokens:] == 9).all() and np.isfinite(T.n(out)).all()


@pytest.mark.gpu
def test_offsets_past_32_bits(pkg, T):
    """Pages further apart than 2^32 bytes."""
    import torch
    m = Made(pkg, "s4", [60], [2], 4, 2, 64, 16, 6)
    want = T.n(m.run(T))
    pages = m.cache[0].shape[0]
    far = (1 << 32) // 4 + 4096
    cache = []
    for t in m.on(T):
        if t.dim() == 4:
            memory = torch.empty((far * pages,), dtype=t.dtype, device="cuda")
            v = torch.as_strided(memory, t.shape, (far, *t.stride()[1:]))
            v.copy_(t)
            t = v
        cache.append(t)
    assert np.array_equal(T.n(m.run(T, tuple(cache))), want)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["s4", "s8", "f32"])
def test_captured(pkg, T, kind):
    """What slopes, prefixes, lengths and queries hold is read when the graph runs; eager work between the replays."""
    import torch
    m = Made(pkg, kind, [900, 40, 300], [1, 1, 1], 8, 2, 128, 16, 3)
    shaped = m.shaped({}, slopes=True, prefixes=[5, 0, 10])
    q, cache, table, starts, lengths = T.t(m.q), m.on(T), T.t(m.table), T.t(m.starts), T.t(m.lengths)
    slopes, prefixes = T.t(shaped["slopes"]), T.t(shaped["prefixes"])
    call = lambda: pkg.paged_attention(q, cache, table, starts, lengths, m.scale, max_length=900, cap=9.0, slopes=slopes, prefixes=prefixes)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call()
        with torch.cuda.graph(graph, stream=stream):
            out = call()
    for seed in range(4):
        rng = np.random.default_rng(seed)
        q.copy_(T.t(rng.normal(size=m.q.shape).astype(np.float32)))
        slopes.mul_(1.5)
        lengths.copy_(T.t(np.array([900 - seed, 40, 200 + seed], np.int32)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call())


@pytest.mark.gpu
def test_a_step_of_a_model(pkg, T):
    """Norm, rotary positions, a write into a 4-bit cache, a fork of its last page, and attention for both sequences."""
    import torch
    rng = np.random.default_rng(11)
    heads, kv, size, page, length = 4, 2, 64, 16, 53
    cache = pkg.paged_cache(8, kv, page, size, torch.uint8)
    x = [rng.normal(size=(length, kv, size)).astype(np.float32) for _ in range(2)]
    table = np.array([[3, 0, 6, 1], [3, 0, 6, 5]], np.int32)  # the fourth page is forked
    slot = lambda i, at: table[i][at // page] * page + at % page
    pkg.cache_write(cache, T.t(x[0]), T.t(x[1]), T.t(np.array([slot(0, a) for a in range(length)], np.int32)))
    pkg.cache_copy(cache, T.t(np.array([page], np.int64)), T.t(np.array([5 * page], np.int64)), T.t(np.array([length - 3 * page], np.int32)))
    # a token more in each
    new = rng.normal(size=(2, 2, kv, size)).astype(np.float32)
    frequencies = torch.tensor(pkg.rotary_frequencies(size)[0], dtype=torch.float64, device="cuda")
    positions = T.t(np.array([length, length], np.int32))
    q = rng.normal(size=(2, heads * size)).astype(np.float32)
    normed, _ = pkg.rms_norm(T.t(q), T.t(np.ones(heads * size, np.float32)), 1e-6)
    turned, keys = pkg.rotary(normed.view(2, heads, size), T.t(new[0]), positions, frequencies)
    pkg.cache_write(cache, keys, T.t(new[1]), T.t(np.array([slot(0, length), slot(1, length)], np.int32)))
    lengths, starts = np.array([length + 1] * 2, np.int32), np.array([0, 1, 2], np.int32)
    got = T.n(pkg.paged_attention(turned, cache, T.t(table), T.t(starts), T.t(lengths), 0.125, cap=30.0)).astype(np.float64)
    # the caches that should be there
    held = [np.stack([np.concatenate([a, b[i:i + 1]]) for i in (0, 1)]) for a, b in ((x[0], T.n(keys)), (x[1], new[1]))]  # [2, length + 1, kv, size]
    want_cache = [t.transpose(0, 2, 1, 3) for t in held]
    n = [R.quantized4(t) for t in want_cache]
    reference = [R.pack(n[0][0]), R.pack(n[1][0]), n[0][1], n[1][1]]
    want, off = R.attention(T.n(turned), reference, np.array([[0], [1]], np.int32), starts, lengths, 0.125, cap=30.0)
    assert (np.abs(got - want) <= off).all()
    back = pkg.cache_read(cache, T.t(table), T.t(np.array([0, length + 1, 2 * length + 2], np.int32)), 2 * length + 2)
    for b, (steps, scale) in zip(back, n):
        assert np.array_equal(T.n(b).reshape(2, length + 1, kv, size), (steps.astype(np.float32) * scale[..., None]).transpose(0, 2, 1, 3))


@pytest.mark.gpu
def test_refused(pkg, T):
    import torch
    m = Made(pkg, "s4", [60], [2], 4, 2, 64, 16, 6)
    f, i = lambda n: torch.zeros(n, device="cuda"), lambda n: torch.zeros(n, dtype=torch.int32, device="cuda")
    for kw in ({"cap": -1.0}, {"cap": float("nan")}, {"cap": float("inf")}, {"cap": 1e39}, {"slopes": f(3)}, {"slopes": f(4).double()}, {"slopes": f(4).cpu()}, {"slopes": f((4, 1))},
               {"prefixes": i(2)}, {"prefixes": i(1).long()}, {"prefixes": i(1).cpu()}, {"prefixes": i(1), "window": 3}, {"prefixes": i(1), "causal": False}):
        with pytest.raises(pkg.InvalidArgumentError):
            m.run(T, **kw)
    narrow = pkg.paged_cache(9, 2, 16, 40, torch.uint8)
    with pytest.raises(pkg.TfccRocmError):
        pkg.paged_attention(f((2, 4, 40)), narrow, T.t(m.table), T.t(m.starts), T.t(m.lengths), 1.0)
