"""Attention over a paged cache by wide tiles of rows, with the keys in one piece and in two, and steps that hold single tokens beside prompts' chunks.  Each
case names the tile and the pieces that it is about, which is checked without a GPU: a rule that moves does not take a test away unseen."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

import generation_reference as R
from conftest import rel_fro
from test_gpu_paged_attention import Made

HOST = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "wechat-tfcc_amd", "host")

# kind, lengths, chunks, heads, kv heads, size, page, more, rows of a tile, pieces
CASES = [
    ("s8", [2500, 2100], [500, 524], 32, 8, 128, 16, {}, 128, 2),
    ("s8", [2600, 300], [700, 330], 32, 8, 64, 20, {}, 128, 2),               # pages that end inside a step; a piece without keys
    ("s8", [2700, 2048], [640, 390], 32, 8, 80, 48, {}, 128, 2),
    ("s8", [4000], [1030], 32, 8, 128, 16, {"window": 2500}, 128, 2),
    ("s8", [2300, 2200], [520, 510], 32, 8, 96, 16, {"causal": False}, 128, 2),
    ("s8", [2600, 2300], [520, 510], 32, 8, 32, 24, {"max_length": 2100}, 128, 2),
    ("s8", [2050, 900, 2200], [1, 1020, 40], 32, 8, 128, 32, {}, 128, 2),      # chunks of one and of many tokens
    ("s8", [2300, 2100], [300, 200], 64, 16, 256, 16, {}, 128, 1),
    # one long prompt and single tokens
    ("s8", [1100] + list(range(500, 1430, 30)), [1100] + [1] * 31, 32, 8, 128, 16, {}, 128, 1),
    ("s8", list(range(400, 1330, 30)) + [1300], [1] * 31 + [1100], 32, 8, 64, 20, {"window": 700}, 128, 1),
    ("s8", [2300] + list(range(1800, 2220, 30)), [1100] + [1] * 14, 32, 8, 128, 16, {}, 128, 2),
    ("s8", [900] * 16 + [300], [1] * 16 + [100], 32, 8, 128, 16, {}, 16, 1),
    ("f32", [1100] + list(range(500, 1430, 30)), [1100] + [1] * 31, 32, 8, 128, 16, {}, 256, 1),
    ("f32", list(range(400, 1330, 30)) + [1300], [1] * 31 + [1100], 32, 8, 64, 20, {"window": 700}, 128, 1),
    ("f32", [2300] + list(range(1800, 2220, 30)), [1100] + [1] * 14, 16, 2, 128, 16, {}, 256, 2),
    ("f32", [2500, 2100], [300, 124], 32, 8, 128, 16, {}, 256, 4),
    ("f32", [900] * 16 + [300], [1] * 16 + [100], 32, 8, 128, 16, {}, 16, 1),
]


def planned(pkg, kind, lengths, chunks, heads, kv, size, page, more):
    """(rows of a tile, pieces) of a call of Made: its table has a page more than the longest sequence.  The pieces are those that the library asks a
    workspace for."""
    width = max(max(1, -(-n // page)) for n in lengths) + 1
    d = pkg.PagedAttentionDesc()
    c = d.cache
    c.keys = c.values = c.key_scales = c.value_scales = 4096
    c.type, c.pages, c.heads, c.page_size, c.size = pkg.S8 if kind == "s8" else pkg.F32, sum(-(-n // page) for n in lengths) + 2, kv, page, size
    c.row_stride, c.head_stride, c.page_stride = size, size * page, size * page * kv
    c.scale_row_stride, c.scale_head_stride, c.scale_page_stride = 1, page, page * kv
    d.heads, d.tokens, d.batch, d.table_width, d.causal = heads, sum(chunks), len(lengths), width, int(more.get("causal", True))
    d.max_length, d.window = more.get("max_length", 0), more.get("window", 0)
    needs = pkg.lib().tfcc_rocm_paged_attention_workspace(C.byref(d))
    most = min(d.max_length or width * page, width * page)
    wide = 0 if page < 16 or page % 4 else (128 if size % 16 == 0 else 0) if kind == "s8" else 128 if size <= 64 else 256 if size <= 128 else 0
    driver = os.path.join(HOST, "build", "paged_attention_plan_print")
    subprocess.check_call(["make", "-s", "-C", HOST, "build/paged_attention_plan_print"])
    line = (d.tokens, d.batch, heads // kv, kv, size, most, d.causal, d.window, wide, int(kind == "f32"))
    rows, _, pieces, _ = map(int, subprocess.run([driver], input=" ".join(map(str, line)), stdout=subprocess.PIPE, text=True, timeout=60).stdout.split())
    assert needs == (0 if pieces == 1 else pieces * d.tokens * heads * (size + 2) * 4)
    return rows, pieces


@pytest.mark.parametrize("case", range(len(CASES)))
def test_planned(pkg, case):
    assert planned(pkg, *CASES[case][:8]) == CASES[case][8:]


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(CASES)))
def test_against_the_definition(pkg, T, case):
    kind, lengths, chunks, heads, kv, size, page, more = CASES[case][:8]
    Made(pkg, kind, lengths, chunks, heads, kv, size, page, 200 + case).check(T, **more)


TWO = CASES[1][:7]  # int8, two pieces, the second sequence's second piece without keys


@pytest.mark.gpu
def test_pages_outside_the_cache_in_pieces(pkg, T):
    m = Made(pkg, *TWO, 31)
    m.table[0, ::5] = -1
    m.table[1, 3:] = len(m.cache[0])
    m.check(T)
    m.table[0, : m.table.shape[1] // 2 + 4] = -1  # a first piece without a key that is there
    m.check(T)


@pytest.mark.gpu
def test_rows_behind_the_last_sequence_in_pieces(pkg, T):
    import torch
    m = Made(pkg, *TWO, 32)
    n = int(m.starts[-1])
    want = m.run(T)
    m.q = np.concatenate([m.q, m.q[:40], m.q[:1] * np.nan])
    out = torch.full(m.q.shape, 3.25, device="cuda")
    m.run(T, out=out)
    assert torch.equal(out[:n], want) and bool((out[n:] == 3.25).all())


@pytest.mark.gpu
def test_queries_and_scales_that_are_not_finite_in_pieces(pkg, T):
    m = Made(pkg, *TWO, 33)
    clean = T.n(m.run(T)).copy()
    for value in (np.nan, np.inf):
        m.q[699, 5, 3] = value
        got = T.n(m.run(T))
        mine = np.zeros(got.shape, bool)
        mine[699, 5] = True
        assert np.isnan(got[mine]).all() and np.array_equal(got[~mine], clean[~mine])
    m.q[699, 5] = 0
    clean = T.n(m.run(T)).copy()
    last = m.lengths[0] - 1  # seen by one token
    for scales, value in ((3, np.inf), (2, np.nan)):
        before = m.cache[scales][m.table[0, last // 20], 2, last % 20]
        m.cache[scales][m.table[0, last // 20], 2, last % 20] = value
        got = T.n(m.run(T))
        mine = np.zeros(got.shape, bool)
        mine[699, 8:12] = True
        assert np.isnan(got[mine]).all() and np.array_equal(got[~mine], clean[~mine])
        m.cache[scales][m.table[0, last // 20], 2, last % 20] = before


# Frames that move, in one piece and in two: int8, rows of a tile 128
MOVING = [([1100], [160], 128, 128, 64, 16, {}, 128, 1), ([2500, 2100], [500, 524], 32, 8, 64, 16, {}, 128, 2)]


@pytest.mark.parametrize("case", range(len(MOVING)))
def test_planned_moving(pkg, case):
    assert planned(pkg, "s8", *MOVING[case][:7]) == MOVING[case][7:]


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(MOVING)))
@pytest.mark.parametrize("order", [1, -1])
def test_scales_further_apart_than_float32_exponents(pkg, T, case, order):
    """The weights of keys whose values are small beside the others' count in full, whichever come first."""
    m = Made(pkg, "s8", *MOVING[case][:6], 34)
    for i, length in enumerate(m.lengths):
        at = np.arange(length)
        scales = np.where((at < length * 3 // 4)[::order], np.float32(1e-25), np.float32(1e25)).astype(np.float32)
        m.cache[3][m.table[i][at // 16], :, at % 16] = scales[:, None]
    m.check(T)


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(MOVING)))
def test_scales_of_all_sizes(pkg, T, case):
    """Rows of values from 10^-20 to 10^20, zeros among them, and queries likewise."""
    m = Made(pkg, "s8", *MOVING[case][:6], 35)
    m.cache[3][:] = np.exp(m.rng.normal(size=m.cache[3].shape) * 15).astype(np.float32)
    m.cache[3][m.rng.random(m.cache[3].shape) < 0.2] = 0
    m.cache[2][m.rng.random(m.cache[2].shape) < 0.2] = 0
    m.q[1] *= 1e-25
    m.q[2] = 0
    m.check(T)
    m.cache[3][:] = 0
    assert not T.n(m.run(T)).any()


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(MOVING)))
def test_large_scores(pkg, T, case):
    m = Made(pkg, "s8", *MOVING[case][:6], 36)
    m.scale *= 100
    m.check(T)
