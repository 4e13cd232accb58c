"""Attention over a paged cache at the ends of what a call may hold: many rows, many workgroups."""
import ctypes as C

import numpy as np
import pytest

import generation_reference as R


def described(pkg, tokens, heads, kv, batch, size=64, page=16, width=200, most=0, kind=None):
    """A call that is complete but for its starts, so that it cannot run: what is wrong with its sizes is said before that."""
    d = pkg.PagedAttentionDesc()
    c = d.cache
    c.keys = c.values = c.key_scales = c.value_scales = 4096
    c.type, c.pages, c.heads, c.page_size, c.size = pkg.S8 if kind is None else kind, 200, kv, page, size
    c.row_stride, c.scale_row_stride = size, 1
    d.heads, d.tokens, d.batch, d.table_width, d.causal, d.max_length = heads, tokens, batch, width, 1, most
    d.q = d.out = d.lengths = d.table = d.workspace = 4096
    d.workspace_bytes = 1 << 62
    return d


@pytest.mark.parametrize("tokens,heads,kv,batch,fits", [
    (131071, 64, 8, 1, True), (131073, 64, 8, 1, True), (1 << 20, 128, 8, 64, True),  # 2^23 rows and more: nothing is joined
    ((1 << 24) - 16, 1, 1, 1 << 30, True), ((1 << 20) - 1, 16, 16, 1 << 20, True), (1 << 20, 16, 16, 1 << 20, False),  # a workgroup to a row
    (1 << 25, 64, 8, 1, False), ((1 << 25) - 4, 64, 1, 1, True), ((1 << 25) - 1, 64, 64, 1, False)])  # 2^24 - 2 and 2^24 tiles of 128 rows
def test_number_of_workgroups(pkg, tokens, heads, kv, batch, fits):
    lib = pkg.lib()
    d = described(pkg, tokens, heads, kv, batch)
    assert lib.tfcc_rocm_paged_attention_f32(None, C.byref(d)) == 1
    said = lib.tfcc_rocm_last_error_string()
    assert (b"null argument" in said) if fits else (b"workgroups" in said or b"tokens of" in said), said
    assert lib.tfcc_rocm_paged_attention_workspace(C.byref(d)) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("size", [8, 16])
def test_more_than_two_to_the_23rd_rows(pkg, T, size):
    """131073 tokens of 64 heads over a few keys: the rows are those of calls with fewer."""
    import torch
    tokens, heads = 131073, 64
    rng = np.random.default_rng(size)
    cache = pkg.paged_cache(2, 1, 16, size)
    for t in cache[:2]:
        t.copy_(T.t(rng.integers(-127, 128, tuple(t.shape), dtype=np.int8)))
    for t in cache[2:]:
        t.copy_(T.t((rng.random(tuple(t.shape)) * 0.02 + 0.01).astype(np.float32)))
    table, lengths = np.array([[1, 0]], np.int32), np.array([20], np.int32)
    g = torch.Generator("cuda").manual_seed(size)
    q = torch.randn((tokens, heads, size), device="cuda", generator=g)
    run = lambda q: pkg.paged_attention(q, cache, T.t(table), T.t(np.array([0, len(q)], np.int32)), T.t(lengths), size ** -0.5, causal=False)
    whole = run(q)
    for first in range(0, tokens, 30000):
        assert torch.equal(whole[first:first + 30000], run(q[first:first + 30000]))
    some = np.r_[:40, tokens - 40:tokens]
    want, off = R.attention(T.n(q[torch.from_numpy(some).cuda()]), [T.n(t) for t in cache], table, [0, len(some)], lengths, size ** -0.5, causal=False)
    assert (np.abs(T.n(whole[torch.from_numpy(some).cuda()]) - want) <= off).all()


@pytest.mark.gpu
def test_a_workgroup_to_each_of_four_million_rows(pkg, T):
    """65536 single tokens of 64 heads with keys of their own: each gets the one value that its sequence holds."""
    import torch
    tokens, heads, size = 65536, 64, 8
    g = torch.Generator("cuda").manual_seed(1)
    cache = pkg.paged_cache(16, heads, 1, size)
    for t in cache[:2]:
        t.copy_(torch.randint(-127, 128, t.shape, device="cuda", generator=g, dtype=torch.int8))
    for t in cache[2:]:
        t.copy_(torch.rand(t.shape, device="cuda", generator=g) + 0.5)
    table = torch.randint(0, 16, (tokens, 1), device="cuda", generator=g, dtype=torch.int32)
    q = torch.randn((tokens, heads, size), device="cuda", generator=g)
    out = pkg.paged_attention(q, cache, table, torch.arange(tokens + 1, dtype=torch.int32, device="cuda"), torch.ones(tokens, dtype=torch.int32, device="cuda"), 1.0)
    held = cache[1][:, :, 0].double() * cache[3][:, :, 0, None].double()
    want = held[table[:, 0].long()]
    # one weight w: w * scale in two pieces (2^-23 of it), the product, the sum of one weight and the quotient
    assert bool(((out.double() - want).abs() <= 6 * 2.0 ** -23 * want.abs()).all())
