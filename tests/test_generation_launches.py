"""Calls of more workgroups than one launch takes, 2^32 threads, are refused before anything is launched.  On the CPU: complete but for one argument, so
that none can run."""
import ctypes as C

import pytest

WIDTHS = [(8, 28), (64, 28), (72, 27), (128, 27), (136, 26), (256, 26)]


def said(pkg, status):
    assert status == 1
    return pkg.lib().tfcc_rocm_last_error_string()


@pytest.mark.parametrize("tokens,fits", [((1 << 24) - 1, True), (1 << 24, False), (0xffffffff, False)])
def test_rotary(pkg, tokens, fits):
    d = pkg.RotaryDesc()
    d.size, d.part, d.tokens, d.position_type = 64, 64, tokens, pkg.S32
    d.heads[0] = 1
    text = said(pkg, pkg.lib().tfcc_rocm_rotary_f32(None, C.byref(d)))
    assert (b"null argument" in text) if fits else (b"tokens" in text)


@pytest.mark.parametrize("size,bits", WIDTHS)
@pytest.mark.parametrize("heads", [1, 8])
def test_cache_write(pkg, size, bits, heads):
    c = pkg.PagedCache()
    c.keys = c.values = c.key_scales = c.value_scales = 4096
    c.type, c.pages, c.heads, c.page_size, c.size, c.head_stride, c.scale_head_stride = pkg.S8, 1, heads, 1, size, size, 1
    for tokens, fits in (((1 << bits) // heads - 16, True), ((1 << bits) // heads, False), (0xffffffff, False)):
        text = said(pkg, pkg.lib().tfcc_rocm_cache_write(None, C.byref(c), None, 0, 0, 64, 0, 0, tokens, 64, pkg.S32))
        assert (b"null argument" in text) if fits else (b"tokens of" in text), (tokens, text)


@pytest.mark.parametrize("tokens,fits", [((1 << 26) - 4, True), ((1 << 26) - 3, False), (0xffffffff, False)])
def test_cache_read(pkg, tokens, fits):
    c = pkg.PagedCache()
    c.keys = c.values = c.key_scales = c.value_scales = 4096
    c.type, c.pages, c.heads, c.page_size, c.size = pkg.S8, 1, 1, 1, 64
    text = said(pkg, pkg.lib().tfcc_rocm_cache_read(None, C.byref(c), 64, 0, 1, 1, None, tokens, 64, 64))
    assert (b"null argument" in text) if fits else (b"tokens of" in text)


@pytest.mark.gpu
def test_reads_and_writes_at_the_ends(pkg, T):
    """The last token of the largest reads and writes that a launch takes, of heads of four values."""
    import torch
    tokens = (1 << 26) - 4
    cache = pkg.paged_cache(4, 1, 16, 4, torch.float32)
    x = torch.arange(64 * 4, device="cuda", dtype=torch.float32).view(64, 1, 4)
    pkg.cache_write(cache, x, -x, T.t(list(range(64))))
    width = -(-tokens // 16)
    table = (torch.arange(width, device="cuda", dtype=torch.int32) % 4)[None]
    keys, values = pkg.cache_read(cache, table, torch.tensor([0, tokens], dtype=torch.int32, device="cuda"), tokens)
    at = torch.arange(tokens, device="cuda")
    assert torch.equal(keys[:, 0, 0], (at % 64 * 4).float()) and torch.equal(values, -keys)
    # all but the first and the last tokens are padding
    tokens = (1 << 28) - 16
    slots = torch.full((tokens,), -1, dtype=torch.int32, device="cuda")
    slots[0], slots[-1] = 5, 63
    new = x[:1].expand(tokens, 1, 4) + 0
    new[-1] = 7
    pkg.cache_write(cache, new, new, slots)
    want = x.clone()
    want[5], want[63] = x[0], 7
    assert torch.equal(cache[0].view(64, 1, 4), want)
