"""Plain 64-bit forms in numpy of the norm with 8-bit output, of caches of 4-bit integers, of copies inside a cache, and of attention with
shaped scores over a cache of any type."""
import numpy as np

from generation_reference import EPS


def pack(n):
    """Integers from -8 to 7 along the last axis, two to a byte, the first in the low half."""
    n = n.astype(np.int64) % 16
    return (n[..., 0::2] | n[..., 1::2] << 4).astype(np.uint8)


def unpack(x):
    n = np.stack([x & 15, x >> 4], -1).reshape(*x.shape[:-1], -1).astype(np.int8)
    return np.where(n > 7, n - 16, n).astype(np.int8)


def quantized4(x):
    """(integers, scales) of rows along the last axis: the definition, with the quotient in 64 bits."""
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        scale = np.abs(x).max(-1) * np.float32(1 / 7)
        good = np.isfinite(scale) & (scale > 0)
        n = np.rint(x.astype(np.float64) / np.where(good, scale, 1).astype(np.float64)[..., None])
        return np.where(good[..., None], np.clip(n, -7, 7), 0).astype(np.int8), scale.astype(np.float32)


def held(cache):
    """Keys and values of a cache (numpy arrays) as float64 [pages, heads, rows, size]."""
    x = [(unpack(c) if c.dtype == np.uint8 else c).astype(np.float64) for c in cache[:2]]
    with np.errstate(invalid="ignore"):
        return [a * s.astype(np.float64)[..., None] for a, s in zip(x, cache[2:])] if len(cache) == 4 else x


def copied(cache, sources, destinations, rows):
    """The cache after runs of rows have been copied inside it."""
    pages, heads, page = cache[0].shape[:3]
    got = [c.copy() for c in cache]
    for i, (a, b) in enumerate(zip(sources, destinations)):
        if not (0 <= a < pages * page and 0 <= b < pages * page):
            continue
        n = page - max(a % page, b % page)
        n = n if rows is None else max(0, min(n, rows[i]))
        for c, g in zip(cache, got):
            g[b // page, :, b % page:b % page + n] = c[a // page, :, a % page:a % page + n]
    return got


def norm(x, weight, eps, residual=None):
    """(h, y, t, top): the sum in float32, the norm in 64 bits, h * weight exactly, the largest of its sizes."""
    h = x if residual is None else x + residual
    t = h.astype(np.float64) * weight.astype(np.float64)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        y = t / np.sqrt((h.astype(np.float64) ** 2).mean(-1, keepdims=True) + eps)
    return h, y, t, np.abs(t).max(-1, keepdims=True)


def norm_steps(t, top):
    """127 t / top to the nearest, ties to even, in whole numbers: t and top are multiples of one power of two."""
    out = np.zeros(t.shape, np.int64)
    for i, (row, most) in enumerate(zip(t.reshape(-1, t.shape[-1]), top.reshape(-1))):
        if most == 0:
            continue
        _, e = np.frexp(row[row != 0])
        unit = int(e.min()) - 53
        whole = [int_of(v, unit) for v in row]
        most = int_of(most, unit)
        for j, v in enumerate(whole):
            q, r = divmod(2 * 127 * abs(v) + most, 2 * most)
            if r == 0 and q % 2:
                q -= 1
            out.reshape(-1, t.shape[-1])[i, j] = q if v >= 0 else -q
    return out


def int_of(v, unit):
    """v / 2^unit, a whole number."""
    n, d = float(v).as_integer_ratio()
    shift = d.bit_length() - 1
    return n << (-unit - shift) if -unit >= shift else n >> (shift + unit)


def attention(q, cache, table, starts, lengths, scale, causal=True, window=0, most=None, cap=0.0, slopes=None, prefixes=None):
    """(out, how far a float32 computation may be off): NaN rows of out are not written."""
    k, v = held(cache)
    pages, heads, page_size, size = k.shape
    group = q.shape[1] // heads
    out, off = np.full(q.shape, np.nan), np.zeros(q.shape)
    most = table.shape[1] * page_size if most is None else most
    largest = {np.dtype(np.uint8): 8, np.dtype(np.int8): 127}.get(cache[0].dtype)
    for i, length in enumerate(lengths):
        n = starts[i + 1] - starts[i]
        cached = max(0, min(int(length), most, table.shape[1] * page_size))
        at = np.arange(cached)
        page = table[i][at // page_size]
        there = (page >= 0) & (page < pages)
        page = np.where(there, page, 0)
        ks, vs = k[page, :, at % page_size], v[page, :, at % page_size]  # [cached, heads, size]
        position = (int(length) - n + np.arange(n))[:, None]
        seen = np.ones((n, cached), bool)
        if causal:
            seen &= at <= position
            if window:
                seen &= at > position - window
            if prefixes is not None:
                seen |= at < prefixes[i]
        seen &= there
        far = np.repeat(np.abs(position - at).astype(np.float64), group, 0)
        seen = np.repeat(seen, group, 0)  # a row for each token and query head of the cache head
        for h in range(heads):
            rows = q[starts[i]:starts[i + 1], h * group:(h + 1) * group].astype(np.float64)
            if not rows.size:
                continue
            x, kk, vv = rows.reshape(-1, size), ks[:, h], vs[:, h]
            with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
                raw = x @ kk.T * scale
                s = np.tanh(raw / cap) * cap if cap else raw
                bias = 0.0
                if slopes is not None:
                    bias = np.tile(slopes[h * group:(h + 1) * group].astype(np.float64), n)[:, None] * far
                    s = s - bias
                s = np.where(seen, s, -np.inf)
                top = s.max(-1, keepdims=True, initial=-np.inf)
                e = np.where(seen, np.exp(s - np.where(np.isfinite(top), top, 0)), 0)
                p = np.where(seen.any(-1, keepdims=True), e / e.sum(-1, keepdims=True), 0)
                y, size_of = p @ vv, p @ np.abs(vv)
                # as for plain scores: float32 sums of `size` products, one of the factors in two pieces that leave 2^-24 of it, a scale; the cap's
                # tanh (a slope of one at most; formed to 8 half steps of the result), the bias and the maximum taken off
                a = np.where(seen, np.abs(x) @ np.abs(kk).T, 0).max(-1, keepdims=True, initial=0) * abs(scale)
                ds = (size + 12) * EPS * a + 4 * EPS * np.abs(np.where(seen, s, 0)).max(-1, keepdims=True, initial=0)
                ds = ds + (12 * EPS * np.minimum(a, cap) if cap else 0) + 4 * EPS * np.abs(np.where(seen, bias, 0)).max(-1, keepdims=True, initial=0)
                rest = 0.0
                if largest is not None:
                    # pieces of queries and of weights times scales are multiples of fixed steps, also beside a key or value of zero
                    ds = ds + size * 2.0 ** -37 * np.abs(x).max(-1, keepdims=True) * np.where(seen, np.abs(kk).max(-1), 0).max(-1, keepdims=True, initial=0) * abs(scale)
                    value_scales = cache[3][page, h, at % page_size].astype(np.float64)
                    rest = seen.sum(-1, keepdims=True) * 2.0 ** -32 * largest * np.where(seen, p * value_scales, 0).max(-1, keepdims=True, initial=0)
                bound = (2 * ds + 48 * EPS + seen.sum(-1, keepdims=True) * EPS) * size_of + rest + 1e-37
            out[starts[i]:starts[i + 1], h * group:(h + 1) * group] = y.reshape(rows.shape)
            off[starts[i]:starts[i + 1], h * group:(h + 1) * group] = bound.reshape(rows.shape)
    return out, off
