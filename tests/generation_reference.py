"""Plain 64-bit forms of the operators of generation (rotary positions, paged cache, attention over it, sampling) in numpy."""
import numpy as np

EPS = 2.0 ** -24  # half a step of float32, relative


def rotary(x, positions, frequencies, interleaved, magnitude=1.0):
    part = 2 * len(frequencies)
    angle = positions.astype(np.float64)[:, None] * np.asarray(frequencies, np.float64)
    c, s = np.cos(angle)[:, None] * magnitude, np.sin(angle)[:, None] * magnitude
    y = x.astype(np.float64).copy()
    first, second = (slice(0, part, 2), slice(1, part, 2)) if interleaved else (slice(0, part // 2), slice(part // 2, part))
    a, b = y[..., first].copy(), y[..., second].copy()
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    size = np.zeros_like(y)
    size[..., first] = size[..., second] = np.abs(a) + np.abs(b)
    return y, size * magnitude


def quantized(x):
    """(integers, scales) of rows along the last axis: the definition, with the quotient in 64 bits."""
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        scale = np.abs(x).max(-1) * np.float32(1 / 127)
        good = np.isfinite(scale) & (scale > 0)
        n = np.rint(x.astype(np.float64) / np.where(good, scale, 1).astype(np.float64)[..., None])
        return np.where(good[..., None], np.clip(n, -127, 127), 0).astype(np.int8), scale.astype(np.float32)


def held(cache):
    """Keys and values of a cache (numpy arrays) as float64 [pages, heads, rows, size]."""
    x = [c.astype(np.float64) for c in cache[:2]]
    with np.errstate(invalid="ignore"):
        return [a * s.astype(np.float64)[..., None] for a, s in zip(x, cache[2:])] if len(cache) == 4 else x


def attention(q, cache, table, starts, lengths, scale, causal=True, window=0, most=None):
    """(out, how far a float32 computation may be off): NaN rows of out are not written."""
    k, v = held(cache)
    pages, heads, page_size, size = k.shape
    group = q.shape[1] // heads
    out = np.full(q.shape, np.nan)
    off = np.zeros(q.shape)
    most = table.shape[1] * page_size if most is None else most
    for i, length in enumerate(lengths):
        n = starts[i + 1] - starts[i]
        cached = max(0, min(int(length), most, table.shape[1] * page_size))
        at = np.arange(cached)
        page = table[i][at // page_size]
        there = (page >= 0) & (page < pages)
        page = np.where(there, page, 0)
        ks, vs = k[page, :, at % page_size], v[page, :, at % page_size]  # [cached, heads, size]
        value_scales = cache[3][page, :, at % page_size].astype(np.float64) if len(cache) == 4 else None
        position = (int(length) - n + np.arange(n))[:, None]
        seen = np.broadcast_to(there, (n, cached)).copy()
        if causal:
            seen &= at <= position
            if window:
                seen &= at > position - window
        seen = np.repeat(seen, group, 0)  # a row for each token and query head of the cache head
        for h in range(heads):
            rows = q[starts[i]:starts[i + 1], h * group:(h + 1) * group].astype(np.float64)
            if not rows.size:
                continue
            x, kk, vv = rows.reshape(-1, size), ks[:, h], vs[:, h]
            with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
                s = np.where(seen, x @ kk.T * scale, -np.inf)
                top = s.max(-1, keepdims=True, initial=-np.inf)
                e = np.where(seen, np.exp(s - np.where(np.isfinite(top), top, 0)), 0)
                p = np.where(seen.any(-1, keepdims=True), e / e.sum(-1, keepdims=True), 0)
                # values of keys that a row does not see are not its own, whatever they are
                odd = ~np.isfinite(vv).all(-1)
                y = p @ np.where(odd[:, None], 0, vv)
                size_of = p @ np.where(odd[:, None], 0, np.abs(vv))
                for j in np.flatnonzero(odd):
                    y = np.where(seen[:, j:j + 1], y + p[:, j:j + 1] * vv[j], y)
                # float32 sums of `size` products, one of the factors in two pieces that leave 2^-24 of it, a scale and the maximum taken
                # off; then a sum of products with weights in two such pieces
                a = np.where(seen, np.abs(x) @ np.abs(kk).T, 0).max(-1, keepdims=True, initial=0) * abs(scale)
                ds = (size + 12) * EPS * a + 4 * EPS * np.abs(np.where(seen, s, 0)).max(-1, keepdims=True, initial=0)
                rest = 0.0
                if len(cache) == 4:
                    # the pieces of a query are multiples of 2^-24 where its largest value is 2^13 or above, those of a weight times a
                    # value's scale where the largest such product of the row is 2^8 or above, or lies 2^7 below one that is and
                    # that a later step outgrew: each is off by 2^-37 and 2^-32 of the largest, also beside a key or value of zero
                    ds = ds + size * 2.0 ** -37 * np.abs(x).max(-1, keepdims=True) * np.where(seen, np.abs(kk).max(-1), 0).max(-1, keepdims=True, initial=0) * abs(scale)
                    rest = seen.sum(-1, keepdims=True) * 2.0 ** -32 * 127 * np.where(seen, p * value_scales[:, h], 0).max(-1, keepdims=True, initial=0)
                bound = (2 * ds + 48 * EPS + seen.sum(-1, keepdims=True) * EPS) * size_of + rest + 1e-37
            out[starts[i]:starts[i + 1], h * group:(h + 1) * group] = y.reshape(rows.shape)
            off[starts[i]:starts[i + 1], h * group:(h + 1) * group] = bound.reshape(rows.shape)
    return out, off


def sample(logits, random, temperature=None, top_k=None, top_p=None, min_p=None):
    """(tokens, probabilities, margins): how near, of the kept sum, a token's choice came to another one."""
    rows, length = logits.shape
    tokens, odds, margins = [], [], []
    for r in range(rows):
        x = logits[r].astype(np.float64)
        x = np.where(np.isnan(x), -np.inf, x)
        t = 1.0 if temperature is None else float(temperature[r])
        order = np.argsort(-x, kind="stable")
        top = x[order[0]]
        if top == -np.inf:
            tokens.append(-1), odds.append(0.0), margins.append(1.0)
            continue
        if not t > 0:
            tokens.append(order[0]), odds.append(1.0), margins.append(1.0)
            continue
        with np.errstate(invalid="ignore", over="ignore"):
            w = np.exp(np.where(x == top, 0.0, (x - top) / t))
        s, n, margin = w[order], length, 1.0
        if top_k is not None and 0 < top_k[r] < n:
            n = int(top_k[r])
        if top_p is not None and top_p[r] < 1:
            sums = np.cumsum(s[:n])
            goal = float(top_p[r]) * sums[-1]
            n = max(1, 1 + int((sums[:-1] < goal).sum()))
            margin = min(margin, np.abs(sums - goal).min() / sums[-1] if goal > 0 else 1.0)
        if min_p is not None and min_p[r] > 0:
            least = min(1.0, float(min_p[r]))
            kept = int((s >= least).sum())
            margin = min(margin, np.abs(s[s != least] - least).min() if (s != least).any() else 1.0)
            n = max(1, min(n, kept))
        left = np.sort(order[:n])
        sums = np.cumsum(w[left])
        goal = min(max(float(random[r]), 0.0), 1.0) * sums[-1]
        at = min(int((sums <= goal).sum()), n - 1)
        while w[left[at]] == 0:  # a random number of 1: the last token with a weight
            at -= 1
        margin = min(margin, np.abs(sums[:-1] - goal).min() / sums[-1] if n > 1 and goal > 0 else 1.0)
        tokens.append(left[at]), odds.append(w[left[at]] / sums[-1]), margins.append(margin)
    return np.array(tokens), np.array(odds), np.array(margins)
