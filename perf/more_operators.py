"""More operators of a language model that answers token by token, as cases that can be timed: the norm in front of its products,
caches of half the size, attention whose scores are shaped, and the moves of pages that a server makes.

  norm       a row divided by its root mean square and multiplied by weights, the residual added first; as float32, or as 8-bit integers
             with a scale for each row, which is what the integer products take, and those turned back into float32 by their rows' scales.
  cache4     keys and values of new tokens written into a paged cache of 4-bit integers with a scale for each token and head, and the
             sequences read back from it.
  copy       rows of pages copied to other pages: sequences forked, and pages moved together.
  attention  a chunk of new tokens of each sequence, or a single one, over a paged cache: of 4-bit integers, or (8-bit, float32) with
             scores that are capped by a tanh, get a bias that falls with distance, or see a prefix as a whole.

Where `own` is false, run() computes them with elementary torch operations; where it is true it calls the package.
"""
import importlib
import math
import random

import torch

own = False

DEVICE = "cuda"


def listed():
    return [
        # the token of one user's decode step, between two products: latency only
        {"name": "norm_1x4096", "kind": "norm", "rows": 1, "width": 4096, "bits": 32, "residual": True},
        # prompts of a small model of an odd width, 8 bits for the integer products
        {"name": "norm_8bit_777x1003", "kind": "norm", "rows": 777, "width": 1003, "bits": 8, "residual": False},
        # a batch of long prompts, 8 bits for the integer products, the residual stream kept in float32
        {"name": "norm_8bit_8192x4096", "kind": "norm", "rows": 8192, "width": 4096, "bits": 8, "residual": True},
        # a few short sequences, one new token each
        {"name": "cache4_8_short", "kind": "cache4", "batch": 8, "chunk": 1, "context": 40, "kv_heads": 8, "size": 128, "page": 16},
        # prompts of a whole batch go into the cache, and their sequences come back as float32
        {"name": "cache4_16_prompts", "kind": "cache4", "batch": 16, "chunk": 2048, "context": 2048, "kv_heads": 8, "size": 128,
         "page": 32},
        # four answers to one question: its last page, half full, is copied for each of them
        {"name": "copy_4_forks", "kind": "copy", "cache": "s8", "count": 4, "whole": False, "kv_heads": 8, "size": 128, "page": 32},
        # a server moves scattered pages together
        {"name": "copy_1500_pages", "kind": "copy", "cache": "s4", "count": 1500, "whole": True, "kv_heads": 8, "size": 128, "page": 64},
        # one user, one token, a short context: latency only
        {"name": "attention4_1_token", "kind": "attention", "cache": "s4", "batch": 1, "chunk": 1, "context": 777, "heads": 12,
         "kv_heads": 12, "size": 64, "page": 16, "window": 0, "cap": 0.0, "slopes": False, "prefix": False},
        # the decode step of a busy server: ragged contexts, grouped heads
        {"name": "attention4_decode_64", "kind": "attention", "cache": "s4", "batch": 64, "chunk": 1, "context": 4096, "heads": 32,
         "kv_heads": 8, "size": 128, "page": 32, "window": 0, "cap": 0.0, "slopes": False, "prefix": False},
        # chunks of prompts over what the cache already holds of them
        {"name": "attention4_chunk", "kind": "attention", "cache": "s4", "batch": 4, "chunk": 1024, "context": 4096, "heads": 32,
         "kv_heads": 8, "size": 128, "page": 32, "window": 0, "cap": 0.0, "slopes": False, "prefix": False},
        # the decode step of a model that caps its scores, every second of whose layers has a window
        {"name": "attention_capped_decode", "kind": "attention", "cache": "s8", "batch": 32, "chunk": 1, "context": 6000, "heads": 16,
         "kv_heads": 8, "size": 256, "page": 32, "window": 4096, "cap": 50.0, "slopes": False, "prefix": False},
        # ragged prompts whose first part is seen as a whole, by heads that differ in how far they look
        {"name": "attention_biased_prefix_f32", "kind": "attention", "cache": "f32", "batch": 6, "chunk": 517, "context": 1201,
         "heads": 12, "kv_heads": 12, "size": 64, "page": 16, "window": 0, "cap": 0.0, "slopes": True, "prefix": True},
    ]


# ---- drawn cases -------------------------------------------------------------------------------------------------
def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    return rng.choice([(12, 12, 64), (16, 16, 64), (32, 8, 128), (32, 32, 128), (16, 2, 128), (8, 1, 256), (24, 4, 96),
                       (20, 5, 80), (64, 8, 128), (16, 8, 256)])


def draw(rng):
    kind = rng.choice(["norm", "cache4", "copy", "attention", "attention", "attention"])
    heads, kv_heads, size = _heads(rng)
    if kind == "norm":
        while True:
            c = {"kind": kind, "rows": _log(rng, 1, 16384), "width": _log(rng, 256, 16384), "bits": rng.choice([8, 8, 32]),
                 "residual": rng.random() < 0.6}
            if c["rows"] * c["width"] <= 8192 * 4096:
                return c
    if kind == "cache4":
        while True:
            chunk = rng.choice([1, _log(rng, 2, 2048)])
            c = {"kind": kind, "batch": _log(rng, 1, 64), "chunk": chunk, "context": chunk + rng.choice([0, _log(rng, 1, 2048)]),
                 "kv_heads": kv_heads, "size": size, "page": rng.choice([16, 32, 64, 128, 24])}
            if c["batch"] * c["context"] * kv_heads * size <= 16 * 2048 * 8 * 128 * 3 // 4:
                return c
    if kind == "copy":
        while True:
            c = {"kind": kind, "cache": rng.choice(["s4", "s8", "f32"]), "count": _log(rng, 1, 4096), "whole": rng.random() < 0.5,
                 "kv_heads": kv_heads, "size": size, "page": rng.choice([16, 32, 64, 128, 24])}
            if c["count"] * c["page"] * kv_heads * size * {"s4": 1, "s8": 2, "f32": 8}[c["cache"]] <= 1500 * 64 * 8 * 128:
                return c
    while True:
        chunk = rng.choice([1, 1, _log(rng, 2, 1024)])
        c = {"kind": kind, "cache": rng.choice(["s4", "s4", "s8", "f32"]), "batch": _log(rng, 1, 64), "chunk": chunk,
             "context": chunk + _log(rng, 1, 16384), "heads": heads, "kv_heads": kv_heads, "size": size,
             "page": rng.choice([16, 32, 64, 128, 24]), "window": rng.choice([0, 0, 0, _log(rng, 64, 4096)]),
             "cap": rng.choice([0.0, 20.0, 30.0, 50.0]), "slopes": rng.random() < 0.4, "prefix": rng.random() < 0.4}
        if c["cache"] == "s4" and rng.random() < 0.5:
            c |= {"cap": 0.0, "slopes": False, "prefix": False}
        if c["window"]:
            c["prefix"] = False
        if c["cache"] != "s4" and not (c["cap"] or c["slopes"] or c["prefix"]):
            c["cap"] = 50.0
        width = {"s4": 1, "s8": 2, "f32": 8}[c["cache"]]
        if (c["batch"] * c["context"] * kv_heads * size * width <= 192 << 20
                and c["batch"] * chunk * c["context"] * heads * size <= 4 * 1024 * 2048 * 32 * 128
                and c["batch"] * chunk * c["context"] * heads <= 1 << 29):
            return c


# ---- inputs ------------------------------------------------------------------------------------------------------
def _lengths(case):
    """Lengths of the sequences and of their chunks: ragged, the first the longest; they belong to the case, not the seed."""
    rng = random.Random(case["batch"] * 1000003 + case["context"] * 101 + case["chunk"])
    lengths, chunks = [], []
    for i in range(case["batch"]):
        chunk = case["chunk"] if i == 0 else rng.randint(max(1, case["chunk"] // 2), case["chunk"])
        chunks.append(chunk)
        lengths.append(case["context"] if i == 0 else rng.randint(max(chunk, case["context"] // 4), case["context"]))
    return lengths, chunks


def _prefixes(case, lengths):
    """How much of each sequence is seen as a whole: nothing of some, a question of others, all of a few."""
    rng = random.Random(case["batch"] * 7919 + case["context"] * 31 + case["chunk"])
    return [rng.choice([0, n, rng.randint(0, n), rng.randint(0, n)]) for n in lengths]


def _copied(case):
    """Rows of each copied page: all of them, or what a sequence's last page holds."""
    rng = random.Random(case["count"] * 1009 + case["page"])
    return [case["page"] if case["whole"] else rng.randint(1, case["page"]) for _ in range(case["count"])]


def _starts(counts):
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    return starts


def _pages(case, lengths, g):
    """A page table with the pages of all sequences mixed up, as a server's free list leaves them."""
    each = [-(-n // case["page"]) for n in lengths]
    pages = sum(each) + 3
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.zeros((len(lengths), max(each)), dtype=torch.int32)
    at = 0
    for i, n in enumerate(each):
        table[i, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    return pages, table


def _cache(case, kind, pages, g):
    shape = (pages, case["kv_heads"], case["page"], case["size"])
    if kind == "f32":
        return tuple(torch.randn(shape, device=DEVICE, generator=g) for _ in range(2))
    most = 127 if kind == "s8" else 7
    values = [torch.randint(-most, most + 1, shape, device=DEVICE, generator=g, dtype=torch.int8) for _ in range(2)]
    scales = [(torch.rand(shape[:3], device=DEVICE, generator=g) * 0.02 + 0.015) * (127 // most) for _ in range(2)]
    if kind == "s4":  # two to a byte, the first in the low half
        values = [((v[..., 0::2] & 15) | (v[..., 1::2] << 4)).view(torch.uint8) for v in values]
    return (*values, *scales)


def prepare(case, seed):
    g = torch.Generator(DEVICE).manual_seed(seed)
    h = torch.Generator().manual_seed(seed)
    state = {"case": case}
    if case["kind"] == "norm":
        shape = (case["rows"], case["width"])
        # a few columns of a model's residual stream are far larger than the others
        column = torch.where(torch.rand((case["width"],), device=DEVICE, generator=g) < 0.01, 20.0, 1.0)
        state["x"] = torch.randn(shape, device=DEVICE, generator=g)
        state["residual"] = torch.randn(shape, device=DEVICE, generator=g) * column if case["residual"] else None
        state["weight"] = torch.rand((case["width"],), device=DEVICE, generator=g) + 0.5
        state["eps"] = 1e-6
        return state
    if case["kind"] == "copy":
        count = case["count"]
        pages = 2 * count + 5
        state["cache"] = _cache(case, case["cache"], pages, g)
        order = torch.randperm(pages, generator=h)
        fork = not case["whole"] and count > 1  # several copies of one page among those of others
        sources = order[:count] if not fork else order[torch.randint(0, max(1, count // 2), (count,), generator=h)]
        state["sources"] = (sources * case["page"]).to(DEVICE)  # the slots of the first rows
        state["destinations"] = (order[count:2 * count] * case["page"]).to(DEVICE)
        state["rows"] = torch.tensor(_copied(case), dtype=torch.int32, device=DEVICE)
        return state
    lengths, chunks = _lengths(case)
    pages, table = _pages(case, lengths, h)
    state["cache"] = _cache(case, case.get("cache", "s4"), pages, g)
    state["table"] = table.to(DEVICE)
    state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=DEVICE)
    state["chunks"] = torch.tensor(chunks, dtype=torch.int32, device=DEVICE)
    state["longest"], state["most"], state["tokens"] = max(lengths), max(chunks), sum(chunks)
    if case["kind"] == "cache4":
        shape = (state["tokens"], case["kv_heads"], case["size"])
        state["k"] = torch.randn(shape, device=DEVICE, generator=g)
        state["v"] = torch.randn(shape, device=DEVICE, generator=g)
        at = torch.cat([torch.arange(n - c, n) for n, c in zip(lengths, chunks)])
        row = torch.cat([torch.full((c,), i) for i, c in enumerate(chunks)])
        slots = table[row, at // case["page"]].long() * case["page"] + at % case["page"]
        state["slots"] = slots.to(DEVICE)
        state["all"] = sum(lengths)
        state["starts"] = torch.tensor(_starts(lengths), dtype=torch.int32, device=DEVICE)
        return state
    # scores spread over what a cap bends
    state["q"] = torch.randn((state["tokens"], case["heads"], case["size"]), device=DEVICE, generator=g) * (4.0 if case["cap"] else 1.0)
    state["starts"] = torch.tensor(_starts(chunks), dtype=torch.int32, device=DEVICE)
    state["scale"] = case["size"] ** -0.5
    state["slopes"] = state["prefixes"] = None
    if case["slopes"]:  # a geometric series over the heads
        state["slopes"] = torch.tensor([2.0 ** (-8.0 * (i + 1) / case["heads"]) for i in range(case["heads"])], device=DEVICE)
    if case["prefix"]:
        state["prefixes"] = torch.tensor(_prefixes(case, lengths), dtype=torch.int32, device=DEVICE)
    return state


# ---- the plain forms ---------------------------------------------------------------------------------------------
def _plain_norm(s):
    c = s["case"]
    held = s["x"] if s["residual"] is None else s["x"] + s["residual"]
    inverse = (held.square().mean(-1, keepdim=True) + s["eps"]).rsqrt()
    if c["bits"] == 32:
        out = (held * inverse * s["weight"],)
    else:
        # 64 bits: which integer a value goes to is decided at borders that float32 may round onto
        wide = held.double() * s["weight"].double()
        top = wide.abs().amax(-1, keepdim=True)
        steps = (wide * 127.0 / top).round()
        scale = (top * inverse.double() / 127.0).float()
        out = steps.float() * scale, (steps.int() + 128).sum(-1, dtype=torch.int32)
    return (*out, held) if c["residual"] else out


def _plain_halves(x):
    """[..., size / 2] bytes as [..., size] integers of 4 bits."""
    signed = x.view(torch.int8)
    return torch.stack(((signed << 4) >> 4, signed >> 4), dim=-1).flatten(-2)


def _plain_quantized(x):
    scale = x.abs().amax(-1) / 7.0
    # 64 bits: which integer a value goes to is decided at borders that a float32 quotient may round onto
    steps = (x.double() / scale.double().clamp_min(1e-300)[..., None]).round().to(torch.int8)
    return ((steps[..., 0::2] & 15) | (steps[..., 1::2] << 4)).view(torch.uint8), scale


def _plain_cache4(s):
    c, cache = s["case"], s["cache"]
    page, inside = s["slots"] // c["page"], s["slots"] % c["page"]
    steps, scale = _plain_quantized(s["k"])
    cache[0][page, :, inside], cache[2][page, :, inside] = steps, scale
    steps, scale = _plain_quantized(s["v"])
    cache[1][page, :, inside], cache[3][page, :, inside] = steps, scale
    at = torch.arange(s["all"], device=DEVICE)
    row = torch.searchsorted(s["starts"][1:].contiguous(), at, right=True)
    at = at - s["starts"][row]
    page, inside = s["table"][row, at // c["page"]].long(), at % c["page"]
    return tuple(_plain_halves(cache[held][page, :, inside]).float() * cache[2 + held][page, :, inside][..., None] for held in (0, 1))


def _plain_copy(s):
    step = torch.arange(s["case"]["page"], device=DEVICE)
    wanted = step < s["rows"][:, None]
    source, destination = (s["sources"][:, None] + step)[wanted], (s["destinations"][:, None] + step)[wanted]
    page = s["case"]["page"]
    return tuple(t.transpose(1, 2).index_put_((destination // page, destination % page),
                                              t.transpose(1, 2)[source // page, source % page]).transpose(1, 2) for t in s["cache"])


def _plain_gathered(s, held):
    """[batch, kv_heads, longest padded to pages, size] of what the cache holds."""
    c, cache = s["case"], s["cache"]
    x = cache[held][s["table"].long()]
    x = (_plain_halves(x) if c["cache"] == "s4" else x).float()
    if c["cache"] != "f32":
        x = x * cache[2 + held][s["table"].long()][..., None]
    return x.transpose(1, 2).flatten(2, 3)


def _plain_attention(s):
    c = s["case"]
    batch, most, group = c["batch"], s["most"], c["heads"] // c["kv_heads"]
    keys, values = _plain_gathered(s, 0), _plain_gathered(s, 1)
    longest = keys.shape[2]
    step = torch.arange(most, device=DEVICE)
    token = (s["starts"][:-1, None] + step).clamp_max(s["tokens"] - 1).long()
    q = s["q"][token]  # [batch, most, heads, size]
    q = q.view(batch, most, c["kv_heads"], group, c["size"]).permute(0, 2, 3, 1, 4).flatten(2, 3)
    scores = torch.matmul(q, keys.transpose(2, 3).contiguous()) * s["scale"]
    scores = scores.view(batch, c["kv_heads"], group, most, longest)
    at = (s["lengths"] - s["chunks"])[:, None] + step  # the position of each new token
    key = torch.arange(longest, device=DEVICE)
    if c["cap"]:
        scores = torch.tanh(scores / c["cap"]) * c["cap"]
    if c["slopes"]:
        distance = (at[..., None] - key).abs().float()
        scores = scores - s["slopes"].view(c["kv_heads"], group, 1, 1) * distance[:, None, None]
    seen = key <= at[..., None]
    if c["window"]:
        seen &= key > at[..., None] - c["window"]
    if c["prefix"]:
        seen |= key < s["prefixes"][:, None, None]
    seen &= key < s["lengths"][:, None, None]
    scores = scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = (scores - top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights.flatten(2, 3), values).view(batch, c["kv_heads"], group, most, c["size"])
    out = torch.where(total > 0, out / total, 0.0)
    out = out.permute(0, 3, 1, 2, 4).reshape(batch, most, c["heads"], c["size"])
    return out[step < s["chunks"][:, None]]


def run(state):
    c = state["case"]
    if own:
        tfcc = importlib.import_module("wechat-tfcc_amd")
        if c["kind"] == "norm" and c["bits"] == 32:
            out, held = tfcc.rms_norm(state["x"], state["weight"], state["eps"], residual=state["residual"])
            return (out, held) if c["residual"] else (out,)
        if c["kind"] == "norm":
            steps, scales, sums, held = tfcc.rms_norm_quantized(state["x"], state["weight"], state["eps"], residual=state["residual"])
            back = tfcc.dequantize_rows(steps, scales, offset=128)
            return (back, sums, held) if c["residual"] else (back, sums)
        if c["kind"] == "cache4":
            tfcc.cache_write(state["cache"], state["k"], state["v"], state["slots"])
            return tfcc.cache_read(state["cache"], state["table"], state["starts"], state["all"])
        if c["kind"] == "copy":
            tfcc.cache_copy(state["cache"], state["sources"], state["destinations"], state["rows"])
            return state["cache"]
        return tfcc.paged_attention(state["q"], state["cache"], state["table"], state["starts"], state["lengths"], state["scale"],
                                    window=c["window"], max_length=state["longest"], cap=c["cap"], slopes=state["slopes"],
                                    prefixes=state["prefixes"])
    if c["kind"] == "norm":
        return _plain_norm(state)
    if c["kind"] == "cache4":
        return _plain_cache4(state)
    if c["kind"] == "copy":
        return _plain_copy(state)
    return _plain_attention(state)


# ---- what a pass cannot do without -------------------------------------------------------------------------------
def _row_bytes(kind, size):
    return {"s4": size // 2 + 4, "s8": size + 4, "f32": 4 * size}[kind]


def work(case):
    if case["kind"] == "norm":
        values = case["rows"] * case["width"]
        moved = (4 + (8 if case["residual"] else 0) + (4 if case["bits"] == 32 else 6)) * values
        return {"bytes": moved + 4 * case["width"] + (8 * case["rows"] if case["bits"] == 8 else 0), "flops": 6 * values}
    if case["kind"] == "copy":
        rows = sum(_copied(case)) * case["kv_heads"]
        return {"bytes": 4 * rows * _row_bytes(case["cache"], case["size"]) + 20 * case["count"], "flops": 0}
    lengths, chunks = _lengths(case)
    row = case["kv_heads"] * _row_bytes(case.get("cache", "s4"), case["size"])
    if case["kind"] == "cache4":
        new, held, wide = sum(chunks), sum(lengths), case["kv_heads"] * case["size"] * 4
        return {"bytes": 2 * (new * wide + new * row + held * row + held * wide) + 8 * new,
                "flops": 2 * case["kv_heads"] * case["size"] * (3 * new + held)}
    used, pairs = 0, 0
    for n, c, whole in zip(lengths, chunks, _prefixes(case, lengths) if case["prefix"] else [0] * len(lengths)):
        first = n - c
        w = case["window"] or n
        used += n - max(0, first + 1 - w)
        if whole > first:  # tokens inside the prefix see all of it
            inside = min(c, whole - first)
            pairs += inside * whole + (c - inside) * whole + (c - inside) * (c - inside + 1) // 2
            continue
        short = max(0, min(c, w - 1 - first))  # tokens whose window is not full yet
        pairs += short * first + short * (short + 1) // 2 + (c - short) * w
    return {"bytes": 2 * used * row + 8 * sum(chunks) * case["heads"] * case["size"],
            "flops": 4 * pairs * case["heads"] * case["size"]}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------
def _exact_norm(case, s):
    x = (s["x"] if s["residual"] is None else torch.add(s["x"], s["residual"])).double()  # the sum is held as float32
    y = x / torch.sqrt((x * x).sum(1) / case["width"] + s["eps"])[:, None] * s["weight"].double()
    got = [y]
    if case["bits"] == 8:
        step = y.abs().max(1).values / 127.0
        n = torch.round((x * s["weight"].double()) / (x * s["weight"].double()).abs().max(1).values[:, None] * 127.0)
        got = [n * step[:, None], (n + 128.0).sum(1).int()]
    return tuple(got + ([x] if case["residual"] else []))


def _exact_integers(x):
    """4-bit integers of bytes, by arithmetic: the low half first, 8 to 15 standing for -8 to -1."""
    byte = x.to(torch.int64)
    low = byte.remainder(16)
    both = torch.empty((*x.shape[:-1], 2 * x.shape[-1]), dtype=torch.float64, device=x.device)
    both[..., ::2] = low - 16 * (low > 7)
    high = torch.div(byte, 16, rounding_mode="floor")
    both[..., 1::2] = high - 16 * (high > 7)
    return both


def _exact_rows(s, i, n):
    """Which page and which row of it hold the first n tokens of sequence i."""
    at = torch.arange(n, device=DEVICE)
    return s["table"][i].long()[torch.div(at, s["case"]["page"], rounding_mode="floor")], at.remainder(s["case"]["page"])


def _exact_held(s, held, page, inside):
    x, kind = s["cache"][held][page, :, inside], s["case"]["cache"]
    x = _exact_integers(x) if kind == "s4" else x.double()
    return x if kind == "f32" else x * s["cache"][held + 2][page, :, inside].double().unsqueeze(-1)


def _exact_attention(case, s):
    group, out, starts = case["heads"] // case["kv_heads"], [], s["starts"].tolist()
    whole = s["prefixes"].tolist() if case["prefix"] else [0] * case["batch"]
    for i, n in enumerate(s["lengths"].tolist()):
        page, inside = _exact_rows(s, i, n)
        k, v = (_exact_held(s, held, page, inside).transpose(0, 1).repeat_interleave(group, 0) for held in (0, 1))
        q = s["q"][starts[i]:starts[i + 1]].double().transpose(0, 1)
        m = q.shape[1]
        seen = torch.ones(m, n, dtype=torch.bool, device=DEVICE).tril(n - m)
        if case["window"]:
            seen &= torch.ones(m, n, dtype=torch.bool, device=DEVICE).triu(n - m - case["window"] + 1)
        seen[:, :whole[i]] = True
        far = torch.arange(n - m, n, device=DEVICE, dtype=torch.float64)[:, None] - torch.arange(n, device=DEVICE, dtype=torch.float64)
        parts = []
        for h in range(0, case["heads"], 4):  # a few heads at a time
            x = torch.bmm(q[h:h + 4], k[h:h + 4].transpose(1, 2).contiguous()) / math.sqrt(case["size"])
            if case["cap"]:
                x = case["cap"] * (1.0 - 2.0 / (torch.exp(2.0 * x / case["cap"]) + 1.0))
            if case["slopes"]:
                x = x - far.abs() * s["slopes"][h:h + 4].double()[:, None, None]
            x = torch.log_softmax(x.masked_fill(~seen, -math.inf), -1).exp()
            parts.append(torch.bmm(x, v[h:h + 4].contiguous()))
        out.append(torch.cat(parts).transpose(0, 1))
    return torch.cat(out)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "norm":
        return _exact_norm(case, s)
    if case["kind"] == "cache4":
        back = []
        for held, new in ((0, s["k"]), (1, s["v"])):
            pool = _exact_integers(s["cache"][held]) * s["cache"][held + 2].double().unsqueeze(-1)
            step = (new.abs().max(-1, keepdim=True).values / 7.0).double()  # held as float32
            flat = pool.transpose(1, 2).reshape(-1, case["kv_heads"], case["size"])
            flat[s["slots"]] = torch.round(new.double() / step) * step
            at = [p * case["page"] + o for p, o in (_exact_rows(s, i, n) for i, n in enumerate(s["lengths"].tolist()))]
            back.append(flat[torch.cat(at)])
        return tuple(back)
    if case["kind"] == "copy":
        got = []
        for t in s["cache"]:
            after = t.double() if t.dtype == torch.float32 else t.clone()
            for a, b, n in zip(s["sources"].tolist(), s["destinations"].tolist(), s["rows"].tolist()):
                after[b // case["page"], :, :n] = t[a // case["page"], :, :n]
            got.append(after)
        return tuple(got)
    return _exact_attention(case, s)
