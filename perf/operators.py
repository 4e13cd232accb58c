"""Operators of a language model that answers token by token, as cases that can be timed: what stands between its matrix
products from the projected heads of new tokens to the token that is chosen.

  rotary     the heads of queries and keys turned by the angles of their positions: neighbouring values or halves of a head
             as pairs, the whole head or its first part, frequencies stretched for contexts longer than the trained one.
  cache      keys and values of new tokens written into a paged cache (8-bit integers with a scale for each token and head,
             or float32) and the sequences read back from it.
  attention  a chunk of new tokens of each sequence, or a single one, attending to what the paged cache holds of it.
  sample     one token for each row of logits: temperature, top-k, top-p, min-p, and a given random number.

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
        # the token of one user's decode step: latency only
        {"name": "rotary_1_token", "kind": "rotary", "tokens": 1, "heads": 32, "kv_heads": 8, "size": 128, "part": 128,
         "interleaved": False, "stretch": 1.0, "far": 4096},
        # a mid-sized batch of prompts, half of each head turned, neighbouring values as pairs
        {"name": "rotary_interleaved_777", "kind": "rotary", "tokens": 777, "heads": 12, "kv_heads": 12, "size": 64,
         "part": 32, "interleaved": True, "stretch": 1.0, "far": 2048},
        # a long prompt's chunk at positions far behind the trained length
        {"name": "rotary_4096_far", "kind": "rotary", "tokens": 4096, "heads": 32, "kv_heads": 8, "size": 128, "part": 128,
         "interleaved": False, "stretch": 8.0, "far": 1000000},
        # a few short sequences, one new token each
        {"name": "cache_8_short", "kind": "cache", "cache": "s8", "batch": 8, "chunk": 1, "context": 40, "kv_heads": 8,
         "size": 128, "page": 16},
        # prompts of a whole batch go into the cache, and their sequences come back as float32
        {"name": "cache_16_prompts", "kind": "cache", "cache": "s8", "batch": 16, "chunk": 2048, "context": 2048,
         "kv_heads": 8, "size": 128, "page": 32},
        # one user, one token, a short context: latency only
        {"name": "attention_1_token", "kind": "attention", "cache": "s8", "batch": 1, "chunk": 1, "context": 777, "heads": 12,
         "kv_heads": 12, "size": 64, "page": 16, "window": 0},
        # the decode step of a busy server: ragged contexts, grouped heads
        {"name": "attention_decode_32", "kind": "attention", "cache": "s8", "batch": 32, "chunk": 1, "context": 4096,
         "heads": 32, "kv_heads": 8, "size": 128, "page": 32, "window": 0},
        # two users with long contexts held in float32
        {"name": "attention_decode_long_f32", "kind": "attention", "cache": "f32", "batch": 2, "chunk": 1, "context": 30011,
         "heads": 32, "kv_heads": 8, "size": 128, "page": 64, "window": 0},
        # chunks of prompts over what the cache already holds of them
        {"name": "attention_chunk_s8", "kind": "attention", "cache": "s8", "batch": 4, "chunk": 1024, "context": 4096,
         "heads": 32, "kv_heads": 8, "size": 128, "page": 32, "window": 0},
        # ragged prompts of a small model with a sliding window, in float32
        {"name": "attention_chunk_f32_window", "kind": "attention", "cache": "f32", "batch": 6, "chunk": 517, "context": 1201,
         "heads": 12, "kv_heads": 12, "size": 64, "page": 16, "window": 512},
        # one user's next token
        {"name": "sample_1x32000", "kind": "sample", "rows": 1, "vocabulary": 32000, "k": True, "p": True, "min": False},
        # the next tokens of a large batch over a large vocabulary
        {"name": "sample_128x100003", "kind": "sample", "rows": 128, "vocabulary": 100003, "k": False, "p": True, "min": True},
    ]


# ---- drawn cases -------------------------------------------------------------------------------------------------
def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    return rng.choice([(12, 12, 64), (16, 16, 64), (32, 8, 128), (32, 32, 128), (16, 2, 128), (8, 1, 256), (24, 4, 96),
                       (20, 5, 80), (64, 8, 128)])


def draw(rng):
    kind = rng.choice(["rotary", "cache", "attention", "attention", "attention", "sample"])
    heads, kv_heads, size = _heads(rng)
    if kind == "rotary":
        while True:
            c = {"kind": kind, "tokens": _log(rng, 1, 8192), "heads": heads, "kv_heads": kv_heads, "size": size,
                 "part": rng.choice([size, size, size // 2, size // 4]), "interleaved": rng.random() < 0.4,
                 "stretch": rng.choice([1.0, 1.0, 4.0, 16.0]), "far": _log(rng, 512, 1000000)}
            if c["tokens"] * (heads + kv_heads) * size <= 4096 * 40 * 128:
                return c
    if kind == "cache":
        while True:
            chunk = rng.choice([1, _log(rng, 2, 2048)])
            c = {"kind": kind, "cache": rng.choice(["s8", "s8", "f32"]), "batch": _log(rng, 1, 64), "chunk": chunk,
                 "context": chunk + rng.choice([0, _log(rng, 1, 2048)]), "kv_heads": kv_heads, "size": size,
                 "page": rng.choice([16, 32, 64, 128, 24])}
            if c["batch"] * c["context"] * kv_heads * size <= 16 * 2048 * 8 * 128 * 3 // 4:
                return c
    if kind == "attention":
        while True:
            chunk = rng.choice([1, 1, _log(rng, 2, 1024)])
            c = {"kind": kind, "cache": rng.choice(["s8", "s8", "f32"]), "batch": _log(rng, 1, 64), "chunk": chunk,
                 "context": chunk + _log(rng, 1, 16384), "heads": heads, "kv_heads": kv_heads, "size": size,
                 "page": rng.choice([16, 32, 64, 128, 24]), "window": rng.choice([0, 0, 0, _log(rng, 64, 4096)])}
            width = 1 if c["cache"] == "s8" else 4
            if (c["batch"] * c["context"] * kv_heads * size * width <= 96 << 20
                    and c["batch"] * chunk * c["context"] * heads * size <= 4 * 1024 * 2048 * 32 * 128
                    and c["batch"] * chunk * c["context"] * heads <= 1 << 29):
                return c
    while True:
        c = {"kind": "sample", "rows": _log(rng, 1, 256), "vocabulary": _log(rng, 1000, 200000), "k": rng.random() < 0.5,
             "p": rng.random() < 0.7, "min": rng.random() < 0.4}
        if c["rows"] * c["vocabulary"] <= 128 * 100003:
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


def _cache(case, pages, g):
    shape = (pages, case["kv_heads"], case["page"], case["size"])
    if case["cache"] == "f32":
        return tuple(torch.randn(shape, device=DEVICE, generator=g) for _ in range(2))
    values = [torch.randint(-127, 128, shape, device=DEVICE, generator=g, dtype=torch.int8) for _ in range(2)]
    scales = [torch.rand(shape[:3], device=DEVICE, generator=g) * 0.02 + 0.015 for _ in range(2)]
    return (*values, *scales)


def prepare(case, seed):
    g = torch.Generator(DEVICE).manual_seed(seed)
    h = torch.Generator().manual_seed(seed)
    state = {"case": case}
    if case["kind"] == "rotary":
        n, part = case["tokens"], case["part"]
        f = [10000.0 ** (-2.0 * i / part) for i in range(part // 2)]
        if case["stretch"] > 1.0:  # pairs that turn less than once over a trained length of 8192 are slowed, fast ones not
            turns = [8192 * x / (2 * math.pi) for x in f]
            kept = [min(1.0, max(0.0, (t - 1.0) / 3.0)) for t in turns]
            f = [x * (r + (1.0 - r) / case["stretch"]) for x, r in zip(f, kept)]
        state["q"] = torch.randn((n, case["heads"], case["size"]), device=DEVICE, generator=g)
        state["k"] = torch.randn((n, case["kv_heads"], case["size"]), device=DEVICE, generator=g)
        state["positions"] = torch.randint(0, case["far"], (n,), device=DEVICE, generator=g, dtype=torch.int32)
        state["frequencies"] = torch.tensor(f, dtype=torch.float64, device=DEVICE)
        return state
    if case["kind"] in ("cache", "attention"):
        lengths, chunks = _lengths(case)
        pages, table = _pages(case, lengths, h)
        state["cache"] = _cache(case, pages, g)
        state["table"] = table.to(DEVICE)
        state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=DEVICE)
        state["chunks"] = torch.tensor(chunks, dtype=torch.int32, device=DEVICE)
        state["longest"], state["most"], state["tokens"] = max(lengths), max(chunks), sum(chunks)
    if case["kind"] == "cache":
        shape = (state["tokens"], case["kv_heads"], case["size"])
        state["k"] = torch.randn(shape, device=DEVICE, generator=g)
        state["v"] = torch.randn(shape, device=DEVICE, generator=g)
        at = torch.cat([torch.arange(n - c, n) for n, c in zip(lengths, chunks)])
        row = torch.cat([torch.full((c,), i) for i, c in enumerate(chunks)])
        slots = table[row, at // case["page"]].long() * case["page"] + at % case["page"]
        state["slots"] = slots.to(DEVICE)
        state["all"] = sum(lengths)
        state["starts"] = torch.tensor(_starts(lengths), dtype=torch.int32, device=DEVICE)
    if case["kind"] == "attention":
        state["q"] = torch.randn((state["tokens"], case["heads"], case["size"]), device=DEVICE, generator=g)
        state["starts"] = torch.tensor(_starts(chunks), dtype=torch.int32, device=DEVICE)
        state["scale"] = case["size"] ** -0.5
    if case["kind"] == "sample":
        n = case["rows"]
        # most of a vocabulary is far from likely, a few dozen tokens of each row are in question
        x = torch.randn((n, case["vocabulary"]), device=DEVICE, generator=g) * 2.0
        at = torch.randint(0, case["vocabulary"], (n, 40), device=DEVICE, generator=g)
        state["logits"] = x.scatter_add(1, at, torch.rand((n, 40), device=DEVICE, generator=g) * 10.0)
        state["random"] = torch.rand((n,), device=DEVICE, generator=g)
        state["temperature"] = torch.rand((n,), device=DEVICE, generator=g) * 1.0 + 0.5
        state["top_k"] = torch.randint(1, 200, (n,), device=DEVICE, generator=g, dtype=torch.int32) if case["k"] else None
        state["top_p"] = torch.rand((n,), device=DEVICE, generator=g) * 0.29 + 0.7 if case["p"] else None
        state["min_p"] = torch.rand((n,), device=DEVICE, generator=g) * 0.1 if case["min"] else None
    return state


# ---- the plain forms ---------------------------------------------------------------------------------------------
def _plain_turn(x, cos, sin, part, interleaved):
    head, rest = x[..., :part], x[..., part:]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = head[..., : part // 2], head[..., part // 2:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, rest), dim=-1)


def _plain_rotary(s):
    c = s["case"]
    angles = s["positions"].double()[:, None] * s["frequencies"][None, :]  # 64 bits: a far position has many turns
    cos, sin = angles.cos().float()[:, None, :], angles.sin().float()[:, None, :]
    return (_plain_turn(s["q"], cos, sin, c["part"], c["interleaved"]),
            _plain_turn(s["k"], cos, sin, c["part"], c["interleaved"]))


def _plain_quantized(x):
    scale = x.abs().amax(-1) / 127.0
    # 64 bits: which integer a value goes to is decided at borders that a float32 quotient may round onto
    steps = (x.double() / scale.double().clamp_min(1e-300)[..., None]).round()
    return steps.to(torch.int8), scale


def _plain_cache(s):
    c, cache = s["case"], s["cache"]
    page, inside = s["slots"] // c["page"], s["slots"] % c["page"]
    for held, new in ((0, s["k"]), (1, s["v"])):
        if c["cache"] == "s8":
            steps, scale = _plain_quantized(new)
            cache[held][page, :, inside] = steps
            cache[2 + held][page, :, inside] = scale
        else:
            cache[held][page, :, inside] = new
    at = torch.arange(s["all"], device=DEVICE)
    row = torch.searchsorted(s["starts"][1:].contiguous(), at, right=True)
    at = at - s["starts"][row]
    page, inside = s["table"][row, at // c["page"]].long(), at % c["page"]
    back = [cache[held][page, :, inside].float() for held in (0, 1)]
    if c["cache"] == "s8":
        back = [b * cache[2 + held][page, :, inside][..., None] for held, b in enumerate(back)]
    return tuple(back)


def _plain_gathered(s, held):
    """[batch, kv_heads, longest padded to pages, size] of what the cache holds."""
    c, cache = s["case"], s["cache"]
    x = cache[held][s["table"].long()].float()
    if c["cache"] == "s8":
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
    at = (s["lengths"] - s["chunks"])[:, None] + step  # the position of each new token
    key = torch.arange(longest, device=DEVICE)
    seen = key <= at[..., None]
    if c["window"]:
        seen &= key > at[..., None] - c["window"]
    seen = seen[:, None, None]
    scores = scores.view(batch, c["kv_heads"], group, most, longest).masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = (scores - top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights.flatten(2, 3), values).view(batch, c["kv_heads"], group, most, c["size"])
    out = torch.where(total > 0, out / total, 0.0)
    out = out.permute(0, 3, 1, 2, 4).reshape(batch, most, c["heads"], c["size"])
    return out[step < s["chunks"][:, None]]


def _plain_sample(s):
    # 64 bits: a token is chosen at borders between long sums
    value, order = torch.sort(s["logits"], dim=-1, descending=True, stable=True)
    weight = ((value.double() - value[:, :1].double()) / s["temperature"].double()[:, None]).exp()
    rank = torch.arange(value.shape[1], device=DEVICE)
    kept = torch.ones_like(weight, dtype=torch.bool)
    if s["top_k"] is not None:
        kept &= rank < s["top_k"][:, None]
    if s["top_p"] is not None:
        before = (weight * kept).cumsum(-1)
        before = before - weight * kept
        kept &= before < s["top_p"].double()[:, None] * (weight * kept).sum(-1, keepdim=True)
    if s["min_p"] is not None:
        kept &= weight >= s["min_p"].double()[:, None]
    weight = torch.zeros_like(weight).scatter_(1, order, weight * kept)
    sums = weight.cumsum(-1)
    total = sums[:, -1:]
    token = (sums <= s["random"].double()[:, None] * total).sum(-1).clamp_max(value.shape[1] - 1)
    return token, (weight.gather(1, token[:, None]) / total)[:, 0].float()


def run(state):
    c = state["case"]
    if own:
        tfcc = importlib.import_module("wechat-tfcc_amd")
        if c["kind"] == "rotary":
            return tfcc.rotary(state["q"], state["k"], state["positions"], state["frequencies"], interleaved=c["interleaved"])
        if c["kind"] == "cache":
            tfcc.cache_write(state["cache"], state["k"], state["v"], state["slots"])
            return tfcc.cache_read(state["cache"], state["table"], state["starts"], state["all"])
        if c["kind"] == "attention":
            return tfcc.paged_attention(state["q"], state["cache"], state["table"], state["starts"], state["lengths"],
                                        state["scale"], window=c["window"], max_length=state["longest"])
        return tfcc.sample(state["logits"], state["random"], temperature=state["temperature"], top_k=state["top_k"],
                           top_p=state["top_p"], min_p=state["min_p"])
    if c["kind"] == "rotary":
        return _plain_rotary(state)
    if c["kind"] == "cache":
        return _plain_cache(state)
    if c["kind"] == "attention":
        return _plain_attention(state)
    return _plain_sample(state)


# ---- what a pass cannot do without -------------------------------------------------------------------------------
def work(case):
    if case["kind"] == "rotary":
        values = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["size"]
        turned = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["part"]
        return {"bytes": 8 * values + 4 * case["tokens"] + 4 * case["part"], "flops": 3 * turned}
    if case["kind"] == "sample":
        values = case["rows"] * case["vocabulary"]
        return {"bytes": 4 * values + 32 * case["rows"], "flops": 6 * values}
    lengths, chunks = _lengths(case)
    row = case["kv_heads"] * (case["size"] + 4 if case["cache"] == "s8" else 4 * case["size"])
    if case["kind"] == "cache":
        new, held, wide = sum(chunks), sum(lengths), case["kv_heads"] * case["size"] * 4
        return {"bytes": 2 * (new * wide + new * row + held * row + held * wide) + 8 * new,
                "flops": 2 * case["kv_heads"] * case["size"] * (3 * new + held)}
    used, pairs = 0, 0
    for n, c in zip(lengths, chunks):
        first = n - c
        w = case["window"] or n
        used += n - max(0, first + 1 - w)
        short = max(0, min(c, w - 1 - first))  # tokens whose window is not full yet
        pairs += short * first + short * (short + 1) // 2 + (c - short) * w
    return {"bytes": 2 * used * row + 8 * sum(chunks) * case["heads"] * case["size"],
            "flops": 4 * pairs * case["heads"] * case["size"]}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------
def _exact_rows(s, i, n):
    """Which page and which row of it hold the first n tokens of sequence i."""
    at = torch.arange(n, device=DEVICE)
    return s["table"][i].long()[torch.div(at, s["case"]["page"], rounding_mode="floor")], at.remainder(s["case"]["page"])


def _exact_held(s, held, page, inside):
    x = s["cache"][held][page, :, inside].double()
    return x * s["cache"][held + 2][page, :, inside].double().unsqueeze(-1) if s["case"]["cache"] == "s8" else x


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rotary":
        angle = torch.outer(s["positions"].double(), s["frequencies"])
        turn = torch.polar(torch.ones_like(angle), angle).unsqueeze(1)
        got = []
        for x in (s["q"].double(), s["k"].double()):
            n, half = case["part"], case["part"] // 2
            first, second = (slice(0, n, 2), slice(1, n, 2)) if case["interleaved"] else (slice(0, half), slice(half, n))
            z = torch.complex(x[..., first], x[..., second]) * turn
            y = x.clone()
            y[..., first], y[..., second] = z.real, z.imag
            got.append(y)
        return tuple(got)
    if case["kind"] == "cache":
        back = []
        for held, new in ((0, s["k"]), (1, s["v"])):
            pool = s["cache"][held].double()
            if case["cache"] == "s8":
                pool = pool * s["cache"][held + 2].double().unsqueeze(-1)
                step = (new.abs().max(-1, keepdim=True).values / 127.0).double()  # held as float32
                new = torch.round(new.double() / step) * step
            flat = pool.transpose(1, 2).reshape(-1, case["kv_heads"], case["size"])
            flat[s["slots"]] = new.double()
            at = [p * case["page"] + o for p, o in (_exact_rows(s, i, n) for i, n in enumerate(s["lengths"].tolist()))]
            back.append(flat[torch.cat(at)])
        return tuple(back)
    if case["kind"] == "attention":
        group, out = case["heads"] // case["kv_heads"], []
        starts = s["starts"].tolist()
        for i, n in enumerate(s["lengths"].tolist()):
            page, inside = _exact_rows(s, i, n)
            k, v = (_exact_held(s, held, page, inside).transpose(0, 1).repeat_interleave(group, 0) for held in (0, 1))
            q = s["q"][starts[i]:starts[i + 1]].double().transpose(0, 1)
            m = q.shape[1]
            seen = torch.ones(m, n, dtype=torch.bool, device=DEVICE).tril(n - m)
            if case["window"]:
                seen &= torch.ones(m, n, dtype=torch.bool, device=DEVICE).triu(n - m - case["window"] + 1)
            parts = []
            for h in range(0, case["heads"], 4):  # a few heads at a time
                x = torch.bmm(q[h:h + 4], k[h:h + 4].transpose(1, 2).contiguous()) / math.sqrt(case["size"])
                x = torch.log_softmax(x.masked_fill(~seen, -math.inf), -1).exp()
                parts.append(torch.bmm(x, v[h:h + 4].contiguous()))
            out.append(torch.cat(parts).transpose(0, 1))
        return torch.cat(out)
    tokens, odds = [], []
    for r in range(case["rows"]):
        x = s["logits"][r].double()
        p = torch.softmax(x / s["temperature"][r].double(), 0)
        by = torch.argsort(-x, stable=True)  # likeliest first, equals by their index
        n = min(int(s["top_k"][r]), x.numel()) if case["k"] else x.numel()
        sums = p[by[:n]].cumsum(0)
        if case["p"]:
            n = min(n, 1 + int((sums[:-1] < s["top_p"][r].double() * sums[-1]).sum()))
        if case["min"]:
            n = min(n, int((p[by] >= s["min_p"][r].double() * p.max()).sum()))
        left = by[:n].sort().values
        sums = p[left].cumsum(0)
        chosen = left[min(n - 1, int((sums <= s["random"][r].double() * sums[-1]).sum()))]
        tokens.append(chosen)
        odds.append(p[chosen] / sums[-1])
    return torch.stack(tokens), torch.stack(odds)
