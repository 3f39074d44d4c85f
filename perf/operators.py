"""The paged key-value cache's operators, as a serving program calls them: what fills the cache and what reads it.

  append    qk_norm_rope_append: per-head RMS norm of queries and keys, rotary embedding, keys and values into their slots
  decode    paged_decode_attention: one new token per sequence against its pages, optionally a window and first tokens
  prefill   paged_prefill_attention: the new tokens of ragged sequences against their pages, causal, the same masks

`run` computes them in elementary torch operations, or, where `own` is true, through camblas_amd._kernels.
"""

import math
import random

import torch

own = False

# The decoder layer that the benchmark measures has 64 query heads, 8 key-value heads and 128 dimensions a head; batch 32 and a
# cache of 2048 tokens are its sizes as well. The others are generic.
LAYER = {"q_heads": 64, "kv_heads": 8, "dim": 128}


def listed():
    return [
        # the smallest call of a decode step: one sequence's new token into the cache
        {"name": "append_1", "op": "append", "tokens": 1, **LAYER, "page": 16, "norm": True, "rotary": 128, "theta": 5e5},
        # a prompt's chunk into the cache
        {"name": "append_4096", "op": "append", "tokens": 4096, **LAYER, "page": 16, "norm": True, "rotary": 128, "theta": 5e5},
        # a model without the norm whose heads are rotated in part; pages of one slot, an odd number of tokens
        {"name": "append_1001_partial", "op": "append", "tokens": 1001, "q_heads": 20, "kv_heads": 5, "dim": 64, "page": 1, "norm": False,
         "rotary": 32, "theta": 1e4},
        # one short conversation: latency
        {"name": "decode_1x129", "op": "decode", "batch": 1, "shortest": 129, "longest": 129, **LAYER, "page": 16, "window": 0, "sinks": 0},
        # the benchmark's decode step
        {"name": "decode_32x2048", "op": "decode", "batch": 32, "shortest": 2048, "longest": 2048, **LAYER, "page": 16, "window": 0, "sinks": 0},
        # one long document
        {"name": "decode_1x131072", "op": "decode", "batch": 1, "shortest": 131072, "longest": 131072, **LAYER, "page": 64, "window": 0, "sinks": 0},
        # a busy server: conversations of every length at once
        {"name": "decode_64_ragged", "op": "decode", "batch": 64, "shortest": 1, "longest": 16384, **LAYER, "page": 16, "window": 0, "sinks": 0},
        # the same where a layer sees a window and the first tokens only; pages of one slot
        {"name": "decode_96_window", "op": "decode", "batch": 96, "shortest": 1, "longest": 10001, "q_heads": 20, "kv_heads": 5, "dim": 64, "page": 1,
         "window": 1024, "sinks": 4},
        # the ends of prompts whose beginnings are in the cache already
        {"name": "prefill_7_tails", "op": "prefill", "batch": 7, "fewest": 1, "most": 41, "past": 2000, "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "window": 0, "sinks": 0},
        # one prompt from its beginning
        {"name": "prefill_4096", "op": "prefill", "batch": 1, "fewest": 4096, "most": 4096, "past": 0, **LAYER, "page": 16, "window": 0, "sinks": 0},
        # a chunk of a long document
        {"name": "prefill_2048_far", "op": "prefill", "batch": 1, "fewest": 2048, "most": 2048, "past": 30001, **LAYER, "page": 64, "window": 0, "sinks": 0},
        # prompts of every length where a layer sees a window and the first tokens only
        {"name": "prefill_6_window", "op": "prefill", "batch": 6, "fewest": 100, "most": 5001, "past": 300, "q_heads": 28, "kv_heads": 4, "dim": 64, "page": 16,
         "window": 1024, "sinks": 4},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["append", "decode", "prefill"])
    dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 5, 8])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16])
    case = {"op": op, "q_heads": min(80 // kv_heads, group) * kv_heads, "kv_heads": kv_heads, "dim": dim, "page": rng.choice([1, 16, 32, 64, 256])}
    if op == "append":
        return {**case, "tokens": _spread(rng, 1, 4096), "norm": rng.random() < 0.7, "rotary": rng.choice([dim, dim, dim // 2]),
                "theta": rng.choice([1e4, 5e5, 1e6])}
    window = rng.choice([0, 0, _spread(rng, 1, 4096)])
    case.update(window=window, sinks=rng.choice([0, 1, 4, 64]) if window else 0)
    if op == "decode":
        batch = _spread(rng, 1, 256)
        longest = _spread(rng, 1, min(131072, 2**30 // (batch * kv_heads * dim)))
        return {**case, "batch": batch, "longest": longest, "shortest": rng.choice([1, longest, max(1, longest // 2)])}
    batch = _spread(rng, 1, 16)
    most = _spread(rng, 1, 4096)
    room = 2**32 // (batch * case["q_heads"] * most)  # of scores for each query
    past = rng.choice([0, _spread(rng, 1, 30001)])
    most = min(most, max(1, room // 2))
    return {**case, "batch": batch, "most": most, "fewest": rng.choice([1, most]), "past": max(0, min(past, room - most))}


def _between(case, low, high, what):
    """`batch` whole numbers between low and high, both among them where there is room; the same for every seed of a case."""
    rng = random.Random("%s %s %s %s" % (what, case["batch"], low, high))
    drawn = [rng.randint(low, high) for _ in range(case["batch"])]
    drawn[0] = high
    if len(drawn) > 1:
        drawn[-1] = low
    return drawn


def _lengths(case):
    """(new tokens, tokens in the cache with them) of every sequence."""
    if case["op"] == "decode":
        lengths = _between(case, case["shortest"], case["longest"], "lengths")
        return [1] * len(lengths), lengths
    new = _between(case, case["fewest"], case["most"], "new")
    past = _between(case, case["past"] // 2, case["past"], "past")
    return new, [n + p for n, p in zip(new, past)]


def _visible(case, position):
    """How many tokens a query at `position` sees."""
    seen = position + 1
    return min(seen, case["window"] + min(case["sinks"], max(0, seen - case["window"]))) if case["window"] else seen


def work(case):
    width = case["dim"] * 2  # bytes of a head's row
    if case["op"] == "append":
        heads = case["q_heads"] + 2 * case["kv_heads"]
        rows = case["tokens"] * heads
        return {"bytes": 2 * rows * width + case["tokens"] * 12, "flops": rows * case["dim"] * 8}
    new, lengths = _lengths(case)
    pairs = sum(_visible(case, p) for n, m in zip(new, lengths) for p in range(m - n, m))
    # rows of the cache that any of a sequence's queries sees
    first = [max(0, m - n + 1 - case["window"]) if case["window"] else 0 for n, m in zip(new, lengths)]
    rows = sum(m - f + min(case["sinks"], f) for m, f in zip(lengths, first))
    tables = sum(-(-r // case["page"]) * 4 for r in lengths)
    return {"bytes": 2 * rows * case["kv_heads"] * width + 2 * sum(new) * case["q_heads"] * width + tables,
            "flops": 4 * pairs * case["q_heads"] * case["dim"]}


def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device).manual_seed(seed)

    def normal(*shape, scale=1.0):
        return torch.empty(shape, dtype=torch.bfloat16, device=device).normal_(0.0, scale, generator=g)

    def numbers(values):
        return torch.tensor(values, dtype=torch.int32, device=device)

    q_heads, kv_heads, dim, page = case["q_heads"], case["kv_heads"], case["dim"], case["page"]
    if case["op"] == "append":
        tokens = case["tokens"]
        pages = -(-tokens // page) + 3
        slots = torch.randperm(pages * page, generator=g, device=device)[:tokens]  # int64
        slots[tokens // 2 + 1::97] = -1  # padding rows of a captured batch: not written
        state = {
            "qkv": normal(tokens, q_heads + 2 * kv_heads, dim),
            "positions": torch.randint(0, 1 << 20, (tokens,), generator=g, device=device, dtype=torch.int32),
            "slots": slots,
            "k_cache": normal(pages, page, kv_heads, dim),
            "v_cache": normal(pages, page, kv_heads, dim),
            "q_weight": (1 + normal(dim, scale=0.2)) if case["norm"] else None,
            "k_weight": (1 + normal(dim, scale=0.2)) if case["norm"] else None,
        }
        return {"case": case, **state}
    new, lengths = _lengths(case)
    held = [-(-m // page) for m in lengths]
    pages = sum(held) + 2
    # a sequence's pages lie anywhere in the cache; entries behind its last page are unset
    order = torch.randperm(pages, generator=g, device=device, dtype=torch.int64).to(torch.int32)
    width = max(held) + 1
    starts = numbers([sum(held[:b]) for b in range(len(held))])
    column = torch.arange(width, device=device, dtype=torch.int32)
    table = torch.where(column < numbers(held)[:, None], order[(starts[:, None] + column).clamp(max=pages - 1).long()], -1)
    state = {
        "q": normal(sum(new), q_heads, dim, scale=2.0),
        "k_cache": normal(pages, page, kv_heads, dim),
        "v_cache": normal(pages, page, kv_heads, dim),
        "page_table": table.contiguous(),
        "lengths": numbers(lengths),
    }
    if case["op"] == "prefill":
        state["query_starts"] = numbers([sum(new[:b]) for b in range(len(new) + 1)])
    return {"case": case, **state}


def _own(state):
    from camblas_amd import _kernels

    case = state["case"]
    if case["op"] == "append":
        q = _kernels.qk_norm_rope_append(
            state["qkv"], state["positions"], state["slots"], state["k_cache"], state["v_cache"], q_heads=case["q_heads"],
            kv_heads=case["kv_heads"], q_weight=state["q_weight"], k_weight=state["k_weight"], epsilon=1e-6, theta=case["theta"],
            rotary_dim=case["rotary"])
        return {"q": q, "k_cache": state["k_cache"], "v_cache": state["v_cache"]}
    if case["op"] == "decode":
        return _kernels.paged_decode_attention(state["q"], state["k_cache"], state["v_cache"], state["page_table"], state["lengths"],
                                               window=case["window"], sinks=case["sinks"])
    return _kernels.paged_prefill_attention(state["q"], state["k_cache"], state["v_cache"], state["page_table"], state["lengths"],
                                            state["query_starts"], window=case["window"], sinks=case["sinks"])


def _plain_append(state):
    case = state["case"]
    q_heads, kv_heads, rotary = case["q_heads"], case["kv_heads"], case["rotary"]
    x = state["qkv"].float()
    q, k, v = x.split([q_heads, kv_heads, kv_heads], dim=1)
    if case["norm"]:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + 1e-6) * state["q_weight"].float()
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + 1e-6) * state["k_weight"].float()
    # (the angle of a far position is a large number of turns: 64 bits)
    frequency = case["theta"] ** (-torch.arange(0, rotary, 2, device=x.device, dtype=torch.float64) / rotary)
    angle = state["positions"].double()[:, None, None] * frequency
    sine, cosine = angle.sin().float(), angle.cos().float()

    def rotated(t):
        low, high, rest = t.split([rotary // 2, rotary // 2, case["dim"] - rotary], dim=-1)
        return torch.cat([low * cosine - high * sine, high * cosine + low * sine, rest], dim=-1).to(torch.bfloat16)

    k_rows, v_rows = state["k_cache"].view(-1, kv_heads, case["dim"]), state["v_cache"].view(-1, kv_heads, case["dim"])
    # a token without a slot writes back what stands in the slot of the first one
    has = (state["slots"] >= 0)[:, None, None]
    first = state["slots"][:1]
    slots = torch.where(state["slots"] >= 0, state["slots"], first)
    k_new, v_new = rotated(k), v.to(torch.bfloat16)
    k_rows[slots] = torch.where(has, k_new, k_new[:1])
    v_rows[slots] = torch.where(has, v_new, v_new[:1])
    return {"q": rotated(q), "k_cache": state["k_cache"], "v_cache": state["v_cache"]}


def _plain_attention(state, q, position):
    """q [batch, queries, heads, dim] at `position` [batch, queries]; 32 bits."""
    case = state["case"]
    batch, queries, q_heads, dim = q.shape
    kv_heads = case["kv_heads"]
    pages = state["page_table"].clamp(min=0).long()
    k = state["k_cache"][pages].view(batch, -1, kv_heads, dim).permute(0, 2, 3, 1).float().contiguous()
    v = state["v_cache"][pages].view(batch, -1, kv_heads, dim).permute(0, 2, 1, 3).float().contiguous()
    group = q_heads // kv_heads
    rows = q.float().view(batch, queries, kv_heads, group, dim).permute(0, 2, 1, 3, 4).reshape(batch, kv_heads, queries * group, dim)
    scores = torch.matmul(rows * dim**-0.5, k).view(batch, kv_heads, queries, group, -1)
    key = torch.arange(k.shape[-1], device=q.device)
    seen = key <= position[:, :, None]
    if case["window"]:
        seen = seen & ((key > position[:, :, None] - case["window"]) | (key < case["sinks"]))
    scores.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = torch.matmul(scores.view(batch, kv_heads, queries * group, -1), v).view(batch, kv_heads, queries, group, dim) / total
    return out.permute(0, 2, 1, 3, 4).reshape(batch, queries, q_heads, dim).to(torch.bfloat16)


def _plain_decode(state):
    return _plain_attention(state, state["q"][:, None], state["lengths"][:, None] - 1)[:, 0]


def _plain_prefill(state):
    case, q, starts = state["case"], state["q"], state["query_starts"].long()
    index = torch.arange(case["most"], device=q.device)
    new = starts[1:] - starts[:-1]
    padded = q[(starts[:-1, None] + index).clamp(max=q.shape[0] - 1)]
    # (rows behind a sequence's last query stand at its last position)
    position = torch.minimum(state["lengths"][:, None] - new[:, None] + index, state["lengths"][:, None] - 1)
    out = _plain_attention(state, padded, position)
    token = torch.arange(q.shape[0], device=q.device)
    sequence = (token[:, None] >= starts[1:]).sum(1)
    return out[sequence, token - starts[sequence]]


def run(state):
    if own:
        return _own(state)
    return {"append": _plain_append, "decode": _plain_decode, "prefill": _plain_prefill}[state["case"]["op"]](state)


def _exact_append(case, state):
    tokens, q_heads, kv_heads, dim = case["tokens"], case["q_heads"], case["kv_heads"], case["dim"]
    half = case["rotary"] // 2
    x = state["qkv"].to(torch.float64)
    exponent = torch.arange(half, dtype=torch.float64, device=x.device) * (-2.0 / case["rotary"])
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device),
                       state["positions"].to(torch.float64)[:, None] * torch.exp(exponent * math.log(case["theta"])))

    def head(h, weight):
        row = x[:, h]
        if case["norm"]:
            row = row / torch.sqrt((row * row).sum(1, keepdim=True) / dim + 1e-6) * weight.to(torch.float64)
        row = row.clone()
        pair = torch.complex(row[:, :half], row[:, half:2 * half]) * turn
        row[:, :half], row[:, half:2 * half] = pair.real, pair.imag
        return row

    q = torch.stack([head(h, state["q_weight"]) for h in range(q_heads)], 1)
    k_cache, v_cache = state["k_cache"].to(torch.float64), state["v_cache"].to(torch.float64)
    written = torch.nonzero(state["slots"] >= 0)[:, 0]
    page, slot = state["slots"][written] // case["page"], state["slots"][written] % case["page"]
    for h in range(kv_heads):
        k_cache[page, slot, h] = head(q_heads + h, state["k_weight"])[written]
        v_cache[page, slot, h] = x[written, q_heads + kv_heads + h]
    return {"q": q.view(tokens, q_heads, dim), "k_cache": k_cache, "v_cache": v_cache}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(case, state)
    new, lengths = _lengths(case)
    group = case["q_heads"] // case["kv_heads"]
    out = torch.empty(state["q"].shape, dtype=torch.float64, device=state["q"].device)
    first = 0
    for b, (n, m) in enumerate(zip(new, lengths)):
        place = torch.arange(m, device=out.device)
        page = state["page_table"][b].long()[place // case["page"]]
        k = state["k_cache"][page, place % case["page"]].to(torch.float64)
        v = state["v_cache"][page, place % case["page"]].to(torch.float64)
        for low in range(0, n, 1024):
            high = min(n, low + 1024)
            age = torch.arange(m - n + low, m - n + high, device=out.device)[:, None] - place
            hidden = age < 0
            if case["window"]:
                hidden |= (age >= case["window"]) & (place >= case["sinks"])
            for h in range(case["q_heads"]):
                q = state["q"][first + low:first + high, h].to(torch.float64)
                weight = torch.softmax((q @ k[:, h // group].T / math.sqrt(case["dim"])).masked_fill(hidden, -math.inf), 1)
                out[first + low:first + high, h] = weight @ v[:, h // group]
        first += n
    return out
