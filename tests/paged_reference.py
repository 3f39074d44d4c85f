"""The paged cache's operators from their definitions in 64 bits on the CPU, position by position, with how far
BF16 outputs may be from them."""

import math

import torch

HALF = 2.0**-8  # half a BF16 step, relative


def visible_positions(query, window, sinks):
    return [p for p in range(query + 1) if window <= 0 or p > query - window or p < sinks]


def attention_row(q, k_cache, v_cache, table, query, *, window, sinks, scale):
    """(output, allowance) [heads, dim] of one token's heads q [heads, dim] at position `query`; CPU tensors."""
    heads, dim = q.shape
    pages, page_size, kv_heads, _ = k_cache.shape
    places = []
    for p in visible_positions(query, window, sinks):
        column = p // page_size
        page = int(table[column]) if column < table.numel() else -1
        if 0 <= page < pages:
            places.append((page, p % page_size))
    if not places:
        return torch.zeros(heads, dim, dtype=torch.float64), torch.zeros(heads, dim, dtype=torch.float64)
    page, slot = (torch.tensor(x) for x in zip(*places))
    k = k_cache[page, slot].double().repeat_interleave(heads // kv_heads, 1)  # [positions, heads, dim]
    v = v_cache[page, slot].double().repeat_interleave(heads // kv_heads, 1)
    q = q.double()
    score = torch.einsum("hd,phd->hp", q, k) * scale
    weight = torch.softmax(score, 1)
    out = torch.einsum("hp,phd->hd", weight, v)
    # Weights are rounded to BF16 (half a step each, of sum w |v|), the output once more (half a step of itself).
    # FP32: a score is off by at most (dim + 8) 2^-24 of sum |q k| scale, which moves every weight and their sum by
    # that much; a sum over n positions by n 2^-24 of sum w |v|.
    spread = torch.einsum("hp,phd->hd", weight, v.abs())
    size = (torch.einsum("hd,phd->hp", q.abs(), k.abs()) * scale).amax(1, keepdim=True)
    single = (2 * (dim + 8) * size + 2 * len(places) + 16) * 2.0**-24
    return out, (HALF * out.abs() + (HALF + single) * spread) * (1 + 2 * HALF)


def attention_rows(q, k_cache, v_cache, table, lengths, new, *, window=0, sinks=0, scale=None):
    """Rows of q [tokens, heads, dim] of sequences with new[b] tokens each, in order."""
    q, k_cache, v_cache, table = (t.cpu() for t in (q, k_cache, v_cache, table))
    scale = q.shape[2] ** -0.5 if scale is None else scale
    capacity = table.shape[1] * k_cache.shape[1]
    outs, allowed, row = [], [], 0
    for b, count in enumerate(new):
        length = max(0, min(int(lengths[b]), capacity))
        for i in range(count):
            out, off = attention_row(q[row], k_cache, v_cache, table[b], length - count + i, window=window, sinks=sinks,
                                     scale=scale)
            outs.append(out)
            allowed.append(off)
            row += 1
    return torch.stack(outs), torch.stack(allowed)


def append(qkv, positions, *, q_heads, kv_heads, q_weight, k_weight, epsilon, theta, rotary):
    """(queries, keys, their allowances) [tokens, heads, dim]."""
    x = qkv.cpu().double()[:, : q_heads + kv_heads]
    tokens, heads, dim = x.shape
    if q_weight is not None:
        weight = torch.cat([q_weight.cpu().double().expand(q_heads, dim), k_weight.cpu().double().expand(kv_heads, dim)])
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + epsilon) * weight
    half = rotary // 2
    out, size = x.clone(), x.abs()
    for i in range(half):
        angle = positions.cpu().double() * theta ** (-2.0 * i / rotary)
        s, c = angle.sin()[:, None], angle.cos()[:, None]
        lo, hi = x[:, :, i], x[:, :, i + half]
        out[:, :, i], out[:, :, i + half] = lo * c - hi * s, hi * c + lo * s
        size[:, :, i] = size[:, :, i + half] = lo.abs() + hi.abs()
    # one rounding to BF16; FP32 before it: the sum of squares is off by dim 2^-24 at most (half of that after the
    # root), sine and cosine by 2^-22, a handful of products and sums by 2^-24 each: under 2^-17 of the pair for 128 dims
    allowed = HALF * out.abs() * (1 + HALF) + 2.0**-17 * size
    return out[:, :q_heads], out[:, q_heads:], allowed[:, :q_heads], allowed[:, q_heads:]


def within(got, want, allowed):
    """Whether every value is as near as allowed; NaN where, and only where, it is wanted."""
    got, want = got.detach().cpu().double(), want.double()
    if not torch.equal(torch.isnan(got), torch.isnan(want)):
        return False
    fine = ~torch.isnan(want)
    infinite = fine & torch.isinf(want)
    if not torch.equal(got[infinite], want[infinite]):
        return False
    fine &= ~infinite
    return bool(((got - want).abs()[fine] <= allowed[fine]).all())


def paged_case(seed, lengths, *, page_size, kv_heads, dim, spare=3, device="cuda", layout="separate", poison=True):
    """(k_cache, v_cache, table): pages anywhere in the cache, every slot that no sequence holds poisoned with NaN and
    infinities, table entries behind a sequence's last page out of range."""
    g = torch.Generator().manual_seed(seed)
    held = [-(-n // page_size) for n in lengths]
    pages = sum(held) + spare
    order = torch.randperm(pages, generator=g).to(torch.int32)
    columns = max(held) + 2
    table = torch.full((len(lengths), columns), -1, dtype=torch.int32)
    table[:, 1::2] = 2**31 - 1
    k = torch.randn(pages, page_size, kv_heads, dim, generator=g)
    v = torch.randn(pages, page_size, kv_heads, dim, generator=g)
    used = torch.zeros(pages, page_size, dtype=torch.bool)
    at = 0
    for b, count in enumerate(held):
        table[b, :count] = order[at:at + count]
        for i in range(count):
            used[order[at + i].long(), : min(page_size, lengths[b] - i * page_size)] = True
        at += count
    if poison:
        k[~used] = math.nan
        v[~used] = torch.tensor([math.inf, math.nan, -math.inf, 3.0e38]).repeat(dim // 4)
    k, v = k.to(torch.bfloat16), v.to(torch.bfloat16)
    if layout == "together":  # views of one tensor [pages, 2, page_size, kv_heads, dim]
        both = torch.stack([k, v], 1).to(device)
        return both[:, 0], both[:, 1], table.to(device)
    if layout == "heads first":  # [pages, kv_heads, page_size, dim] in memory
        k, v = (t.transpose(1, 2).contiguous().to(device).transpose(1, 2) for t in (k, v))
        return k, v, table.to(device)
    return k.to(device), v.to(device), table.to(device)


def cache_layouts():
    """(keys, values) as views of one tensor, and whether all their rows are apart: [pages, slots, heads, dim]."""
    def room(*shape):
        return torch.zeros(*shape, dtype=torch.bfloat16)

    P, S, H, D = 5, 16, 3, 64
    both = room(2, P, S, H, D)
    yield both[0], both[1], True
    both = room(P, 2, S, H, D)
    yield both[:, 0], both[:, 1], True
    yield both[:, 1], both[:, 0], True
    both = room(P, 2, H, S, D)
    yield both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2), True
    both = room(P, S, H, 2 * D)
    yield both[..., :D], both[..., D:], True
    yield both[..., :D], both[..., 8:D + 8], False
    both = room(P, S, 2 * H, D)
    yield both[:, :, :H], both[:, :, H:], True
    yield both[:, :, ::2], both[:, :, 1::2], True
    yield both[:, :, :H], both[:, :, H - 1:-1], False
    both = room(P, 2 * S, H, D)
    yield both[:, ::2], both[:, 1::2], True
    yield both[:, :S], both[:, S:], True
    yield both[:, :S], both[:, S // 2:S // 2 + S], False
    both = room(2 * P, S, H, D)
    yield both[::2], both[1::2], True
    yield both[:P], both[P:], True
    yield both[:P], both[P - 1:-1], False
    yield both[:-1], both[1:], False
    flat = room(4 * P * S * H * D)
    yield flat.as_strided((P, S, H, D), (S * D, D, D, 1)), flat.as_strided((P, S, H, D), (S * D, D, D, 1), 2 * P * S * H * D), False
    yield flat.as_strided((P, S, H, D), (D, P * D, S * P * D, 1)), flat.as_strided((P, S, H, D), (D, P * D, S * P * D, 1), P * S * H * D), True
    yield flat.as_strided((1, S, 1, D), (0, D, 0, 1)), flat.as_strided((1, S, 1, D), (0, D, 0, 1), S * D), True
