"""The paged key-value cache on the GPU: append with per-head norm and rotation, decode and prefill attention,
against their definitions in 64 bits; a run of them together; captured graphs; refusals.

Slots that no sequence holds are filled with NaN and infinities, and table entries behind a sequence's pages
are out of range: neither may reach an output."""

import ctypes as ct
import math

import pytest
import torch

import paged_reference as reference
from camblas_amd import _kernels, _native

pytestmark = pytest.mark.gpu


def queries(seed, tokens, heads, dim, device, scale=1.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(tokens, heads, dim, generator=g) * scale).to(torch.bfloat16).to(device)


def starts_of(new, device):
    at = [0]
    for count in new:
        at.append(at[-1] + count)
    return torch.tensor(at, dtype=torch.int32, device=device)


def check_decode(device, seed, lengths, *, q_heads, kv_heads, dim, page_size, window=0, sinks=0, scale=None, layout="separate"):
    k, v, table = reference.paged_case(seed, lengths, page_size=page_size, kv_heads=kv_heads, dim=dim, device=device, layout=layout)
    q = queries(seed + 1, len(lengths), q_heads, dim, device)
    held = torch.tensor(lengths, dtype=torch.int32, device=device)
    got = _kernels.paged_decode_attention(q, k, v, table, held, window=window, sinks=sinks, scale=scale)
    want, allowed = reference.attention_rows(q, k, v, table, lengths, [1] * len(lengths), window=window, sinks=sinks, scale=scale)
    assert reference.within(got, want, allowed)
    return got


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page_size", [1, 16, 64])
@pytest.mark.parametrize("q_heads,kv_heads", [(8, 1), (6, 3), (4, 4), (20, 1), (66, 2)])
def test_decode_lengths_heads_and_pages(device, dim, page_size, q_heads, kv_heads):
    check_decode(device, 100, [1, 31, 32, 33, 0, 127, 128, 129, 300, 5], q_heads=q_heads, kv_heads=kv_heads, dim=dim, page_size=page_size)


@pytest.mark.parametrize("page_size", [2, 4, 8, 32, 128, 1024])
def test_decode_page_sizes(device, page_size):
    check_decode(device, 150, [700, 1, 65, 511], q_heads=8, kv_heads=2, dim=128, page_size=page_size)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 3), (32, 0), (33, 64), (100, 4), (128, 33), (1000, 2000), (5000, 4)])
def test_decode_windows_and_first_tokens(device, dim, window, sinks):
    check_decode(device, 200, [1, 2, 31, 64, 65, 100, 101, 160, 777, 0], q_heads=10, kv_heads=2, dim=dim, page_size=16, window=window, sinks=sinks)


@pytest.mark.parametrize("lengths", [[4000], [1, 3000, 1, 1, 2500, 0, 0, 700], [513] * 20, [0, 0, 2000], [1] * 300 + [1500]])
def test_decode_divided_over_workgroups(device, lengths):
    check_decode(device, 300, lengths, q_heads=8, kv_heads=2, dim=128, page_size=16)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page_size", [1, 16])
@pytest.mark.parametrize("window,sinks", [(1500, 0), (1700, 4), (2500, 64)])
@pytest.mark.parametrize("lengths", [[3300], [3100, 1, 2600, 700]])
def test_decode_windows_divided_over_workgroups(device, dim, page_size, window, sinks, lengths):
    q_heads, kv_heads = 8, 2
    cache = _native.PagedCache(16, 32, page_size * kv_heads * dim, kv_heads * dim, dim, 4, page_size, kv_heads, dim)  # (sizes only)
    columns = -(-max(lengths) // page_size) + 2
    assert _native.library().camblas_cuda_paged_decode_workspace_size(_native.context(device).handle, len(lengths), q_heads, ct.byref(cache), columns,
                                                                      window, sinks) > 0
    check_decode(device, 310, lengths, q_heads=q_heads, kv_heads=kv_heads, dim=dim, page_size=page_size, window=window, sinks=sinks)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page_size", [4, 16])
@pytest.mark.parametrize("longest,window", [(1, 0), (67, 0), (256, 0), (600, 90)])
def test_decode_many_sequences_of_few_positions(device, dim, page_size, longest, window):
    # several workgroups per compute unit
    lengths = [b * 41 % (longest + 1) for b in range(70)]
    check_decode(device, 350, lengths, q_heads=8, kv_heads=8, dim=dim, page_size=page_size, window=window, sinks=3)


@pytest.mark.parametrize("layout", ["together", "heads first"])
def test_decode_layouts_of_the_cache(device, layout):
    check_decode(device, 400, [5, 200, 1030], q_heads=9, kv_heads=3, dim=64, page_size=16, layout=layout)


def test_decode_strided_queries_outputs_and_table(device):
    lengths = [40, 3, 700]
    k, v, table = reference.paged_case(500, lengths, page_size=16, kv_heads=2, dim=128, device=device)
    qkv = queries(501, 3, 12, 128, device)
    wide = torch.full((3, table.shape[1] + 5), -7, dtype=torch.int32, device=device)
    wide[:, : table.shape[1]] = table
    out = torch.full((3, 16, 128), 9.0, dtype=torch.bfloat16, device=device)
    held = torch.tensor(lengths, dtype=torch.int32, device=device)
    _kernels.paged_decode_attention(qkv[:, :8], k, v, wide[:, : table.shape[1]], held, out=out[:, 4:12])
    plain = _kernels.paged_decode_attention(qkv[:, :8].contiguous(), k, v, table, held)
    assert torch.equal(out[:, 4:12], plain)
    assert (out[:, :4] == 9).all() and (out[:, 12:] == 9).all()


def test_decode_pages_that_do_not_exist_hold_nothing(device):
    lengths = [200, 64]
    k, v, table = reference.paged_case(600, lengths, page_size=16, kv_heads=1, dim=128, device=device)
    table[0, 3], table[0, 7], table[0, 12] = -1, k.shape[0], -2**31
    table[1, :] = 2**30  # a sequence none of whose pages exists
    q = queries(601, 2, 8, 128, device)
    got = _kernels.paged_decode_attention(q, k, v, table, torch.tensor([200, 64], dtype=torch.int32, device=device))
    want, allowed = reference.attention_rows(q, k, v, table, lengths, [1, 1])
    assert reference.within(got, want, allowed) and not got[1].any()


def test_decode_lengths_outside_the_table(device):
    k, v, table = reference.paged_case(650, [64, 64, 64], page_size=16, kv_heads=1, dim=64, device=device, poison=False)
    table = table[:, :4].contiguous()
    q = queries(651, 3, 4, 64, device)
    got = _kernels.paged_decode_attention(q, k, v, table, torch.tensor([2**31 - 1, -5, 65], dtype=torch.int32, device=device))
    want, allowed = reference.attention_rows(q, k, v, table, [64, 0, 64], [1, 1, 1])
    assert reference.within(got, want, allowed)


def test_decode_values_that_are_not_numbers_where_they_are_seen(device):
    lengths = [100, 100, 100]
    k, v, table = reference.paged_case(700, lengths, page_size=16, kv_heads=1, dim=128, device=device)
    rows = [(int(table[b, 40 // 16]), 40 % 16) for b in range(3)]
    v[rows[0]][0, 5] = math.nan
    v[rows[1]][0, 6] = math.inf
    k[rows[2]][0, 7] = math.nan
    q = queries(701, 3, 8, 128, device)
    got = _kernels.paged_decode_attention(q, k, v, table, torch.tensor(lengths, dtype=torch.int32, device=device))
    assert torch.isnan(got[0, :, 5]).all() and torch.isinf(got[1, :, 6]).all() and torch.isnan(got[2]).all()
    assert torch.isnan(got[0]).sum() == 8 and not torch.isnan(got[1]).any() and torch.isinf(got[1]).sum() == 8


def test_decode_far_scores_and_extreme_scales(device):
    # scores of +-700: weights underflow, the maximum moves by hundreds between tiles
    lengths = [640]
    k, v, table = reference.paged_case(750, lengths, page_size=16, kv_heads=1, dim=64, device=device)
    q = queries(751, 1, 8, 64, device, scale=30.0)
    got = _kernels.paged_decode_attention(q, k, v, table, torch.tensor(lengths, dtype=torch.int32, device=device), scale=1.0)
    want, allowed = reference.attention_rows(q, k, v, table, lengths, [1], scale=1.0)
    assert reference.within(got, want, allowed)


def check_prefill(device, seed, new, past, *, q_heads, kv_heads, dim, page_size, window=0, sinks=0, layout="separate"):
    lengths = [n + p for n, p in zip(new, past)]
    k, v, table = reference.paged_case(seed, lengths, page_size=page_size, kv_heads=kv_heads, dim=dim, device=device, layout=layout)
    q = queries(seed + 1, sum(new) + 3, q_heads, dim, device)
    out = torch.full(q.shape, 5.0, dtype=torch.bfloat16, device=device)
    _kernels.paged_prefill_attention(q, k, v, table, torch.tensor(lengths, dtype=torch.int32, device=device),
                                     starts_of(new, device), window=window, sinks=sinks, out=out)
    want, allowed = reference.attention_rows(q, k, v, table, lengths, new, window=window, sinks=sinks)
    assert reference.within(out[: sum(new)], want, allowed)
    assert (out[sum(new):] == 5).all()  # rows behind the last sequence


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q_heads,kv_heads", [(8, 1), (4, 4), (6, 2), (7, 1), (20, 1)])
def test_prefill_ragged(device, dim, q_heads, kv_heads):
    check_prefill(device, 1000, [1, 17, 0, 64, 65, 3], [0, 40, 9, 0, 63, 200], q_heads=q_heads, kv_heads=kv_heads, dim=dim, page_size=16)


@pytest.mark.parametrize("page_size", [1, 8, 64, 256])
def test_prefill_page_sizes(device, page_size):
    check_prefill(device, 1100, [70, 5, 128], [0, 333, 1], q_heads=4, kv_heads=2, dim=128, page_size=page_size)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 2), (16, 4), (64, 0), (65, 70), (100, 1), (1000, 8)])
def test_prefill_windows_and_first_tokens(device, dim, window, sinks):
    check_prefill(device, 1200, [150, 33, 1], [0, 190, 64], q_heads=6, kv_heads=2, dim=dim, page_size=16, window=window, sinks=sinks)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,past,window,sinks", [
    ([1], [3000], 0, 0), ([1, 17, 0, 40], [3001, 0, 77, 2500], 0, 0), ([9, 3], [2000, 2], 700, 100), ([1] * 5, [1500, 0, 3, 640, 1], 0, 0),
    ([130], [1300], 1000, 0)])
def test_prefill_positions_divided_over_workgroups(device, dim, new, past, window, sinks):
    check_prefill(device, 1250, new, past, q_heads=6, kv_heads=2, dim=dim, page_size=16, window=window, sinks=sinks)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page_size,window,sinks", [(16, 0, 0), (64, 0, 0), (4, 0, 0), (16, 1200, 70)])
def test_prefill_long_and_undivided(device, dim, page_size, window, sinks):
    """Blocks of rows that walk dozens of tiles by themselves; a sample of the tokens against the definition, twice the same."""
    new, past, q_heads, kv_heads = 2100, 333, 28, 7
    lengths = [new + past]
    k, v, table = reference.paged_case(1270, lengths, page_size=page_size, kv_heads=kv_heads, dim=dim, device=device)
    cache = _native.PagedCache(k.data_ptr(), v.data_ptr(), *k.stride()[:3], *k.shape)
    assert _native.library().camblas_cuda_paged_prefill_workspace_size(_native.context(device).handle, 1, new, q_heads, ct.byref(cache),
                                                                       table.shape[1], window, sinks) == 0
    q = queries(1271, new, q_heads, dim, device)
    held = torch.tensor(lengths, dtype=torch.int32, device=device)
    call = lambda: _kernels.paged_prefill_attention(q, k, v, table, held, starts_of([new], device), window=window, sinks=sinks)
    got = call()
    assert torch.equal(got, call())
    g = torch.Generator().manual_seed(1272)
    for token in [0, 1, 31, 32, new - 1, *torch.randint(0, new, (12,), generator=g).tolist()]:
        want, allowed = reference.attention_row(q[token].cpu(), k.cpu(), v.cpu(), table[0].cpu(), past + token, window=window, sinks=sinks,
                                                scale=dim**-0.5)
        assert reference.within(got[token], want, allowed), token


@pytest.mark.parametrize("layout", ["together", "heads first"])
def test_prefill_layouts_of_the_cache(device, layout):
    check_prefill(device, 1300, [40, 100], [10, 0], q_heads=4, kv_heads=2, dim=128, page_size=16, layout=layout)


def test_prefill_more_queries_than_positions(device):
    # 10 new tokens, 4 positions in the cache: the first six see nothing
    k, v, table = reference.paged_case(1400, [4, 20], page_size=4, kv_heads=1, dim=64, device=device)
    q = queries(1401, 30, 4, 64, device)
    new, lengths = [10, 20], [4, 20]
    got = _kernels.paged_prefill_attention(q, k, v, table, torch.tensor(lengths, dtype=torch.int32, device=device), starts_of(new, device))
    want, allowed = reference.attention_rows(q, k, v, table, lengths, new)
    assert reference.within(got, want, allowed) and not got[:6].any()


def test_prefill_pages_that_do_not_exist_hold_nothing(device):
    new, lengths = [30, 50], [200, 50]
    k, v, table = reference.paged_case(1500, lengths, page_size=16, kv_heads=2, dim=128, device=device)
    table[0, 2], table[0, 11], table[1, :] = -3, k.shape[0], 2**31 - 1
    q = queries(1501, 80, 8, 128, device)
    got = _kernels.paged_prefill_attention(q, k, v, table, torch.tensor(lengths, dtype=torch.int32, device=device), starts_of(new, device))
    want, allowed = reference.attention_rows(q, k, v, table, lengths, new)
    assert reference.within(got, want, allowed) and not got[30:].any()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("past", [0, 1500])
def test_prefill_infinite_and_nan_values_reach_only_who_sees_them(device, dim, past):
    """Rows of the prompt itself that hold NaN and infinities: earlier tokens, and later ones beyond the window, stay
    finite."""
    new, window = 200, 70
    lengths = [past + new]
    k, v, table = reference.paged_case(1550, lengths, page_size=16, kv_heads=2, dim=dim, device=device)
    marks = {past + 50: (3, math.nan), past + 51: (4, math.inf), past + 127: (dim - 1, -math.inf), past + 128: (9, math.inf)}
    for position, (d, value) in marks.items():
        v[int(table[0, position // 16]), position % 16, 1, d] = value
    k[int(table[0, (past + 160) // 16]), (past + 160) % 16, 0, 2] = math.nan
    q = queries(1551, new, 6, dim, device)
    got = _kernels.paged_prefill_attention(q, k, v, table, torch.tensor(lengths, dtype=torch.int32, device=device), starts_of([new], device),
                                           window=window, sinks=0)
    want, allowed = reference.attention_rows(q, k, v, table, lengths, [new], window=window, sinks=0)
    assert reference.within(got, want, allowed)
    assert torch.isnan(want).any() and torch.isinf(want).any()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("past,window,scale", [(0, 0, None), (3000, 0, None), (3000, 40, None), (3000, 1500, None), (0, 0, 5.0), (3000, 0, 5.0)])
def test_scores_of_minus_infinity(device, dim, past, window, scale):
    """Keys of minus infinity take a weight of zero; where a token sees such keys only, the softmax is 0 / 0 and the output
    NaN, not the zeros of a token that sees nothing."""
    new, q_heads, kv_heads, page_size = 70, 6, 2, 16
    lengths = [past + new, 5, 0, 3]
    k, v, table = reference.paged_case(760, lengths, page_size=page_size, kv_heads=kv_heads, dim=dim, device=device)
    hidden = list(range(0, past + 20)) + list(range(past + 50, past + 64))  # of the first sequence, for every head
    place = torch.tensor(hidden)
    page = table[0].cpu()[place // page_size].long().to(device)
    k[page, (place % page_size).to(device), :, 3] = -math.inf
    k[int(table[1, 0]), :5, 1, 7] = -math.inf  # all of the second's, one head
    table[3, :] = -1  # no page: nothing is seen
    q = queries(761, new + 5 + 3, q_heads, dim, device)
    q[:, :, 3], q[:, :, 7] = q[:, :, 3].abs() + 0.1, q[:, :, 7].abs() + 0.1
    held = torch.tensor(lengths, dtype=torch.int32, device=device)
    counts = [new, 5, 0, 3]
    got = _kernels.paged_prefill_attention(q, k, v, table, held, starts_of(counts, device), window=window, sinks=0, scale=scale)
    want, allowed = reference.attention_rows(q, k, v, table, lengths, counts, window=window, sinks=0, scale=scale)
    assert torch.isnan(want[:20]).all() and not torch.isnan(want[20:50]).any() and torch.isnan(want[new:new + 5, 3:]).all()
    assert reference.within(got, want, allowed) and not got[new + 5:].any()
    # single tokens, at a length where all of the first sequence's keys are such and at its end
    for length in (past + 20, past + new):
        now = [length, 5, 0, 3]
        held = torch.tensor(now, dtype=torch.int32, device=device)
        got = _kernels.paged_decode_attention(q[:4], k, v, table, held, window=window, scale=scale)
        want, allowed = reference.attention_rows(q[:4], k, v, table, now, [1] * 4, window=window, scale=scale)
        assert torch.isnan(want[0]).all().item() == (length == past + 20)
        assert reference.within(got, want, allowed) and not got[2:].any()


def test_prefill_one_token_each_equals_decode_within_rounding(device):
    lengths = [1, 70, 1030, 257]
    k, v, table = reference.paged_case(1600, lengths, page_size=16, kv_heads=2, dim=128, device=device)
    q = queries(1601, 4, 16, 128, device)
    held = torch.tensor(lengths, dtype=torch.int32, device=device)
    a = _kernels.paged_decode_attention(q, k, v, table, held)
    b = _kernels.paged_prefill_attention(q, k, v, table, held, starts_of([1] * 4, device))
    want, allowed = reference.attention_rows(q, k, v, table, lengths, [1] * 4)
    assert reference.within(a, want, allowed) and reference.within(b, want, allowed)


APPEND_CASES = [
    # tokens, q_heads, kv_heads, dim, rotary, norm, page_size
    (1, 64, 8, 128, 128, torch.bfloat16, 16), (7, 6, 2, 64, 64, torch.float32, 1), (33, 5, 1, 128, 64, None, 4),
    (130, 3, 3, 64, 16, torch.bfloat16, 64), (65, 8, 8, 128, 0, torch.float32, 16), (3000, 4, 1, 64, 32, torch.bfloat16, 16),
    (2, 1, 1, 128, 112, None, 32)]


@pytest.mark.parametrize("tokens,q_heads,kv_heads,dim,rotary,norm,page_size", APPEND_CASES)
def test_append(device, tokens, q_heads, kv_heads, dim, rotary, norm, page_size):
    g = torch.Generator().manual_seed(2000 + tokens)
    wide = torch.randn(tokens, q_heads + 2 * kv_heads + 1, dim, generator=g).to(torch.bfloat16)
    wide[0, 0] *= 1e-4  # a head whose mean square is of the size of epsilon
    wide = wide.to(device)
    qkv = wide[:, : q_heads + 2 * kv_heads]
    positions = torch.randint(0, 2**31 - 1, (tokens,), generator=g, dtype=torch.int64).to(torch.int32)
    positions[0] = 0
    pages = -(-tokens // page_size) + 2
    slots = torch.randperm(pages * page_size, generator=g)[:tokens]
    slots[tokens // 3 + 1::5] = -1
    if tokens > 2:
        slots[-1] = pages * page_size  # the first behind the cache
    weights = [None, None] if norm is None else [(1 + 0.3 * torch.randn(dim, generator=g)).to(norm).to(device) for _ in range(2)]
    before = torch.randn(2, pages, page_size, kv_heads, dim, generator=g).to(torch.bfloat16).to(device)
    k, v = before[0].clone(), before[1].clone()
    got = _kernels.qk_norm_rope_append(qkv, positions.to(device), slots.to(device), k, v, q_heads=q_heads, kv_heads=kv_heads,
                                       q_weight=weights[0], k_weight=weights[1], epsilon=1e-6, theta=10000.0, rotary_dim=rotary)
    q_want, k_want, q_off, k_off = reference.append(qkv, positions, q_heads=q_heads, kv_heads=kv_heads, q_weight=weights[0],
                                                    k_weight=weights[1], epsilon=1e-6, theta=10000.0, rotary=rotary)
    assert reference.within(got, q_want, q_off)
    kept = (slots >= 0) & (slots < pages * page_size)
    where = slots[kept].to(device)
    assert reference.within(k.view(-1, kv_heads, dim)[where], k_want[kept], k_off[kept])
    assert torch.equal(v.view(-1, kv_heads, dim)[where], qkv[:, q_heads + kv_heads:][kept.to(device)])
    others = torch.ones(pages * page_size, dtype=torch.bool, device=device)
    others[where] = False
    for cache, old in ((k, before[0]), (v, before[1])):
        assert torch.equal(cache.view(-1, kv_heads, dim)[others], old.view(-1, kv_heads, dim)[others])


@pytest.mark.parametrize("theta", [500000 * 8 ** (128 / 126), 10000 * 4 ** (128 / 126)])
@pytest.mark.parametrize("dim,rotary", [(64, 64), (128, 64), (128, 128)])
def test_append_bases_that_32_bits_do_not_hold(device, theta, dim, rotary):
    """Rescaled bases, up to the farthest position. Allowed is 2^-17 of a pair: a turn of lane i is a product of i powers
    of one (relative error (3 i + 8) 2^-53 at most: one step for the power, doubled and rounded with every square, six
    products, two roundings of the position's turn) and theta^(-2 i / rotary) 2^31 / 2 pi turns long, so off by at most 10.5 * 2^-53
    * 2^28.35 turns = 2^-18.6 radians for the bases and dims here (the largest (3 i + 8) theta^(-2 i / rotary) is 10.5);
    the reference's angle by 2^-21, the FP32 fraction of a turn, sine, cosine and products by 2^-21 together. These
    bases rounded to 32 bits are off by up to 2^-10 of a radian at 2^20."""
    tokens, q_heads, kv_heads = 40, 3, 2
    assert ct.c_float(theta).value != theta
    qkv = queries(2150, tokens, q_heads + 2 * kv_heads, dim, device)
    g = torch.Generator().manual_seed(2151)
    positions = torch.randint(0, 2**31 - 1, (tokens,), generator=g, dtype=torch.int64).to(torch.int32)
    positions[:5] = torch.tensor([0, 1, 2**20, 2**30, 2**31 - 1])
    positions[5:20] = positions[5:20] % 2**20
    k, v = (torch.zeros(tokens, 1, kv_heads, dim, dtype=torch.bfloat16, device=device) for _ in range(2))
    got = _kernels.qk_norm_rope_append(qkv, positions.to(device), torch.arange(tokens, device=device), k, v, q_heads=q_heads, kv_heads=kv_heads,
                                       theta=theta, rotary_dim=rotary)
    q_want, k_want, q_off, k_off = reference.append(qkv, positions, q_heads=q_heads, kv_heads=kv_heads, q_weight=None, k_weight=None,
                                                    epsilon=0.0, theta=theta, rotary=rotary)
    assert reference.within(got, q_want, q_off)
    assert reference.within(k[:, 0], k_want, k_off)
    for other in (1e300, 1e-60, math.inf):  # outside of what 32 bits hold at all
        refused(_kernels.qk_norm_rope_append, qkv, positions.to(device), torch.arange(tokens, device=device), k, v, q_heads=q_heads,
                kv_heads=kv_heads, theta=other, rotary_dim=rotary)


def test_append_in_place_and_into_views_of_one_cache(device):
    tokens, q_heads, kv_heads, dim = 50, 12, 3, 128
    qkv = queries(2100, tokens, q_heads + 2 * kv_heads, dim, device)
    weight = torch.rand(dim, device=device) + 0.5
    positions = torch.arange(tokens, dtype=torch.int32, device=device)
    slots = torch.arange(tokens, device=device) * 2
    options = dict(q_heads=q_heads, kv_heads=kv_heads, q_weight=weight, k_weight=weight, rotary_dim=64)
    k, v = (torch.zeros(8, 16, kv_heads, dim, dtype=torch.bfloat16, device=device) for _ in range(2))
    apart = _kernels.qk_norm_rope_append(qkv, positions, slots, k, v, **options)
    both = torch.zeros(8, 2, kv_heads, 16, dim, dtype=torch.bfloat16, device=device)
    k2, v2 = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    copy = qkv.clone()
    _kernels.qk_norm_rope_append(copy, positions, slots, k2, v2, out=copy[:, :q_heads], **options)
    assert torch.equal(copy[:, :q_heads], apart) and torch.equal(copy[:, q_heads:], qkv[:, q_heads:])
    assert torch.equal(k2, k) and torch.equal(v2, v)


def test_append_into_every_layout_of_a_cache_and_none_that_overlaps(device):
    tokens, q_heads, kv_heads, dim = 30, 4, 3, 64
    qkv = queries(2110, tokens, q_heads + 2 * kv_heads, dim, device)
    positions = torch.arange(tokens, dtype=torch.int32, device=device)
    slots = torch.arange(tokens, device=device) * 2 + 1
    options = dict(q_heads=q_heads, kv_heads=kv_heads)
    want = [torch.zeros(5, 16, kv_heads, dim, dtype=torch.bfloat16, device=device) for _ in range(2)]
    _kernels.qk_norm_rope_append(qkv, positions, slots, *want, **options)
    seen = 0
    for k, v, apart in reference.cache_layouts():
        if k.shape[2] != kv_heads:
            continue
        room = torch.zeros(k.untyped_storage().nbytes() // 2, dtype=torch.bfloat16, device=device)
        k, v = (room.as_strided(t.shape, t.stride(), t.storage_offset()) for t in (k, v))
        if apart:
            _kernels.qk_norm_rope_append(qkv, positions, slots, k, v, **options)
            assert torch.equal(k[:5], want[0]) and torch.equal(v[:5], want[1])
        else:
            with pytest.raises(RuntimeError, match="share memory"):
                _kernels.qk_norm_rope_append(qkv, positions, slots, k, v, **options)
            assert not room.any()
        seen += 1
    assert seen >= 15


def test_a_sequence_from_prompt_to_decode_steps(device):
    """A prompt in two ragged chunks, then single tokens, through append and attention; every attention against
    the definition on what the caches hold."""
    q_heads, kv_heads, dim, page_size = 8, 2, 128, 16
    g = torch.Generator().manual_seed(2200)
    table = torch.randperm(40, generator=g).to(torch.int32).view(2, 20).to(device)
    k, v = (torch.full((40, page_size, kv_heads, dim), math.nan, dtype=torch.bfloat16, device=device) for _ in range(2))
    weight = (torch.rand(dim, generator=g) + 0.5).to(device)
    held = [0, 0]
    for step, new in enumerate([[100, 37], [60, 0], [1, 90], [1, 1], [1, 1]]):
        tokens = sum(new)
        qkv = queries(2201 + step, tokens, q_heads + 2 * kv_heads, dim, device)
        position = torch.cat([torch.arange(held[b], held[b] + new[b]) for b in range(2)]).to(torch.int32).to(device)
        sequence = torch.tensor([0] * new[0] + [1] * new[1], device=device)
        slots = table[sequence, (position // page_size).long()].long() * page_size + position % page_size
        q = _kernels.qk_norm_rope_append(qkv, position, slots, k, v, q_heads=q_heads, kv_heads=kv_heads, q_weight=weight, k_weight=weight)
        held = [held[b] + new[b] for b in range(2)]
        lengths = torch.tensor(held, dtype=torch.int32, device=device)
        if new == [1, 1]:
            got = _kernels.paged_decode_attention(q, k, v, table, lengths, window=64, sinks=4)
        else:
            got = _kernels.paged_prefill_attention(q, k, v, table, lengths, starts_of(new, device), window=64, sinks=4)
        want, allowed = reference.attention_rows(q, k, v, table, held, new, window=64, sinks=4)
        assert reference.within(got, want, allowed), step


def test_captured_steps_replay_with_other_lengths(device):
    """Append and both attentions in two graphs on one stream; lengths, slots and inputs change between replays."""
    q_heads, kv_heads, dim, page_size, batch = 8, 1, 128, 16, 3
    k, v, table = reference.paged_case(2300, [1400, 900, 640], page_size=page_size, kv_heads=kv_heads, dim=dim, device=device)
    table = table[:, :88].contiguous()
    stream = torch.cuda.Stream()
    lengths = torch.tensor([1, 1, 1], dtype=torch.int32, device=device)
    qkv = queries(2301, batch, q_heads + 2 * kv_heads, dim, device)
    new = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=device)

    def step():
        position = lengths - 1
        slots = table.gather(1, (position // page_size).long()[:, None])[:, 0].long() * page_size + position % page_size
        q = _kernels.qk_norm_rope_append(qkv, position, slots, k, v, q_heads=q_heads, kv_heads=kv_heads)
        return q, _kernels.paged_decode_attention(q, k, v, table, lengths), _kernels.paged_prefill_attention(q, k, v, table, lengths, new)

    graphs = []
    with torch.cuda.stream(stream):
        step()
        torch.cuda.synchronize()
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                held = step()
            graphs.append((graph, held))
    torch.cuda.synchronize()
    for turn, held in enumerate([[3, 900, 17], [1400, 1, 640], [33, 511, 512]]):
        lengths.copy_(torch.tensor(held, dtype=torch.int32))
        qkv.copy_(queries(2310 + turn, batch, q_heads + 2 * kv_heads, dim, device))
        eager = [t.clone() for t in step()]
        torch.cuda.synchronize()
        for graph, outputs in graphs:
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outputs, eager)), turn
        want, allowed = reference.attention_rows(eager[0], k, v, table, held, [1, 1, 1])
        assert reference.within(eager[1], want, allowed) and reference.within(eager[2], want, allowed)


def test_results_repeat_bit_for_bit_on_two_streams(device):
    lengths = [5000, 3, 700, 2048]
    k, v, table = reference.paged_case(2400, lengths, page_size=16, kv_heads=2, dim=64, device=device)
    q = queries(2401, 4, 14, 64, device)
    held = torch.tensor(lengths, dtype=torch.int32, device=device)
    first = _kernels.paged_decode_attention(q, k, v, table, held)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(3):
        for stream in streams:
            with torch.cuda.stream(stream):
                outs.append(_kernels.paged_decode_attention(q, k, v, table, held))
    torch.cuda.synchronize()
    assert all(torch.equal(first, other) for other in outs)


@pytest.mark.parametrize("dim", [64, 128])
def test_divided_prefill_repeats_bit_for_bit_on_two_streams(device, dim):
    new, past = [1, 17, 0, 40], [3001, 0, 77, 2500]
    lengths = [n + p for n, p in zip(new, past)]
    k, v, table = reference.paged_case(2410, lengths, page_size=16, kv_heads=2, dim=dim, device=device)
    q = queries(2411, sum(new), 6, dim, device)
    held, starts = torch.tensor(lengths, dtype=torch.int32, device=device), starts_of(new, device)
    first = _kernels.paged_prefill_attention(q, k, v, table, held, starts)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(3):
        for stream in streams:
            with torch.cuda.stream(stream):
                outs.append(_kernels.paged_prefill_attention(q, k, v, table, held, starts))
    torch.cuda.synchronize()
    assert all(torch.equal(first, other) for other in outs)


def test_empty_batches(device):
    k, v, table = reference.paged_case(2500, [20], page_size=16, kv_heads=1, dim=64, device=device)
    none = torch.zeros(0, dtype=torch.int32, device=device)
    q = queries(2501, 0, 4, 64, device)
    assert _kernels.paged_decode_attention(q, k, v, table[:0], none).shape == (0, 4, 64)
    assert _kernels.paged_prefill_attention(q, k, v, table[:0], none, torch.zeros(1, dtype=torch.int32, device=device)).shape == (0, 4, 64)
    assert _kernels.qk_norm_rope_append(queries(2502, 0, 6, 64, device), none, none.long(), k, v, q_heads=4, kv_heads=1).shape == (0, 4, 64)
    # sequences, but a table without columns: nothing is held
    q = queries(2503, 2, 4, 64, device)
    held = torch.tensor([7, 1], dtype=torch.int32, device=device)
    assert not _kernels.paged_decode_attention(q, k, v, table[:1, :0].expand(2, 0).contiguous(), held).any()


def test_axes_of_one_element_and_shared_table_rows(device):
    # strides of axes of one element are anything; a table row may serve several sequences
    k, v, table = reference.paged_case(2550, [50], page_size=64, kv_heads=1, dim=64, device=device, spare=0)
    odd = [torch.as_strided(t.clone(), t.shape, (7, 64, 3, 1)) for t in (k, v)]
    q = queries(2551, 3, 4, 64, device)
    held = torch.tensor([50, 7, 33], dtype=torch.int32, device=device)
    rows = table[:1].expand(3, table.shape[1])
    got = _kernels.paged_decode_attention(q, *odd, rows, held)
    want, allowed = reference.attention_rows(q, k, v, rows, [50, 7, 33], [1, 1, 1])
    assert reference.within(got, want, allowed)
    one = torch.as_strided(q, (1, 4, 64), (5, 64, 1))
    starts = torch.tensor([0, 1], dtype=torch.int32, device=device)
    got = _kernels.paged_prefill_attention(one, *odd, rows[:1], held[:1], starts)
    assert reference.within(got, want[:1], allowed[:1])


def test_starts_out_of_order_write_only_rows_of_sequences(device):
    k, v, table = reference.paged_case(2560, [20, 20], page_size=16, kv_heads=1, dim=64, device=device)
    q = queries(2561, 9, 4, 64, device)
    held = torch.tensor([20, 20], dtype=torch.int32, device=device)
    out = torch.full_like(q, 3.0)
    starts = torch.tensor([5, 2, 1000], dtype=torch.int32, device=device)  # the first has none, the second rows 2 to 8
    _kernels.paged_prefill_attention(q, k, v, table, held, starts, out=out)
    want, allowed = reference.attention_rows(q[2:], k, v, table[1:], [20], [7])
    assert (out[:2] == 3).all() and reference.within(out[2:], want, allowed)


@pytest.mark.parametrize("q_heads, kv_heads, dim", [(5, 1, 128), (6, 2, 64), (40, 2, 128)])
def test_shares_of_a_long_past_join_for_rows_of_sequences_only(q_heads, kv_heads, dim, device):
    # positions divided over more workgroups than are joined at once; rows before, between and behind the sequences
    k, v, table = reference.paged_case(2580, [9001, 17], page_size=16, kv_heads=kv_heads, dim=dim, device=device)
    q = queries(2581, 9, q_heads, dim, device)
    held = torch.tensor([9001, 17], dtype=torch.int32, device=device)
    out = torch.full_like(q, 3.0)
    starts = torch.tensor([2, 5, 6], dtype=torch.int32, device=device)
    _kernels.paged_prefill_attention(q, k, v, table, held, starts, out=out)
    want, allowed = reference.attention_rows(q[2:6], k, v, table, [9001, 17], [3, 1])
    assert (out[:2] == 3).all() and (out[6:] == 3).all()
    assert reference.within(out[2:6], want, allowed)


@pytest.mark.parametrize("dim", [64, 128])
def test_few_rows_over_a_long_past_with_values_that_are_not_numbers(dim, device):
    # three tokens of two heads fill a part of one wavefront of a block; its neighbours take part in cleaning the tiles
    past, new = 4001, 3
    k, v, table = reference.paged_case(2590, [past + new], page_size=16, kv_heads=1, dim=dim, device=device)
    q = queries(2591, new, 2, dim, device)
    for position, (column, value) in {past + 1: (3, math.nan), past + 2: (4, math.inf), past - 3: (5, -math.inf)}.items():
        v[int(table[0, position // 16]), position % 16, 0, column] = value
    held, starts = (torch.tensor(x, dtype=torch.int32, device=device) for x in ([past + new], [0, new]))
    got = _kernels.paged_prefill_attention(q, k, v, table, held, starts)
    want, allowed = reference.attention_rows(q, k, v, table, [past + new], [new])
    assert torch.isnan(want[:, :, 3]).any(1).tolist() == [False, True, True] and torch.isinf(want[:, :, 4]).any(1).tolist() == [False, False, True]
    assert reference.within(got, want, allowed)


@pytest.mark.parametrize("batch, every", [(65, 1), (300, 3), (4200, 60)])
def test_prefill_finds_its_rows_among_many_sequences(batch, every, device):
    # most sequences have no new tokens
    new = [(b // every) % 3 + 1 if b % every == every - 1 else 0 for b in range(batch)]
    lengths = [n + b % 7 for b, n in enumerate(new)]
    k, v, table = reference.paged_case(2575, lengths, page_size=16, kv_heads=1, dim=64, device=device)
    q = queries(2576, sum(new), 50, 64, device)
    held = torch.tensor(lengths, dtype=torch.int32, device=device)
    got = _kernels.paged_prefill_attention(q, k, v, table, held, starts_of(new, device))
    some = [b for b in range(batch) if new[b]]
    want, allowed = reference.attention_rows(q, k, v, table[some], [lengths[b] for b in some], [new[b] for b in some])
    assert reference.within(got, want, allowed)


def test_starts_in_no_order_stay_inside(device):
    batch, tokens = 600, 70
    k, v, table = reference.paged_case(2570, [30] * batch, page_size=16, kv_heads=2, dim=64, device=device)
    room = torch.full((tokens + 40, 4, 64), 3.0, dtype=torch.bfloat16, device=device)
    q = queries(2571, tokens, 4, 64, device)
    generator = torch.Generator().manual_seed(2572)
    starts = torch.randint(-50, 200, (batch + 1,), generator=generator, dtype=torch.int32).to(device)
    held = torch.full((batch,), 30, dtype=torch.int32, device=device)
    _kernels.paged_prefill_attention(q, k, v, table, held, starts, out=room[20:-20])
    assert (room[:20] == 3).all() and (room[-20:] == 3).all() and torch.isfinite(room).all()


def refused(call, *arguments, **options):
    with pytest.raises((RuntimeError, ValueError, TypeError)):
        call(*arguments, **options)


def test_refusals(device):
    lengths = [40, 3]
    k, v, table = reference.paged_case(2600, lengths, page_size=16, kv_heads=2, dim=128, device=device)
    q = queries(2601, 2, 8, 128, device)
    held = torch.tensor(lengths, dtype=torch.int32, device=device)
    decode = _kernels.paged_decode_attention
    decode(q, k, v, table, held)
    refused(decode, q.float(), k, v, table, held)
    refused(decode, q.cpu(), k, v, table, held)
    refused(decode, q[:, :7], k, v, table, held)                      # heads not a multiple of the cache's
    refused(decode, q[:, :, :64], k, v, table, held)                  # another head size
    refused(decode, q[:1], k, v, table, held)                         # one query, two sequences
    refused(decode, q, k, v[:-1], table, held)
    refused(decode, q, k, k, table, held)                             # keys and values in one place
    refused(decode, q, k.float(), v.float(), table, held)
    refused(decode, q, k[:, :12], v[:, :12], table, held)             # pages of twelve
    refused(decode, q, k, v, table.long(), held)
    refused(decode, q, k, v, table.t().contiguous().t(), held)        # columns apart
    refused(decode, q, k, v, table, held.long())
    refused(decode, q, k, v, table, held[:1])
    for scale in (0.0, -1.0, math.nan, math.inf):
        refused(decode, q, k, v, table, held, scale=scale)
    refused(decode, q, k, v, table, held, window=-1)
    refused(decode, q, k, v, table, held, sinks=-1)
    refused(decode, q, k, v, table, held, out=q)
    wide = queries(2603, 2, 20, 128, device)
    decode(wide[:, :8], k, v, table, held, out=wide[:, 12:])          # heads of one activation beside each other
    refused(decode, wide[:, :8], k, v, table, held, out=wide[:, 6:14])  # and on each other
    refused(decode, q, k, v, table, held, out=k.flatten()[: q.numel()].view_as(q))  # into the cache
    refused(decode, q.clone().requires_grad_(), k, v, table, held)
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device=device)
    prefill = _kernels.paged_prefill_attention
    prefill(q, k, v, table, held, starts)
    refused(prefill, q, k, v, table, held, starts[:2])
    refused(prefill, q, k, v, table, held, starts.long())
    refused(prefill, q, k, v, table, held, starts, window=-2)
    refused(prefill, q, k, v, table, held, starts, out=q)
    qkv = queries(2602, 2, 12, 128, device)
    position, slots = held - 1, torch.tensor([0, 1], device=device)
    append = _kernels.qk_norm_rope_append
    options = dict(q_heads=8, kv_heads=2)
    weight = torch.ones(128, device=device)
    append(qkv, position, slots, k, v, **options)
    refused(append, qkv, position, slots, k, v, q_heads=7, kv_heads=2)
    refused(append, qkv, position, slots, k, v, q_heads=10, kv_heads=1)
    refused(append, qkv, position.long(), slots, k, v, **options)
    refused(append, qkv, position, slots.int(), k, v, **options)
    refused(append, qkv, position, slots, k, v, q_weight=weight, **options)
    refused(append, qkv, position, slots, k, v, q_weight=weight, k_weight=weight.bfloat16(), **options)
    refused(append, qkv, position, slots, k, v, q_weight=weight[:64], k_weight=weight[:64], **options)
    for rotary in (8, 136, -16, 120):
        refused(append, qkv, position, slots, k, v, rotary_dim=rotary, **options)
    for theta in (0.0, -5.0, math.nan):
        refused(append, qkv, position, slots, k, v, theta=theta, **options)
    refused(append, qkv, position, slots, k, v, epsilon=-1.0, **options)
    refused(append, qkv, position, slots, k, v, out=qkv[:, 1:9], **options)
    refused(append, k.flatten()[: qkv.numel()].view_as(qkv), position, slots, k, v, **options)
    refused(append, qkv, position, slots, k, v, out=torch.empty(2, 7, 128, dtype=torch.bfloat16, device=device), **options)


def test_tensors_written_in_place_move_their_version(device):
    """Another operation's backward must not read what an append or attention has overwritten."""
    k, v, table = reference.paged_case(2620, [40, 3], page_size=16, kv_heads=2, dim=64, device=device, poison=False)
    qkv = queries(2621, 2, 8, 64, device)
    held = torch.tensor([40, 3], dtype=torch.int32, device=device)
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device=device)
    slots = torch.tensor([5, 6], device=device)
    append, decode, prefill = _kernels.qk_norm_rope_append, _kernels.paged_decode_attention, _kernels.paged_prefill_attention
    q = append(qkv, held - 1, slots, k, v, q_heads=4, kv_heads=2).clone()
    calls = {
        "keys": (k, lambda: append(qkv, held - 1, slots, k, v, q_heads=4, kv_heads=2)),
        "values": (v, lambda: append(qkv, held - 1, slots, k, v, q_heads=4, kv_heads=2)),
        "in place": (qkv, lambda: append(qkv, held - 1, slots, k, v, q_heads=4, kv_heads=2, out=qkv[:, :4])),
        "decode": (torch.zeros_like(q),) * 2, "prefill": (torch.zeros_like(q),) * 2,
    }
    calls["decode"] = (calls["decode"][0], lambda: decode(q, k, v, table, held, out=calls["decode"][0]))
    calls["prefill"] = (calls["prefill"][0], lambda: prefill(q, k, v, table, held, starts, out=calls["prefill"][0]))
    for name, (written, call) in calls.items():
        factor = torch.ones_like(written, requires_grad=True)
        product = factor * written  # keeps `written` for its backward
        before = written._version
        with torch.no_grad():
            call()
        assert written._version > before, name
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            product.sum().backward()
    # what is only read, and what a call makes, stays as it was
    versions = [t._version for t in (q, k, v, table, held)]
    assert decode(q, k, v, table, held)._version == 0 and prefill(q, k, v, table, held, starts)._version == 0
    assert versions == [t._version for t in (q, k, v, table, held)]
    with torch.inference_mode():
        k2, v2, qkv2, out = k.clone(), v.clone(), qkv.clone(), torch.zeros_like(q)
        decode(append(qkv2, held - 1, slots, k2, v2, q_heads=4, kv_heads=2), k2, v2, table, held, out=out)
    # tensors of inference mode have no version; they are written outside of it as before
    again = decode(append(qkv2, held - 1, slots, k2, v2, q_heads=4, kv_heads=2), k2, v2, table, held, out=out)
    assert again.data_ptr() == out.data_ptr()


def test_the_c_entry_refuses_a_small_or_missing_workspace(device):
    lengths = [2000]
    k, v, table = reference.paged_case(2700, lengths, page_size=16, kv_heads=1, dim=64, device=device)
    q = queries(2701, 1, 4, 64, device)
    out = torch.zeros_like(q)
    held = torch.tensor(lengths, dtype=torch.int32, device=device)
    native = _native.context(device)
    cache = _native.PagedCache(k.data_ptr(), v.data_ptr(), *k.stride()[:3], *k.shape)
    columns = table.shape[1]
    size = _native.library().camblas_cuda_paged_decode_workspace_size(native.handle, 1, 4, ct.byref(cache), columns, 0, 0)
    assert size > 0
    room = torch.empty(size + 16, dtype=torch.uint8, device=device)

    def call(address, count):
        native.call("paged_decode_attention", 1, 4, ct.byref(cache), table.data_ptr(), columns, columns, held.data_ptr(), 0, 0, 0.125,
                    q.data_ptr(), 256, address, count, out.data_ptr(), 256)

    for address, count in ((None, size), (room.data_ptr(), size - 1), (room.data_ptr() + 4, size)):
        with pytest.raises(RuntimeError, match="workspace"):
            call(address, count)
    assert not out.any()
    call(room.data_ptr(), size)
    want, allowed = reference.attention_rows(q, k, v, table, lengths, [1])
    assert reference.within(out, want, allowed)
