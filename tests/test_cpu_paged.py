"""The paged cache without a GPU: the arithmetic its kernels share (compiled for the CPU), checked position by
position; refusals that need no device; the bounds the tests' own reference gives."""

import ctypes as ct
import random
import subprocess
from pathlib import Path

import pytest
import torch

import paged_reference as reference
from camblas_amd import _kernels, _native

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    target = tmp_path_factory.mktemp("paged") / "paged_span_host.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-shared", "-fPIC", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    f"-I{ROOT / 'camblas_amd' / 'csrc'}", str(ROOT / "tests" / "support" / "paged_span_host.cpp"), "-o", str(target)],
                   check=True)
    lib = ct.CDLL(str(target))
    for name in ("find_row", "find_share_begin", "find_share"):
        getattr(lib, name).restype = ct.c_int64
    lib.find_row.argtypes = [ct.c_int64, ct.c_int64, ct.c_int, ct.c_int, ct.c_int]
    lib.find_share_begin.argtypes = lib.find_share.argtypes = [ct.c_int64] * 3
    return lib


@pytest.mark.parametrize("tile", [32, 64])
@pytest.mark.parametrize("seed", range(6))
def test_tiles_hold_every_seen_position_once(host, tile, seed):
    rng = random.Random(seed)
    room = (ct.c_int * 4096)()
    for _ in range(150):
        first = rng.choice([-5, -1, 0, 1, 31, 32, 63, 64, rng.randint(0, 900)])
        last = first + rng.choice([0, 0, 1, 15, 40])
        window = rng.choice([0, 1, 2, 32, 63, 64, 65, rng.randint(1, 900), 2**30])
        sinks = rng.choice([0, 1, 31, 32, 64, 65, rng.randint(0, 900), 2**30])
        count = host.span_tiles(tile, window, sinks, first, last, room, 4096)
        starts = list(room[:count])
        assert starts == sorted(set(starts)) and all(s % tile == 0 and 0 <= s <= last for s in starts)
        for query in range(first, last + 1):
            for position in range(max(0, last + tile)):
                if host.is_seen(window, sinks, query, position):
                    assert position // tile * tile in starts
        # no tile that nobody sees a position of
        for s in starts:
            assert any(host.is_seen(window, sinks, q, p) for q in range(max(first, 0), last + 1) for p in range(s, s + tile))


def test_clipping_changes_nothing_that_is_seen(host):
    room = (ct.c_int * 2)()
    for capacity in (1, 16, 40):
        for window in (0, 1, capacity - 1, capacity, capacity + 1, 2**31 - 1):
            for sinks in (0, 1, capacity, 2**31 - 1):
                host.clip(window, sinks, ct.c_int64(capacity), room)
                assert 0 <= room[0] < max(capacity, 1) and 0 <= room[1] <= capacity
                for query in range(capacity):
                    assert ([bool(host.is_seen(room[0], room[1], query, p)) for p in range(capacity)]
                            == [p in reference.visible_positions(query, window, sinks) for p in range(capacity)])


def test_what_a_query_sees(host):
    for window, sinks in ((0, 0), (0, 9), (5, 0), (5, 3), (1, 1), (100, 100)):
        for query in range(30):
            seen = [p for p in range(40) if host.is_seen(window, sinks, query, p)]
            assert seen == reference.visible_positions(query, window, sinks)


@pytest.mark.parametrize("shift", [0, 4, 8])
def test_bad_pages_and_lengths(host, shift):
    row = (ct.c_int32 * 5)(3, -1, 7, -2**31, 6)
    size = 1 << shift
    wanted = [3, -1, -1, -1, 6, -1, -1]  # seven pages; two columns behind the table
    for position in range(7 * size):
        assert host.find_page(row, 5, 7, shift, position) == wanted[position // size]
    assert host.find_page(row, 0, 7, shift, 0) == -1
    assert [host.find_length(n, 5, shift) for n in (-2**31, -1, 0, 1, 5 * size, 5 * size + 1, 2**31 - 1)] == [0, 0, 0, 1, 5 * size, 5 * size, 5 * size]


def test_row_offsets_beyond_32_bits(host):
    page_stride, slot_stride = 16 * 1024, 1024
    for page in (0, 1, 2**17, 2**20, 2**31 - 1):
        for position in (0, 15, 16, 2**30 - 1):
            assert host.find_row(page_stride, slot_stride, 4, page, position) == page * page_stride + position % 16 * slot_stride


@pytest.mark.parametrize("workers", [1, 7, 512])
def test_steps_dealt_to_workgroups(host, workers):
    for all_steps in (workers, workers + 1, 3 * workers - 1, 1000 + workers, 2**40 + 12345):
        begins = [host.find_share_begin(all_steps, workers, g) for g in range(workers + 1)]
        assert begins[0] == 0 and begins[-1] == all_steps and all(b > a for a, b in zip(begins, begins[1:]))
        for g in range(workers):
            assert host.find_share(all_steps, workers, begins[g]) == g == host.find_share(all_steps, workers, begins[g + 1] - 1)


def test_numbers_of_row_blocks(host):
    rng = random.Random(3)
    for _ in range(200):
        group, rows = rng.choice([1, 3, 7, 8, 16, 200]), 128
        counts = [rng.choice([0, 1, 5, 16, 17, 43, 200]) for _ in range(rng.randint(1, 12))]
        starts = [sum(counts[:b]) for b in range(len(counts) + 1)]
        first = [host.find_first_block(t, group, rows, b) for b, t in enumerate(starts)]
        used = set()
        for b, count in enumerate(counts):
            needed = -(-count * group // rows)
            assert first[b] + needed <= first[b + 1]
            assert not used & set(range(first[b], first[b] + needed))
            used |= set(range(first[b], first[b] + needed))
        assert first[-1] == starts[-1] * group // rows + len(counts) and all(n < first[-1] for n in used)


def test_rows_that_share_memory(host):
    rng = random.Random(4)
    host.find_apart.argtypes = [ct.c_int64] * 8
    seen = set()
    for _ in range(3000):
        stride = rng.choice([4, 8, 12])
        a, b = ([rng.randint(0, 30), rng.randint(0, 3), rng.randint(1, 6), rng.choice([stride, stride, stride, 5])] for _ in range(2))
        cells = [{x[0] + r * x[3] + i for r in range(x[1]) for i in range(x[2])} for x in (a, b)]
        apart = bool(host.find_apart(*a, *b))
        if apart:
            assert not cells[0] & cells[1]
        elif a[3] == b[3] and a[2] <= stride and b[2] <= stride and a[1] > 1 and b[1] > 1 and a[1] == b[1]:
            # rows of one stride that are refused share an element, at least were both to go on
            go_on = [{x[0] + r * x[3] + i for r in range(-12, 12) for i in range(x[2])} for x in (a, b)]
            assert go_on[0] & go_on[1]
        seen.add(apart)
    assert seen == {True, False}
    assert host.find_apart(0, 5, 8, 24, 8, 5, 8, 24) and not host.find_apart(0, 5, 8, 24, 7, 5, 8, 24)


def test_tensors_without_a_gpu_are_refused():
    q, cache = torch.zeros(2, 4, 64, dtype=torch.bfloat16), torch.zeros(3, 16, 2, 64, dtype=torch.bfloat16)
    table, lengths = torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        _kernels.paged_decode_attention(q, cache, cache.clone(), table, lengths)
    with pytest.raises(ValueError):
        _kernels.paged_prefill_attention(q, cache, cache.clone(), table, lengths, torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError):
        _kernels.qk_norm_rope_append(torch.zeros(2, 8, 64, dtype=torch.bfloat16), lengths, lengths.long(), cache, cache.clone(), q_heads=4, kv_heads=2)


def test_the_c_entries_refuse_a_missing_context():
    lib = _native.library()
    cache = _native.PagedCache()
    described = ct.byref(cache)
    assert lib.camblas_cuda_paged_decode_workspace_size(None, 1, 1, described, 1, 0, 0) == 0
    assert lib.camblas_cuda_paged_prefill_workspace_size(None, 1, 1, 1, described, 1, 0, 0) == 0
    assert lib.camblas_cuda_qk_norm_rope_append(None, 1, 1, 64, 1e4, 0, 1e-6, None, None, None, None, None, 64, None, 64, described) == -1
    assert lib.camblas_cuda_paged_decode_attention(None, 1, 1, described, None, 1, 1, None, 0, 0, 1.0, None, 64, None, 0, None, 64) == -1
    assert lib.camblas_cuda_paged_prefill_attention(None, 1, 1, 1, described, None, 1, 1, None, None, 0, 0, 1.0, None, 64, None, 0, None, 64) == -1
    assert b"missing context" in lib.camblas_cuda_error(None)


def test_the_reference_agrees_with_a_dense_softmax():
    g = torch.Generator().manual_seed(5)
    k, v, table = reference.paged_case(6, [50], page_size=8, kv_heads=2, dim=64, device="cpu")
    q = torch.randn(1, 4, 64, generator=g).to(torch.bfloat16)
    got, allowed = reference.attention_rows(q, k, v, table, [50], [1])
    flat = [t[table[0, :7].long()].reshape(-1, 2, 64)[:50].double().repeat_interleave(2, 1) for t in (k, v)]
    weight = torch.softmax(torch.einsum("hd,phd->hp", q[0].double(), flat[0]) / 8, 1)
    assert torch.allclose(got[0], torch.einsum("hp,phd->hd", weight, flat[1]), rtol=0, atol=1e-12)
    # a rounding of the output alone is allowed, one of twice that size is not
    assert reference.within(got.to(torch.bfloat16), got, allowed)
    assert not reference.within(got + 3 * allowed, got, allowed)


def test_the_append_with_a_wide_base_refuses_a_missing_context():
    lib = _native.library()
    described = ct.byref(_native.PagedCache())
    assert lib.camblas_cuda_qk_norm_rope_append_wide_theta(None, 1, 1, 64, 1e4, 0, 1e-6, None, None, None, None, None, 64, None, 64, described) == -1
    assert b"missing context" in lib.camblas_cuda_error(None)


def test_caches_whose_rows_share_memory(host):
    number = ct.c_int64 * 3
    host.find_places_apart.argtypes = [number, number, ct.c_int64, ct.c_int64]
    for at, (k, v, apart) in enumerate(reference.cache_layouts()):
        offset = (v.data_ptr() - k.data_ptr()) // 2
        assert bool(host.find_places_apart(number(*k.shape[:3]), number(*k.stride()[:3]), k.shape[3], offset)) == apart, at
    # any strides at all, element by element
    rng, seen = random.Random(7), set()
    for _ in range(4000):
        counts = [rng.choice([1, 1, 2, 3, 4]) for _ in range(3)]
        width = rng.choice([1, 2, 3])
        strides = [rng.randint(1, 30) for _ in range(3)]
        offset = rng.randint(-60, 60)
        rows = [a * strides[0] + b * strides[1] + c * strides[2] for a in range(counts[0]) for b in range(counts[1]) for c in range(counts[2])]
        cells = [r + i + o for o in (0, offset) for r in rows for i in range(width)]
        apart = bool(host.find_places_apart(number(*counts), number(*strides), width, offset))
        assert apart == (len(set(cells)) == len(cells)), (counts, strides, width, offset)
        seen.add(apart)
    assert seen == {True, False}
    # the largest that an entry lets through: no overflow, and an end
    for strides in ((2**31 - 8, 2**32, 2**32), (128, 128 * 2**16, 128), (2**16 * 128, 8 * 17, 128)):
        host.find_places_apart(number(2**15, 2**16, 2**16), number(*strides), 128, 2**46)
