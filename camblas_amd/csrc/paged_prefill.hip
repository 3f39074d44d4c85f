// Attention of the new tokens of ragged sequences over their pages: out = softmax(scale q K^T) V, every
// token over the positions up to its own (optionally a window and the first tokens only), grouped query
// heads, BF16 storage.
//
// A workgroup takes rows (token, query head of one key-value head) of one sequence, the heads of a token
// next to each other, and walks the positions they see in tiles of 64. The query heads of a group share the
// keys and values they read, and few tokens lie on the diagonal of a tile. Both products run on
// v_mfma_f32_32x32x16_bf16 with the rows as columns:
//   scores  S[position, row] = K[position, :] . Q[row, :]
//   output  O[dim, row]      = V[position, dim]^T . P[position, row]
// so that a lane holds one row: its maximum, its sum and the factor its outputs are rescaled by are the
// lane's own (two lanes share a row and exchange their maximum), and what the first product leaves in a lane
// is an operand of the second as it stands, once the order of that product's K index is taken to be the
// order of the positions in the lane. V is then wanted with the positions of a dim together; it lies in LDS
// as rows and is gathered by transposing reads (ds_read_b64_tr_b16: within sixteen lanes, lane s points at
// row s / 4 of four rows, values 4 (s % 4) .. + 3, and receives the four values of column s).
//
// Rows of K and V pass through registers into LDS, a tile ahead of the products. The maximum that weights
// refer to is moved only when a score exceeds it by 2^8; weights are rounded to BF16 for the second product,
// their sum is kept in FP32.
#include "common.hpp"
#include "device.hpp"
#include "dma.hpp"
#include "paged_cache.hpp"

namespace camblas_hip
{
namespace
{
constexpr int WAVES = 4, THREADS = WAVES * 64, ROWS = WAVES * 32, TILE = 64;
constexpr int VECTOR = 0x2, MATRIX = 0x8, DS_READS = 0x100; // kinds of instructions for the scheduler
constexpr float LOG2E = 1.4426950408889634f;

struct PrefillParams {
    int batch, tokens, group, row_blocks;
    PagedCache cache;
    PageTable table;
    Visibility see;
    const int32_t *starts; // [batch + 1]: first token of each sequence
    float scale;           // times log2(e)
    const unsigned short *q;
    unsigned short *out;
    int64_t q_stride, out_stride;
};

typedef short i16x4_t __attribute__((ext_vector_type(4)));
typedef short i16x8_t __attribute__((ext_vector_type(8)));
__device__ __forceinline__ i16x4_t gather_column(const unsigned char *address)
{
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4_t *)(address));
}

// Which 16-byte chunk of a tile's row lies at place `chunk`: the rows are turned so that reads meet no bank
// twice. Keys are read as 16 rows of one chunk, values by transposing reads of 64 bytes of four rows.
template <int DIM> __device__ __forceinline__ int turn_keys(int row)
{
    return DIM == 128 ? row & 15 : ((row >> 1) & 7) ^ ((row & 1) << 2);
}
template <int DIM> __device__ __forceinline__ int turn_values(int row)
{
    return DIM == 128 ? 4 * (row & 3) : 4 * ((row >> 1) & 1);
}

// Loads to LDS outside the compiler's bookkeeping, complete after a wait for vmcnt that the caller places:
// 16 bytes per lane and load, load i to `to` + 1024 i + 16 * lane. M0 is put back as it was; a load to LDS
// needs a wait state after a write of M0, and five after a vector instruction wrote the scalar registers of
// its address, which the compiler, not looking into the text, does not see to.
// The first form reads from base (the same in every lane) + a lane's own offsets in bytes.
template <int LOADS> __device__ __forceinline__ void fetch_rows(const unsigned short *base, const unsigned (&offset)[LOADS], const void *to)
{
    static_assert(LOADS == 2 || LOADS == 4, "a wavefront's share of a tile");
    const uintptr_t address = reinterpret_cast<uintptr_t>(base);
    const uint64_t uniform = (uint64_t(unsigned(__builtin_amdgcn_readfirstlane(unsigned(address >> 32)))) << 32) |
                             unsigned(__builtin_amdgcn_readfirstlane(unsigned(address)));
    const unsigned lds = __builtin_amdgcn_readfirstlane(static_cast<unsigned>(reinterpret_cast<uintptr_t>(to)));
    unsigned saved;
    if constexpr (LOADS == 4)
        asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 4\n\t"
                     "global_load_lds_dwordx4 %2, %6\n\ts_add_u32 m0, m0, 0x400\n\ts_nop 0\n\t"
                     "global_load_lds_dwordx4 %3, %6\n\ts_add_u32 m0, m0, 0x400\n\ts_nop 0\n\t"
                     "global_load_lds_dwordx4 %4, %6\n\ts_add_u32 m0, m0, 0x400\n\ts_nop 0\n\t"
                     "global_load_lds_dwordx4 %5, %6\n\ts_mov_b32 m0, %0\n\ts_nop 0"
                     : "=&s"(saved)
                     : "s"(lds), "v"(offset[0]), "v"(offset[1]), "v"(offset[LOADS - 2]), "v"(offset[LOADS - 1]), "s"(uniform)
                     : "memory", "scc");
    else
        asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 4\n\t"
                     "global_load_lds_dwordx4 %2, %4\n\ts_add_u32 m0, m0, 0x400\n\ts_nop 0\n\t"
                     "global_load_lds_dwordx4 %3, %4\n\ts_mov_b32 m0, %0\n\ts_nop 0"
                     : "=&s"(saved)
                     : "s"(lds), "v"(offset[0]), "v"(offset[1]), "s"(uniform)
                     : "memory", "scc");
}
// One load from a lane's own address.
__device__ __forceinline__ void fetch_row(const unsigned short *address, const void *to)
{
    const unsigned lds = __builtin_amdgcn_readfirstlane(static_cast<unsigned>(reinterpret_cast<uintptr_t>(to)));
    unsigned saved;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\t"
                 "global_load_lds_dwordx4 %2, off\n\ts_mov_b32 m0, %0\n\ts_nop 0"
                 : "=&s"(saved)
                 : "s"(lds), "v"(address)
                 : "memory");
}

// the bits below bit `count`
__device__ __forceinline__ uint64_t below(int count)
{
    return count <= 0 ? 0 : count >= 64 ? ~uint64_t(0) : (uint64_t(1) << count) - 1;
}

// a value that is the same in every lane, in a scalar register
__device__ __forceinline__ int uniform(int value) { return __builtin_amdgcn_readfirstlane(value); }

__device__ __forceinline__ int first_token(const PrefillParams &p, int sequence)
{
    return min(max(p.starts[sequence], 0), p.tokens);
}

template <int DIM> __global__ __launch_bounds__(THREADS, DIM == 64 ? 3 : 2) void paged_prefill_kernel(PrefillParams p)
{
    constexpr int CHUNKS = DIM / 8, FETCH = 64 / CHUNKS, FETCHES = TILE / FETCH / WAVES; // rows of a load, a wavefront's loads
    __shared__ __attribute__((aligned(16))) unsigned char keys0[TILE * DIM * 2], keys1[TILE * DIM * 2];
    __shared__ __attribute__((aligned(16))) unsigned char values0[TILE * DIM * 2], values1[TILE * DIM * 2];
    __shared__ int found;
    const int thread = threadIdx.x, lane = thread % 64, wave = uniform(thread / 64);
    const int column = lane % 32, half = lane / 32;
    // the last blocks of a causal sequence see most: they start first
    const int kv_head = int(blockIdx.x) % p.cache.kv_heads;
    const int block = p.row_blocks - 1 - int(blockIdx.x) / p.cache.kv_heads;

    // Blocks of sequence b are numbered from floor(first token * group / ROWS) + b: a number that needs no
    // sum over the sequences before, leaves room for a last block that is not full, and at most one unused
    // number per sequence.
    if (thread == 0)
        found = 0;
    __syncthreads();
    for (int b = thread; b < p.batch; b += THREADS) {
        const int64_t here = int64_t(first_token(p, b)) * p.group / ROWS + b;
        const int64_t next = int64_t(first_token(p, b + 1)) * p.group / ROWS + b + 1;
        if (here <= block && block < next)
            found = b;
    }
    __syncthreads();
    const int sequence = __builtin_amdgcn_readfirstlane(found);
    const int token0 = uniform(first_token(p, sequence)), tokens = uniform(first_token(p, sequence + 1)) - token0;
    const int64_t row0 = (block - (int64_t(token0) * p.group / ROWS + sequence)) * ROWS;
    const int64_t rows = int64_t(tokens) * p.group - row0;
    if (row0 < 0 || rows <= 0)
        return;

    // ---- this lane's row: token and query head, position
    const int past = uniform(live_positions(p.table, p.cache, sequence)) - tokens;
    int query;
    bf16x8_t q[DIM / 16];
    {
        const int64_t row = row0 + wave * 32 + column;
        const int64_t kept = row < rows + row0 ? row : rows + row0 - 1;
        const int token = int(kept / p.group), head = kv_head * p.group + int(kept % p.group);
        query = past + token;
        const unsigned short *from = p.q + int64_t(token0 + token) * p.q_stride + int64_t(head) * DIM + 8 * half;
#pragma unroll
        for (int s = 0; s < DIM / 16; ++s)
            q[s] = *reinterpret_cast<const bf16x8_t *>(from + 16 * s);
    }
    const int first_query = uniform(past + int(row0 / p.group));
    const int last_query = uniform(past + int((row0 + min(rows, int64_t(ROWS)) - 1) / p.group));
    const TileSpan<TILE> span(p.see, first_query, last_query);

    // ---- fetching tiles: lane r of every wavefront knows the page of tile row r
    const int32_t *pages = p.table.pages + int64_t(sequence) * p.table.stride;
    const auto page_at = [&](int tile) {
        return tile < span.tiles ? page_of(p.cache, pages, p.table.columns, span.position(tile) + lane) : -1;
    };
    // which rows of a tile exist and are seen by some query of the block
    const auto wanted_rows = [&](int tile, int page) {
        const int position = span.position(tile) + lane;
        return __ballot(page >= 0 && position <= last_query &&
                        (p.see.window <= 0 || position > first_query - p.see.window || position < p.see.sinks));
    };
    // A wavefront brings rows 16 * wave .. + 15, FETCH of them with a load, in the order of their turned chunks. Where
    // pages hold at least 16 rows those lie in one page, at offsets that are the same for every tile.
    const int own_row = 16 * wave;
    const bool one_page = (16 >> p.cache.page_shift) <= 1 && p.cache.slot_stride < (int64_t(1) << 26);
    const int64_t head_at = int64_t(kv_head) * p.cache.head_stride;
    unsigned key_from[FETCHES], value_from[FETCHES]; // bytes
#pragma unroll
    for (int i = 0; i < FETCHES; ++i) {
        const int r = FETCH * i + lane / CHUNKS;
        const unsigned along = one_page ? unsigned(r) * unsigned(p.cache.slot_stride) * 2 : 0;
        key_from[i] = along + unsigned((lane % CHUNKS) ^ turn_keys<DIM>(r)) * 16;
        value_from[i] = along + unsigned((lane % CHUNKS) ^ turn_values<DIM>(r)) * 16;
    }
    // where the wavefront's first row of a tile lies (a row that does not exist: some row that does, and is not used)
    const auto place = [&](int tile, int page) {
        return row_offset(p.cache, max(__builtin_amdgcn_readlane(page, own_row), 0), span.position(tile) + own_row) + head_at;
    };
    const auto fetch = [&](const unsigned short *array, const unsigned (&from)[FETCHES], int64_t at, int tile, int page,
                           unsigned char *to) {
        if (one_page) { // (uniform)
            fetch_rows(array + at, from, to + own_row * DIM * 2);
        } else {
#pragma unroll
            for (int i = 0; i < FETCHES; ++i) {
                const int r = own_row + FETCH * i + lane / CHUNKS;
                const int64_t own = row_offset(p.cache, max(__shfl(page, r), 0), span.position(tile) + r) + head_at;
                fetch_row(array + own + from[i] / 2, to + (own_row + FETCH * i) * DIM * 2);
            }
        }
    };

    // ---- reading tiles
    int key_at[DIM / 16], value_at[DIM / 32]; // byte offsets of this lane's operands
#pragma unroll
    for (int s = 0; s < DIM / 16; ++s)
        key_at[s] = column * DIM * 2 + ((2 * s + half) ^ turn_keys<DIM>(column)) * 16;
    {
        const int spot = 4 * half + lane % 16 / 4; // (position 16 u + spot, and eight further)
#pragma unroll
        for (int d = 0; d < DIM / 32; ++d) {
            const int dim = 32 * d + 16 * (lane / 16 % 2) + 4 * (lane % 4);
            value_at[d] = spot * DIM * 2 + ((dim / 8) ^ turn_values<DIM>(spot)) * 16 + dim % 8 * 2;
        }
    }
    const auto multiply_keys = [&](const unsigned char *tile, f32x16_t (&score)[2]) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int r = 0; r < 16; ++r)
                score[t][r] = 0.f;
#pragma unroll
            for (int s = 0; s < DIM / 16; ++s) {
                const bf16x8_t k = *reinterpret_cast<const bf16x8_t *>(tile + key_at[s] + 32 * t * DIM * 2);
                score[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k, q[s], score[t], 0, 0, 0);
            }
        }
    };

    f32x16_t acc[DIM / 32];
    float top = -INFINITY, total = 0.f;
#pragma unroll
    for (int d = 0; d < DIM / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r)
            acc[d][r] = 0.f;

    // Turn `tile`: its scores are in `score`, its values in `values`, the keys of the next tile in `next_keys`.
    // Fetched meanwhile: the next tile's values, the keys of the one after. The next tile's scores are multiplied
    // while this one's weights are worked out.
    uint64_t wanted;
    int page, next_page; // of the rows of the next tile and of the one after
    int64_t at = 0;      // place() of the next tile
    const auto turn = [&](int tile, f32x16_t (&score)[2], f32x16_t (&next_score)[2], unsigned char *keys,
                          const unsigned char *next_keys, unsigned char *values, unsigned char *next_values) {
        const int base = span.position(tile);
        const uint64_t next_wanted = wanted_rows(tile + 1, page);
        if (tile + 1 < span.tiles)
            fetch(p.cache.v, value_from, at, tile + 1, page, next_values);
        page = next_page;
        if (tile + 2 < span.tiles) {
            at = place(tile + 2, page);
            fetch(p.cache.k, key_from, at, tile + 2, page, keys);
        }
        next_page = page_at(tile + 3);
        const bool whole = wanted == ~uint64_t(0) && base + TILE - 1 <= first_query &&
                           (p.see.window <= 0 || base > last_query - p.see.window || base + TILE <= p.see.sinks);
        if (!whole) { // (the same in every wavefront)
            // bit n: the lane's query sees position base + n
            uint64_t seen = wanted & below(query - base + 1);
            if (p.see.window > 0)
                seen &= ~below(query - base + 1 - p.see.window) | below(p.see.sinks - base);
            seen >>= 4 * half;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    // (all bits of a lane's own bit, and a bitwise choice: no masks in scalar registers)
                    const int keep = __builtin_amdgcn_sbfe(int(seen >> (32 * t)), 8 * (r / 4) + r % 4, 1);
                    score[t][r] = __int_as_float((__float_as_int(score[t][r]) & keep) | (int(0xff800000u) & ~keep));
                }
            // rows that nobody sees: zeros, which no weight turns into NaN
            for (int piece = thread; piece < TILE * CHUNKS; piece += THREADS)
                if (!((wanted >> (piece / CHUNKS)) & 1))
                    *reinterpret_cast<u32x4_t *>(values + piece * 16) = u32x4_t{0, 0, 0, 0};
            __syncthreads();
        }
        float highest = -INFINITY;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                highest = fmaxf(highest, score[t][r]);
        highest *= p.scale;
        if (__any(highest > top + 8.f)) {
            highest = fmaxf(highest, __shfl_xor(highest, 32));
            highest = fmaxf(highest, top);
            const float factor = top == highest ? 1.f : __builtin_amdgcn_exp2f(top - highest);
            top = highest;
            total *= factor;
#pragma unroll
            for (int d = 0; d < DIM / 32; ++d)
                acc[d] *= factor;
        }
        const float reference = top == -INFINITY ? 0.f : top;
        multiply_keys(next_keys, next_score);
        bf16x8_t weights[4];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                score[t][r] = __builtin_amdgcn_exp2f(fmaf(score[t][r], p.scale, -reference));
                total += score[t][r];
            }
#pragma unroll
            for (int u = 0; u < 2; ++u)
                weights[2 * t + u] = __builtin_bit_cast(
                    bf16x8_t, u32x4_t{round_pair(score[t][8 * u], score[t][8 * u + 1]),
                                      round_pair(score[t][8 * u + 2], score[t][8 * u + 3]),
                                      round_pair(score[t][8 * u + 4], score[t][8 * u + 5]),
                                      round_pair(score[t][8 * u + 6], score[t][8 * u + 7])});
        }
#pragma unroll
        for (int u = 0; u < TILE / 16; ++u)
#pragma unroll
            for (int d = 0; d < DIM / 32; ++d) {
                const i16x4_t lower = gather_column(values + value_at[d] + 16 * u * DIM * 2);
                const i16x4_t upper = gather_column(values + value_at[d] + (16 * u + 8) * DIM * 2);
                const bf16x8_t v = __builtin_bit_cast(
                    bf16x8_t, i16x8_t{lower[0], lower[1], lower[2], lower[3], upper[0], upper[1], upper[2], upper[3]});
                acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, weights[u], acc[d], 0, 0, 0);
            }
        // The order asked of the compiler: every matrix instruction is followed by vector instructions that fill
        // its 32 cycles and by the reads of an operand to come (left alone it put the products of the scores in a
        // row: 2264 against 2177 us at 2048 tokens after 30001).
        __builtin_amdgcn_sched_group_barrier(DS_READS, 4, 0);
#pragma unroll
        for (int i = 0; i < 2 * DIM / 16; ++i) {
            __builtin_amdgcn_sched_group_barrier(MATRIX, 1, 0);
            __builtin_amdgcn_sched_group_barrier(DS_READS, 1, 0);
            __builtin_amdgcn_sched_group_barrier(VECTOR, 5, 0);
        }
#pragma unroll
        for (int i = 0; i < TILE / 16 * DIM / 32; ++i) {
            __builtin_amdgcn_sched_group_barrier(MATRIX, 1, 0);
            __builtin_amdgcn_sched_group_barrier(DS_READS, 2, 0);
            __builtin_amdgcn_sched_group_barrier(VECTOR, 2, 0);
        }
        wanted = next_wanted;
        asm volatile("" ::: "memory");
        pipeline_barrier<0>();
        asm volatile("" ::: "memory");
    };

    if (span.tiles > 0) {
        page = page_at(0);
        wanted = wanted_rows(0, page);
        at = place(0, page);
        fetch(p.cache.k, key_from, at, 0, page, keys0);
        fetch(p.cache.v, value_from, at, 0, page, values0);
        page = page_at(1);
        next_page = page_at(2);
        if (span.tiles > 1) {
            at = place(1, page);
            fetch(p.cache.k, key_from, at, 1, page, keys1);
        }
        pipeline_barrier<0>();
        asm volatile("" ::: "memory");
        f32x16_t even[2], odd[2];
        multiply_keys(keys0, even);
        asm volatile("" ::: "memory");
        pipeline_barrier<0>();
        asm volatile("" ::: "memory");
        for (int tile = 0; tile < span.tiles; tile += 2) {
            turn(tile, even, odd, keys0, keys1, values0, values1);
            if (tile + 1 >= span.tiles)
                break;
            turn(tile + 1, odd, even, keys1, keys0, values1, values0);
        }
    }

    const int64_t row = row0 + wave * 32 + column;
    const float sum = total + __shfl_xor(total, 32);
    if (row >= row0 + rows)
        return;
    // (no position seen: zero; a sum that is NaN stays NaN)
    const float inverse = sum == 0.f ? 0.f : 1.f / sum;
    const int token = token0 + int(row / p.group), head = kv_head * p.group + int(row % p.group);
    unsigned short *to = p.out + int64_t(token) * p.out_stride + int64_t(head) * DIM + 4 * half;
#pragma unroll
    for (int d = 0; d < DIM / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *reinterpret_cast<u32x2_t *>(to + 32 * d + 8 * g) =
                u32x2_t{round_pair(acc[d][4 * g] * inverse, acc[d][4 * g + 1] * inverse),
                        round_pair(acc[d][4 * g + 2] * inverse, acc[d][4 * g + 3] * inverse)};
}
} // namespace

hipError_t launch_paged_prefill(hipStream_t stream, int batch, int tokens, int q_heads, int dim, const PagedCache &cache,
                                const PageTable &table, const Visibility &see, const int32_t *starts, float scale,
                                const void *q, int64_t q_stride, void *out, int64_t out_stride, int compute_units)
{
    PrefillParams p = {};
    p.batch = batch;
    p.tokens = tokens;
    p.group = q_heads / cache.kv_heads;
    const int64_t blocks = int64_t(tokens) * p.group / ROWS + batch;
    if (blocks * cache.kv_heads > INT32_MAX)
        return hipErrorInvalidValue;
    p.row_blocks = int(blocks);
    p.cache = cache;
    p.table = table;
    p.see = see;
    p.starts = starts;
    p.scale = scale * LOG2E;
    p.q = static_cast<const unsigned short *>(q);
    p.out = static_cast<unsigned short *>(out);
    p.q_stride = q_stride;
    p.out_stride = out_stride;
    const unsigned grid = unsigned(blocks * cache.kv_heads);
    if (dim == 128)
        paged_prefill_kernel<128><<<grid, WAVES * 64, 0, stream>>>(p);
    else
        paged_prefill_kernel<64><<<grid, WAVES * 64, 0, stream>>>(p);
    return launch_status();
}
} // namespace camblas_hip
