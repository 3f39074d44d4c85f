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
// Rows of K and V go from memory into LDS directly, a tile ahead of the products. The maximum that weights
// refer to is moved only when a score exceeds it by 2^8. Sums, maxima and partials are FP32; weights are rounded to
// BF16 for the second product, whose matrix instruction takes them in the type of V (a second BF16 part for the bits
// lost would double that product). It costs 1.3 to 1.4 times the distance from the softmax in 64 bits that FP32
// weights have behind the same rounding of the output.
//
// Measured, 64 query and 8 key-value heads of 128: 2048 tokens after 30001 positions 1.87 to 2.01 ms from card to card,
// 1036 to 1113 TFLOP/s; 4096 tokens from the beginning 270 to 284 us, 968 to 1018 TFLOP/s (a large matrix product reaches 1410).
// Matrix units are busy 62 % and 57 % of the cycles, which run at 1.5 to 1.75 GHz under this load: both the clock and
// the cycles without a matrix instruction bound them. Six prompts of 28 query and 4 key-value heads of 64 behind a window of
// 1024: 145 to 154 us, 655 to 696 TFLOP/s; the work on scores is the same for half the products (matrix units busy 36 %,
// vector instructions issued in 72 % of the cycles, at 1.85 GHz).
#include "common.hpp"
#include "device.hpp"
#include "dma.hpp"
#include "paged_cache.hpp"

namespace camblas_hip
{
namespace
{
constexpr int WAVES = 4, THREADS = WAVES * 64, ROWS = WAVES * 32, TILE = 64, MOST_SHARES = 32;
constexpr int VECTOR = 0x2, MATRIX = 0x8, DS_READS = 0x100; // kinds of instructions for the scheduler
constexpr float LOG2E = 1.4426950408889634f;

struct PrefillParams {
    int batch, tokens, group, row_blocks;
    PagedCache cache;
    PageTable table;
    Visibility see;
    const int32_t *starts; // [batch + 1]: first token of each sequence
    float scale;           // times log2(e)
    float lowest;          // no finite score is below it, and its product with the scale is finite
    const unsigned short *q;
    unsigned short *out;
    int64_t q_stride, out_stride;
    // where positions are divided over `shares` workgroups per block of rows: [share][token][query head][dim], [..][..][..]
    int shares;
    float *part_o, *part_m, *part_l;
};

typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
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

// The upper 32 lanes of `first` against the lower 32 of `second`.
__device__ __forceinline__ u32x2_t swap_halves(unsigned first, unsigned second)
{
    return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_permlane32_swap(first, second, false, false));
}

// eight BF16 values: is one of them NaN or an infinity; those replaced by zero
__device__ __forceinline__ bool holds_infinite(u32x4_t packed)
{
    bool found = false;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        found = found || (packed[e] & 0x7f80u) == 0x7f80u || (packed[e] & 0x7f800000u) == 0x7f800000u;
    return found;
}
__device__ __forceinline__ u32x4_t without_infinite(u32x4_t packed)
{
#pragma unroll
    for (int e = 0; e < 4; ++e)
        packed[e] = ((packed[e] & 0x7f80u) == 0x7f80u ? 0 : packed[e] & 0xffffu) |
                    ((packed[e] & 0x7f800000u) == 0x7f800000u ? 0 : packed[e] & 0xffff0000u);
    return packed;
}

// a value that is the same in every lane, in a scalar register
__device__ __forceinline__ int uniform(int value) { return __builtin_amdgcn_readfirstlane(value); }

__device__ __forceinline__ int first_token(const PrefillParams &p, int sequence)
{
    return min(max(p.starts[sequence], 0), p.tokens);
}

// A block of ROWS rows of one key-value head: row r of it is query head r % group of token r / group.
struct Block {
    int sequence, kv_head, token0, tokens; // the sequence's first token and how many it has
    int length;                            // positions of the sequence
    int row0, rows;                        // the block's first row, how many rows the sequence has from there on
};

// The block of a number (first_block); false for one that is not used. A sequence's first block number grows with
// the sequence, so every wavefront looks for it among 64 at a time, without meeting the others; what is known of
// the sequence travels with the starts: a small call is a chain of trips to memory
// (one sequence a thread and the finder's words through LDS: 12 tokens past 165 8.6 / 8.3 us).
__device__ __forceinline__ bool find_block(const PrefillParams &p, int number, Block &block)
{
    // the last blocks of a causal sequence see most: they start first
    block.kv_head = number % p.cache.kv_heads;
    const int wanted = p.row_blocks - 1 - number / p.cache.kv_heads, lane = threadIdx.x % 64;
    int low = 0, count = p.batch;
    for (;;) {
        const int step = (count + 63) / 64, sequence = low + min(lane * step, count - 1);
        const int begin = first_token(p, sequence), end = first_token(p, sequence + 1);
        const int length = live_positions(p.table, p.cache, sequence);
        const uint64_t before = __ballot(lane * step < count && first_block(begin, p.group, ROWS, sequence) <= wanted);
        if (before == 0)
            return false;
        const int last = 63 - __builtin_clzll(before);
        low += last * step;
        count = min(step, count - last * step);
        if (step > 1)
            continue;
        block.sequence = low;
        block.token0 = __builtin_amdgcn_readlane(begin, last);
        block.tokens = __builtin_amdgcn_readlane(end, last) - block.token0;
        block.length = __builtin_amdgcn_readlane(length, last);
        block.row0 = (wanted - first_block(block.token0, p.group, ROWS, low)) * ROWS;
        block.rows = block.tokens * p.group - block.row0;
        return block.row0 >= 0 && block.rows > 0;
    }
}

// SHARED: blockIdx.y of `shares` workgroups takes its part of the tiles and leaves what it has for the join.
template <int DIM, bool SHARED> __global__ __launch_bounds__(THREADS, DIM == 64 ? 3 : 2) void paged_prefill_kernel(PrefillParams p)
{
    constexpr bool AHEAD = DIM == 128; // the next tile's scores are multiplied while this one's weights are worked out
    constexpr int CHUNKS = DIM / 8, FETCH = 64 / CHUNKS, FETCHES = TILE / FETCH / WAVES; // rows of a load, a wavefront's loads
    __shared__ __attribute__((aligned(16))) unsigned char keys0[TILE * DIM * 2], keys1[TILE * DIM * 2];
    __shared__ __attribute__((aligned(16))) unsigned char values0[TILE * DIM * 2], values1[TILE * DIM * 2];
    __shared__ unsigned infinite[2]; // which rows of a tile hold values that are not finite
    const int thread = threadIdx.x, lane = thread % 64, wave = uniform(thread / 64);
    const int column = lane % 32, half = lane / 32;
    if (thread < 2)
        infinite[thread] = 0;
    Block block;
    if (!find_block(p, blockIdx.x, block))
        return;
    const int sequence = block.sequence, kv_head = block.kv_head, token0 = block.token0, tokens = block.tokens;
    const int row0 = block.row0, rows = block.rows;

    // ---- this lane's row: token and query head, position
    const int past = block.length - tokens;
    int query;
    bf16x8_t q[DIM / 16];
    {
        const unsigned row = unsigned(min(row0 + wave * 32 + column, row0 + rows - 1)), group = p.group;
        const int token = int(row / group), head = kv_head * p.group + int(row % group);
        query = past + token;
        const unsigned short *from = p.q + int64_t(token0 + token) * p.q_stride + int64_t(head) * DIM + 8 * half;
#pragma unroll
        for (int s = 0; s < DIM / 16; ++s)
            q[s] = *reinterpret_cast<const bf16x8_t *>(from + 16 * s);
    }
    const int first_query = uniform(past + int(unsigned(row0) / unsigned(p.group)));
    const int last_query = uniform(past + int(unsigned(row0 + min(rows, ROWS) - 1) / unsigned(p.group)));
    const TileSpan<TILE> span(p.see, first_query, last_query);
    const int first = SHARED ? int(int64_t(span.tiles) * blockIdx.y / p.shares) : 0;
    const int end = SHARED ? int(int64_t(span.tiles) * (blockIdx.y + 1) / p.shares) : span.tiles;

    // which rows of the tile at hand exist and are seen by some query of the block
    uint64_t wanted = 0;
    // Few new tokens leave wavefronts without a row: those only fetch (16 tokens past 1000 positions each 23.9 / 22.0 us, 4
    // times 100 past 4000 53.4 / 51.5).
    const bool works = !SHARED || wave * 32 < rows;
    // bit n: the lane's query sees position base + n
    const auto seen_rows = [&](int base) {
        uint64_t seen = wanted & below(query - base + 1);
        if (p.see.window > 0)
            seen &= ~below(query - base + 1 - p.see.window) | below(p.see.sinks - base);
        return seen;
    };

    // ---- fetching tiles: lane r of every wavefront knows the page of tile row r
    const int32_t *pages = p.table.pages + int64_t(sequence) * p.table.stride;
    // (loaded a turn before it is looked at; a tile behind the last one: the last one's)
    const auto column_of = [&](int tile) { return (span.position(min(tile, end - 1)) + lane) >> p.cache.page_shift; };
    const auto load_page = [&](int tile) { return pages[min(column_of(tile), p.table.columns - 1)]; };
    const auto checked = [&](int tile, int page) {
        return (column_of(tile) < p.table.columns) & (unsigned(page) < unsigned(p.cache.pages)) ? page : -1;
    };
    // which rows of a tile exist and are seen by some query of the block
    const auto wanted_rows = [&](int tile, int page) {
        const int position = span.position(min(tile, end - 1)) + lane;
        return __ballot((page >= 0) & (position <= last_query) &
                        ((p.see.window <= 0) | (position > first_query - p.see.window) | (position < p.see.sinks)));
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
        return row_offset(p.cache, max(__builtin_amdgcn_readlane(page, own_row), 0), span.position(min(tile, end - 1)) + own_row) + head_at;
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

    // Turn `tile`: its keys and values are in `keys` and `values`. Heads of 128 (AHEAD) have its scores in `score` already
    // and multiply the next tile's, whose keys are in `next_keys`, into `next_score` while the weights are worked out:
    // fetched meanwhile are the next tile's values and the keys of the one after. Heads of 64 multiply their scores now
    // and fetch the next tile: three wavefronts of a SIMD fill each other's gaps, and the registers of a second set of
    // scores are better spent (windowed prompts 159 / 154 us).
    // Page numbers are loaded before the loads to LDS (a wait for them would be one for those too), looked at a turn
    // later, and made into addresses in the shadow of the products (all at the start of a turn it took 1000 of
    // 3400 cycles: 2048 tokens after 30001 2000 / 1898 us).
    uint64_t wanted1 = 0, wanted2 = 0;  // of the next tile and the one after
    int page1 = 0, page2 = 0, raw3 = 0; // their pages, and what the table holds for the one after those
    int64_t at1 = 0, at2 = 0;           // their place()
    const auto turn = [&](int tile, f32x16_t (&score)[2], f32x16_t (&next_score)[2], unsigned char *keys,
                          const unsigned char *next_keys, unsigned char *values, unsigned char *next_values) {
        const int base = span.position(tile);
        int page3 = checked(tile + 3, raw3);
        asm volatile("" : "+v"(page3));
        raw3 = load_page(tile + 4);
        if (tile + 1 < end)
            fetch(p.cache.v, value_from, at1, tile + 1, page1, next_values);
        if constexpr (AHEAD) {
            if (tile + 2 < end)
                fetch(p.cache.k, key_from, at2, tile + 2, page2, keys);
        } else {
            if (tile + 1 < end)
                fetch(p.cache.k, key_from, at1, tile + 1, page1, const_cast<unsigned char *>(next_keys));
            if (works)
                multiply_keys(keys, score);
        }
        const auto look_ahead = [&]() {
            wanted = wanted1;
            wanted1 = wanted2;
            page1 = page2;
            at1 = at2;
            page2 = page3;
            wanted2 = wanted_rows(tile + 3, page2);
            at2 = place(tile + 3, page2);
        };
        const bool whole = wanted == ~uint64_t(0) && base + TILE - 1 <= first_query &&
                           (p.see.window <= 0 || base > last_query - p.see.window || base + TILE <= p.see.sinks);
        uint64_t rows_infinite = 0;
        float highest = p.lowest; // a row that sees a position has a finite maximum, whatever its scores are
        if (!whole) { // (the same in every wavefront)
            const uint64_t own = seen_rows(base) >> (4 * half);
            highest = own ? p.lowest : -INFINITY;
            if (works)
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        // (all bits of a lane's own bit, and a bitwise choice: no masks in scalar registers)
                        const int keep = __builtin_amdgcn_sbfe(int(own >> (32 * t)), 8 * (r / 4) + r % 4, 1);
                        score[t][r] = __int_as_float((__float_as_int(score[t][r]) & keep) | (int(0xff800000u) & ~keep));
                    }
            // A weight of zero times NaN or infinity would reach the output. Rows that nobody sees become zeros. A
            // row that some see and that holds such values has them taken out of the product and added, as they
            // are, to the sums of those who see it: no weight changes what becomes of those.
            constexpr int PIECES = TILE * CHUNKS / THREADS;
            u32x4_t *own_pieces = reinterpret_cast<u32x4_t *>(values) + thread, piece[PIECES];
#pragma unroll
            for (int i = 0; i < PIECES; ++i)
                piece[i] = own_pieces[i * THREADS];
            u16x2_t largest = {0, 0}; // of the bits without the sign: those of infinities and NaN are the largest
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                const int r = (thread + i * THREADS) / CHUNKS;
                if (!((wanted >> r) & 1)) {
                    piece[i] = u32x4_t{0, 0, 0, 0};
                    own_pieces[i * THREADS] = piece[i];
                }
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    largest = __builtin_elementwise_max(largest, __builtin_bit_cast(u16x2_t, piece[i][e] & 0x7fff7fffu));
            }
            if (largest[0] >= 0x7f80 || largest[1] >= 0x7f80)
#pragma unroll
                for (int i = 0; i < PIECES; ++i)
                    if (holds_infinite(piece[i])) {
                        const int r = (thread + i * THREADS) / CHUNKS;
                        atomicOr(&infinite[r / 32], 1u << (r % 32));
                    }
            __syncthreads();
            rows_infinite = uint64_t(unsigned(uniform(int(infinite[0])))) | uint64_t(unsigned(uniform(int(infinite[1])))) << 32;
        }
        if (works) {
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
        }
        if (rows_infinite) {
            const uint64_t seen = seen_rows(base);
            for (uint64_t left = works ? rows_infinite : 0; left; left &= left - 1) {
                const int r = __builtin_ctzll(left);
                const bool sees_it = (seen >> r) & 1;
#pragma unroll
                for (int d = 0; d < DIM / 32; ++d) {
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const int dim = 32 * d + 8 * g + 4 * half;
                        const u32x2_t packed = *reinterpret_cast<const u32x2_t *>(
                            values + r * DIM * 2 + ((dim / 8) ^ turn_values<DIM>(r)) * 16 + dim % 8 * 2);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float v = __uint_as_float(e % 2 ? packed[e / 2] & 0xffff0000u : packed[e / 2] << 16);
                            acc[d][4 * g + e] += sees_it && !(fabsf(v) < INFINITY) ? v : 0.f;
                        }
                    }
                    asm volatile("" ::: "memory"); // (few values at a time in registers)
                }
            }
            __syncthreads();
            for (int piece = thread; piece < TILE * CHUNKS; piece += THREADS) {
                u32x4_t *at_piece = reinterpret_cast<u32x4_t *>(values + piece * 16);
                if (holds_infinite(*at_piece))
                    *at_piece = without_infinite(*at_piece);
            }
            if (thread < 2)
                infinite[thread] = 0;
            __syncthreads();
        }
        if (works) {
            const float reference = top == -INFINITY ? 0.f : top;
            if constexpr (AHEAD)
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
            look_ahead();
            // The order asked of the compiler: every matrix instruction is followed by vector instructions that fill
            // its 32 cycles and by the reads of an operand to come (left alone it put the products of the scores in a
            // row: 2264 against 2177 us at 2048 tokens after 30001).
            if constexpr (AHEAD) {
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
            }
        } else {
            look_ahead();
        }
        asm volatile("" ::: "memory");
        pipeline_barrier<0>();
        asm volatile("" ::: "memory");
    };

    if (first < end) {
        const int raw0 = load_page(first), raw1 = load_page(first + 1), raw2 = load_page(first + 2);
        raw3 = load_page(first + 3);
        const int page0 = checked(first, raw0);
        page1 = checked(first + 1, raw1);
        page2 = checked(first + 2, raw2);
        asm volatile("" : "+v"(page1), "+v"(page2), "+v"(raw3));
        const int64_t at0 = place(first, page0);
        at1 = place(first + 1, page1);
        fetch(p.cache.k, key_from, at0, first, page0, keys0);
        fetch(p.cache.v, value_from, at0, first, page0, values0);
        if (AHEAD && first + 1 < end)
            fetch(p.cache.k, key_from, at1, first + 1, page1, keys1);
        at2 = place(first + 2, page2);
        wanted = wanted_rows(first, page0);
        wanted1 = wanted_rows(first + 1, page1);
        wanted2 = wanted_rows(first + 2, page2);
        pipeline_barrier<0>();
        asm volatile("" ::: "memory");
        f32x16_t even[2], odd[2];
        if constexpr (AHEAD) {
            multiply_keys(keys0, even);
            asm volatile("" ::: "memory");
            pipeline_barrier<0>();
        }
        asm volatile("" ::: "memory");
        for (int tile = first; tile < end; tile += 2) {
            turn(tile, even, AHEAD ? odd : even, keys0, keys1, values0, values1);
            if (tile + 1 >= end)
                break;
            turn(tile + 1, AHEAD ? odd : even, even, keys1, keys0, values1, values0);
        }
    }

    const int row = row0 + wave * 32 + column;
    const float sum = total + __shfl_xor(total, 32);
    const bool kept = row < row0 + rows; // (the others' lanes still take part in the exchange)
    const int token = token0 + int(unsigned(row) / unsigned(p.group));
    const int head = kv_head * p.group + int(unsigned(row) % unsigned(p.group));
    if constexpr (SHARED) {
        if (!kept)
            return;
        const size_t at_row = (size_t(blockIdx.y) * p.tokens + token) * (p.cache.kv_heads * p.group) + head;
        if (half == 0) {
            p.part_m[at_row] = top;
            p.part_l[at_row] = sum;
        }
        float *to = p.part_o + at_row * DIM + 4 * half;
#pragma unroll
        for (int d = 0; d < DIM / 32; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<f32x4_t *>(to + 32 * d + 8 * g) =
                    f32x4_t{acc[d][4 * g], acc[d][4 * g + 1], acc[d][4 * g + 2], acc[d][4 * g + 3]};
    } else {
        const float inverse = normaliser(top, sum);
        // The two lanes of a row hold four dims each of every eight: the upper gives its half of the even eights for
        // the lower's half of the odd ones, and each writes eight dims in one piece.
        unsigned short *to = p.out + int64_t(token) * p.out_stride + int64_t(head) * DIM + 8 * half;
#pragma unroll
        for (int d = 0; d < DIM / 32; ++d)
#pragma unroll
            for (int g = 0; g < 4; g += 2) {
                u32x4_t whole;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const unsigned even = round_pair(acc[d][4 * g + 2 * e] * inverse, acc[d][4 * g + 2 * e + 1] * inverse);
                    const unsigned odd = round_pair(acc[d][4 * g + 4 + 2 * e] * inverse, acc[d][4 * g + 5 + 2 * e] * inverse);
                    const u32x2_t swapped = swap_halves(even, odd);
                    whole[e] = swapped[0];
                    whole[2 + e] = swapped[1];
                }
                if (kept)
                    *reinterpret_cast<u32x4_t *>(to + 32 * d + 8 * g) = whole;
            }
    }
}

// Joins the shares of a token's heads in their order; DIM / 4 threads take a head. What the shares left is on its way
// while the starts tell whether the token is any sequence's (finding the block first cost a trip to memory of its own).
template <int DIM> constexpr int join_heads() { return THREADS / (DIM / 4); }
template <int DIM> __global__ __launch_bounds__(THREADS) void paged_prefill_join_kernel(PrefillParams p)
{
    constexpr int ROW = DIM / 4, HEADS = join_heads<DIM>(), AT_ONCE = 8; // shares on their way together
    const int q_heads = p.cache.kv_heads * p.group, parts = (q_heads + HEADS - 1) / HEADS;
    const int token = blockIdx.x / parts, head = blockIdx.x % parts * HEADS + threadIdx.x / ROW;
    const int d = 4 * (threadIdx.x % ROW);
    const size_t first = size_t(token) * q_heads + min(head, q_heads - 1), step = size_t(p.tokens) * q_heads;
    bool owned = false;
    for (int b = threadIdx.x; b < p.batch; b += THREADS)
        owned = owned || (first_token(p, b) <= token && token < first_token(p, b + 1));
    float top = -INFINITY, sum = 0.f;
    f32x4_t o = {0.f, 0.f, 0.f, 0.f};
    for (int share = 0; share < p.shares; share += AT_ONCE) {
        float m[AT_ONCE], l[AT_ONCE];
        f32x4_t part[AT_ONCE];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            const size_t at = first + size_t(min(share + i, p.shares - 1)) * step;
            m[i] = p.part_m[at];
            l[i] = p.part_l[at];
            part[i] = *reinterpret_cast<const f32x4_t *>(p.part_o + at * DIM + d);
        }
        if (share == 0 && !__syncthreads_or(owned))
            return;
        const float before = top;
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i)
            top = fmaxf(top, m[i]);
        const float reference = top == -INFINITY ? 0.f : top, kept = __builtin_amdgcn_exp2f(before - reference);
        sum *= kept;
        o *= kept;
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i)
            if (share + i < p.shares) {
                const float factor = __builtin_amdgcn_exp2f(m[i] - reference);
                sum = fmaf(factor, l[i], sum);
                o += factor * part[i];
            }
    }
    if (head >= q_heads)
        return;
    o *= normaliser(top, sum);
    *reinterpret_cast<u32x2_t *>(p.out + int64_t(token) * p.out_stride + int64_t(head) * DIM + d) =
        u32x2_t{round_pair(o[0], o[1]), round_pair(o[2], o[3])};
}

int64_t prefill_blocks(int batch, int tokens, int group) { return int64_t(tokens) * group / ROWS + batch; }

// Over how many workgroups the positions of a block of rows are divided: as many as fill the chip where the
// blocks alone do not, with a few tiles each, going by what the table has room for, or the window: the host does not see the
// lengths. Measured, one workgroup / shares, before later steps: 7 sequences of up to 41 tokens past 2000 positions 56 / 27
// us (24.5 now); 15 of one token past 7000 154 / 20; 64 tokens past 16000 389 / 57. Shares that hold no tile still leave
// their partials (a table that fits / of 131072 positions: one prompt of 16 tokens 7.1 / 19.4 us, of 324 12.1 / 23.5).
int prefill_shares(int64_t blocks, int dim, int64_t positions, int compute_units)
{
    const int64_t room = int64_t(dim == 64 ? 3 : 2) * compute_units / (blocks > 0 ? blocks : 1);
    const int64_t enough = positions / (4 * TILE);
    const int64_t shares = room < enough ? room : enough;
    return shares < 2 ? 1 : shares < MOST_SHARES ? int(shares) : MOST_SHARES;
}

// the most positions that a block of rows can see
int64_t prefill_positions(int64_t capacity, const Visibility &see, int tokens, int group)
{
    const int64_t reach = int64_t(see.window) + see.sinks + (tokens < ROWS / group + 1 ? tokens : ROWS / group + 1);
    return see.window > 0 && reach < capacity ? reach : capacity;
}
} // namespace

size_t paged_prefill_workspace(int batch, int tokens, int q_heads, int kv_heads, int dim, int64_t capacity,
                               const Visibility &see, int compute_units)
{
    const int group = q_heads / kv_heads;
    const int shares = prefill_shares(prefill_blocks(batch, tokens, group) * kv_heads, dim,
                                      prefill_positions(capacity, see, tokens, group), compute_units);
    return shares > 1 ? size_t(shares) * tokens * q_heads * (size_t(dim) + 2) * sizeof(float) : 0;
}

hipError_t launch_paged_prefill(hipStream_t stream, int batch, int tokens, int q_heads, int dim, const PagedCache &cache,
                                const PageTable &table, const Visibility &see, const int32_t *starts, float scale,
                                const void *q, int64_t q_stride, void *out, int64_t out_stride, void *workspace,
                                int compute_units)
{
    PrefillParams p = {};
    p.batch = batch;
    p.tokens = tokens;
    p.group = q_heads / cache.kv_heads;
    const int64_t blocks = prefill_blocks(batch, tokens, p.group);
    if (blocks * cache.kv_heads >= (int64_t(1) << 32) / THREADS) // (threads of a launch are counted in 32 bits)
        return hipErrorInvalidValue;
    const int64_t capacity = int64_t(table.columns) << cache.page_shift;
    p.shares = prefill_shares(blocks * cache.kv_heads, dim, prefill_positions(capacity, see, tokens, p.group), compute_units);
    p.row_blocks = int(blocks);
    p.cache = cache;
    p.table = table;
    p.see = see;
    p.starts = starts;
    p.scale = scale * LOG2E;
    p.lowest = -FLT_MAX / (p.scale > 1.f ? 2.f * p.scale : 1.f);
    p.q = static_cast<const unsigned short *>(q);
    p.out = static_cast<unsigned short *>(out);
    p.q_stride = q_stride;
    p.out_stride = out_stride;
    const unsigned numbers = unsigned(blocks * cache.kv_heads);
    if (p.shares == 1) {
        const auto kernel = dim == 128 ? paged_prefill_kernel<128, false> : paged_prefill_kernel<64, false>;
        kernel<<<numbers, THREADS, 0, stream>>>(p);
        return launch_status();
    }
    const size_t rows = size_t(p.shares) * tokens * q_heads;
    p.part_o = static_cast<float *>(workspace);
    p.part_m = p.part_o + rows * dim;
    p.part_l = p.part_m + rows;
    const auto kernel = dim == 128 ? paged_prefill_kernel<128, true> : paged_prefill_kernel<64, true>;
    kernel<<<dim3(numbers, p.shares), THREADS, 0, stream>>>(p);
    const hipError_t status = launch_status();
    if (status != hipSuccess)
        return status;
    const auto join = dim == 128 ? paged_prefill_join_kernel<128> : paged_prefill_join_kernel<64>;
    const int heads = dim == 128 ? join_heads<128>() : join_heads<64>();
    join<<<unsigned(tokens) * ((q_heads + heads - 1) / heads), THREADS, 0, stream>>>(p);
    return launch_status();
}
} // namespace camblas_hip
