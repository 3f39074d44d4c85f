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
#include "paged_cache.hpp"

namespace camblas_hip
{
namespace
{
constexpr int WAVES = 4, TILE = 64;
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
__device__ __forceinline__ i16x4_t gather_column(const unsigned short *address)
{
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4_t *)(address));
}

// Where 16-byte chunk `chunk` of tile row `row` lies, in elements. Keys: 16 (8 for 64 dims) consecutive rows
// put a chunk on different banks. Values: pairs of chunks are moved, so that the four rows of a transposing
// read lie on different banks.
template <int DIM> __device__ __forceinline__ int key_slot(int row, int chunk)
{
    constexpr int CHUNKS = DIM / 8;
    const int turned = CHUNKS == 16 ? row & 15 : ((row >> 1) & 7) ^ ((row & 1) << 2);
    return (row * CHUNKS + (chunk ^ turned)) * 8;
}
template <int DIM> __device__ __forceinline__ int value_slot(int row, int chunk)
{
    constexpr int CHUNKS = DIM / 8;
    return (row * CHUNKS + (chunk ^ (2 * (row & 3)))) * 8;
}

__device__ __forceinline__ int first_token(const PrefillParams &p, int sequence)
{
    return min(max(p.starts[sequence], 0), p.tokens);
}

// COLS: 32-row column tiles per wavefront
template <int DIM, int COLS> __global__ __launch_bounds__(WAVES * 64, 2) void paged_prefill_kernel(PrefillParams p)
{
    constexpr int ROWS = WAVES * COLS * 32, THREADS = WAVES * 64, CHUNKS = DIM / 8;
    constexpr int PIECES = TILE * CHUNKS / THREADS, PIECE_ROWS = THREADS / CHUNKS; // 16-byte chunks a thread moves
    __shared__ __attribute__((aligned(16))) unsigned short key_tile[2][TILE * DIM], value_tile[2][TILE * DIM];
    __shared__ int found;
    const int thread = threadIdx.x, lane = thread % 64, wave = thread / 64;
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
    const int token0 = first_token(p, sequence), tokens = first_token(p, sequence + 1) - token0;
    const int64_t row0 = (block - (int64_t(token0) * p.group / ROWS + sequence)) * ROWS;
    const int64_t rows = int64_t(tokens) * p.group - row0;
    if (row0 < 0 || rows <= 0)
        return;

    // ---- this lane's rows: token and query head, position
    const int length = live_positions(p.table, p.cache, sequence);
    const int past = length - tokens;
    int query[COLS];
    bf16x8_t q[COLS][DIM / 16];
#pragma unroll
    for (int c = 0; c < COLS; ++c) {
        const int64_t row = row0 + (wave * COLS + c) * 32 + column;
        const int64_t kept = row < rows + row0 ? row : rows + row0 - 1;
        const int token = int(kept / p.group), head = kv_head * p.group + int(kept % p.group);
        query[c] = past + token;
        const unsigned short *from = p.q + int64_t(token0 + token) * p.q_stride + int64_t(head) * DIM + 8 * half;
#pragma unroll
        for (int s = 0; s < DIM / 16; ++s)
            q[c][s] = *reinterpret_cast<const bf16x8_t *>(from + 16 * s);
    }
    const int first_query = past + int(row0 / p.group);
    const int last_query = past + int((row0 + min(rows, int64_t(ROWS)) - 1) / p.group);
    const TileSpan<TILE> span(p.see, first_query, last_query);

    // ---- moving tiles: lane r of every wavefront knows the page of tile row r
    const int32_t *pages = p.table.pages + int64_t(sequence) * p.table.stride;
    const int chunk = thread % CHUNKS, piece_row = thread / CHUNKS;
    const int64_t head_at = int64_t(kv_head) * p.cache.head_stride;
    u32x4_t k_moving[PIECES], v_moving[PIECES];
    auto page_at = [&](int tile) {
        // (-1 as well for a row that no query of the block sees)
        const int position = span.position(tile) + lane;
        const bool wanted = position <= last_query &&
                            (p.see.window <= 0 || position > first_query - p.see.window || position < p.see.sinks);
        return wanted ? page_of(p.cache, pages, p.table.columns, position) : -1;
    };
    auto load = [&](int tile, int page) {
        const int base = span.position(tile);
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int r = piece_row + i * PIECE_ROWS;
            const int known = __shfl(max(page, 0), r); // (a row that is not wanted: some row that exists)
            const int64_t at = row_offset(p.cache, known, base + r) + head_at + 8 * chunk;
            k_moving[i] = *reinterpret_cast<const u32x4_t *>(p.cache.k + at);
            v_moving[i] = *reinterpret_cast<const u32x4_t *>(p.cache.v + at);
        }
    };
    auto store = [&](int buffer, uint64_t wanted) {
        if (wanted != ~uint64_t(0)) { // (uniform) zeros, which no weight turns into NaN
#pragma unroll
            for (int i = 0; i < PIECES; ++i)
                if (!((wanted >> (piece_row + i * PIECE_ROWS)) & 1))
                    v_moving[i] = u32x4_t{0, 0, 0, 0};
        }
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int r = piece_row + i * PIECE_ROWS;
            *reinterpret_cast<u32x4_t *>(&key_tile[buffer][key_slot<DIM>(r, chunk)]) = k_moving[i];
            *reinterpret_cast<u32x4_t *>(&value_tile[buffer][value_slot<DIM>(r, chunk)]) = v_moving[i];
        }
    };

    f32x16_t acc[COLS][DIM / 32];
    float top[COLS], total[COLS];
#pragma unroll
    for (int c = 0; c < COLS; ++c) {
        top[c] = -INFINITY;
        total[c] = 0.f;
#pragma unroll
        for (int d = 0; d < DIM / 32; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                acc[c][d][r] = 0.f;
    }

    uint64_t held = 0, next_held = 0; // which rows of a tile exist
    if (span.tiles > 0) {
        const int page = page_at(0);
        held = __ballot(page >= 0);
        load(0, page);
        store(0, held);
    }
    int next_page = span.tiles > 1 ? page_at(1) : -1;
    __syncthreads();
    for (int tile = 0; tile < span.tiles; ++tile) {
        const int buffer = tile & 1, base = span.position(tile);
        if (tile + 1 < span.tiles) {
            next_held = __ballot(next_page >= 0);
            load(tile + 1, next_page);
            if (tile + 2 < span.tiles)
                next_page = page_at(tile + 2);
        }
        const bool whole = held == ~uint64_t(0) && base + TILE - 1 <= first_query &&
                           (p.see.window <= 0 || base > last_query - p.see.window || base + TILE <= p.see.sinks);

        f32x16_t score[COLS][2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int c = 0; c < COLS; ++c)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    score[c][t][r] = 0.f;
#pragma unroll
            for (int s = 0; s < DIM / 16; ++s) {
                const bf16x8_t k =
                    *reinterpret_cast<const bf16x8_t *>(&key_tile[buffer][key_slot<DIM>(32 * t + column, 2 * s + half)]);
#pragma unroll
                for (int c = 0; c < COLS; ++c)
                    score[c][t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k, q[c][s], score[c][t], 0, 0, 0);
            }
        }
        bf16x8_t weights[COLS][4];
#pragma unroll
        for (int c = 0; c < COLS; ++c) {
            if (!whole) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int at = 32 * t + 8 * (r / 4) + 4 * half + r % 4;
                        if (!((held >> at) & 1) || !sees(p.see, query[c], base + at))
                            score[c][t][r] = -INFINITY;
                    }
            }
            float highest = -INFINITY;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    highest = fmaxf(highest, score[c][t][r]);
            highest *= p.scale;
            if (__any(highest > top[c] + 8.f)) {
                highest = fmaxf(highest, __shfl_xor(highest, 32));
                highest = fmaxf(highest, top[c]);
                const float factor = top[c] == highest ? 1.f : __builtin_amdgcn_exp2f(top[c] - highest);
                top[c] = highest;
                total[c] *= factor;
#pragma unroll
                for (int d = 0; d < DIM / 32; ++d)
                    acc[c][d] *= factor;
            }
            const float reference = top[c] == -INFINITY ? 0.f : top[c];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    score[c][t][r] = __builtin_amdgcn_exp2f(fmaf(score[c][t][r], p.scale, -reference));
                    total[c] += score[c][t][r];
                }
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    weights[c][2 * t + u] = __builtin_bit_cast(
                        bf16x8_t, u32x4_t{round_pair(score[c][t][8 * u], score[c][t][8 * u + 1]),
                                          round_pair(score[c][t][8 * u + 2], score[c][t][8 * u + 3]),
                                          round_pair(score[c][t][8 * u + 4], score[c][t][8 * u + 5]),
                                          round_pair(score[c][t][8 * u + 6], score[c][t][8 * u + 7])});
            }
        }
        // this lane points at position 16 u + 4 half + (lane % 16) / 4 (and eight further), dims of its sixteen
        const int spot = 4 * half + (lane % 16) / 4;
#pragma unroll
        for (int u = 0; u < TILE / 16; ++u)
#pragma unroll
            for (int d = 0; d < DIM / 32; ++d) {
                const int dims = 32 * d + 16 * (lane / 16 % 2) + 4 * (lane % 4);
                const i16x4_t lower =
                    gather_column(&value_tile[buffer][value_slot<DIM>(16 * u + spot, dims / 8) + dims % 8]);
                const i16x4_t upper =
                    gather_column(&value_tile[buffer][value_slot<DIM>(16 * u + 8 + spot, dims / 8) + dims % 8]);
                const bf16x8_t v = __builtin_bit_cast(
                    bf16x8_t, i16x8_t{lower[0], lower[1], lower[2], lower[3], upper[0], upper[1], upper[2], upper[3]});
#pragma unroll
                for (int c = 0; c < COLS; ++c)
                    acc[c][d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, weights[c][u], acc[c][d], 0, 0, 0);
            }
        if (tile + 1 < span.tiles)
            store(1 - buffer, next_held);
        held = next_held;
        __syncthreads();
    }

#pragma unroll
    for (int c = 0; c < COLS; ++c) {
        const int64_t row = row0 + (wave * COLS + c) * 32 + column;
        const float sum = total[c] + __shfl_xor(total[c], 32);
        if (row >= row0 + rows)
            continue;
        // (no position seen: zero; a sum that is NaN stays NaN)
        const float inverse = sum == 0.f ? 0.f : 1.f / sum;
        const int token = token0 + int(row / p.group), head = kv_head * p.group + int(row % p.group);
        unsigned short *to = p.out + int64_t(token) * p.out_stride + int64_t(head) * DIM + 4 * half;
#pragma unroll
        for (int d = 0; d < DIM / 32; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<u32x2_t *>(to + 32 * d + 8 * g) =
                    u32x2_t{round_pair(acc[c][d][4 * g] * inverse, acc[c][d][4 * g + 1] * inverse),
                            round_pair(acc[c][d][4 * g + 2] * inverse, acc[c][d][4 * g + 3] * inverse)};
    }
}
} // namespace

hipError_t launch_paged_prefill(hipStream_t stream, int batch, int tokens, int q_heads, int dim, const PagedCache &cache,
                                const PageTable &table, const Visibility &see, const int32_t *starts, float scale,
                                const void *q, int64_t q_stride, void *out, int64_t out_stride, int compute_units)
{
    constexpr int COLS = 1, ROWS = WAVES * COLS * 32;
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
        paged_prefill_kernel<128, COLS><<<grid, WAVES * 64, 0, stream>>>(p);
    else
        paged_prefill_kernel<64, COLS><<<grid, WAVES * 64, 0, stream>>>(p);
    return launch_status();
}
} // namespace camblas_hip
