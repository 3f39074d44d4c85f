// One new token of every sequence against its pages: out = softmax(scale q K^T) V over the positions the
// token sees, grouped query heads, BF16 storage.
//
// The kernel is bound by the cache's rows, which are read once: 2 * positions * dim * 2 bytes per
// key-value head. A wavefront takes 32 positions at a time and runs both products on the matrix cores with
// the query heads of a group padded to 16 (v_mfma_f32_16x16x32_bf16):
//   scores  S[position, head] = K[position, :] . Q[head, :]
//   output  O[dim, head]      = V[position, dim]^T . P[position, head]
// A lane leaves the first product with head lane % 16 and eight positions, which is the operand layout of
// the second once the order of its K index is taken to be the order the lane holds. All rows are loaded whole,
// past the caches: those of K are turned into operands through the wavefront's own part of LDS, those of V in
// registers by byte permutes, so that product w yields the dims (dim / 16) m + w. The running maximum, the
// sum and the outputs of a head stay in the lanes of that head: the maximum that weights refer to is moved only when a
// score exceeds it by 2^8 (a published technique), so that the outputs are rarely rescaled. Sums, maxima and partials are
// FP32. Weights are rounded to BF16 for the second product: the matrix instruction takes them in the type of V, and a
// second BF16 part for the bits lost would double that product. It costs 1.05 to 1.4 times the distance from
// the softmax in 64 bits that FP32 weights have behind the same rounding of the output.
//
// Measured, 64 query and 8 key-value heads of 128: 32 sequences of 2048 positions 44.5 us, 6.05 TB/s; 64 of 1 to
// 16384 378 us, 6.0 TB/s; one of 131072 96 us, 5.6 TB/s (a copy of 2 GiB moves 4.9 TB/s, reads alone are faster);
// one of 129 5.2 us. Small calls are bound by their trips to memory, one after the other: length and page, K and V.
//
// Work is divided by what the sequences hold, not by what the table could hold: all steps of a tile for each
// wavefront (sequence, key-value head and 16 query heads, positions) are numbered and every workgroup takes an equal
// run of them, so lengths may differ by any factor (that it is divided at all goes by the table: decode_shares). A workgroup's wavefronts meet in LDS at the end of each
// (sequence, heads); one that covered it whole writes the output, the others leave a partial (at most two
// per workgroup) that a second kernel joins in order. Where the workgroups that one (sequence, heads) each
// would make are enough, there are no partials and one launch.
#include "common.hpp"
#include "device.hpp"
#include "paged_cache.hpp"

namespace camblas_hip
{
namespace
{
constexpr int TILE = 32, HEADS = 16, JOIN_THREADS = 256, MOST_SHARES = 1024, SHARE_WAVES = 4;
constexpr float LOG2E = 1.4426950408889634f;

struct DecodeParams {
    int batch, group, head_tiles; // query heads per key-value head, tiles of 16 of them
    PagedCache cache;
    PageTable table;
    Visibility see;
    float scale; // times log2(e)
    const unsigned short *q;
    unsigned short *out;
    int64_t q_stride, out_stride;
    float *part_o, *part_m, *part_l; // [2 * workgroups][16][dim], [..][16], [..][16]
    int2 *joins;                     // per (sequence, heads): first and last workgroup that holds a part of it
};

// ---- one (sequence, heads): steps first .. last - 1 of it by this workgroup's wavefronts

struct Item {
    int sequence, kv_head, head0, heads; // first query head and how many of them
};

template <int DIM> struct Running {
    static constexpr int DIMS = DIM / 16; // dims a lane holds of a V row
    f32x4_t acc[DIMS];                    // acc[w][r]: dim DIMS * (4 j + r) + w of head m
    float top, total;
};

__device__ __forceinline__ int fetch_page(const DecodeParams &p, const int32_t *row, int base, int lane)
{
    return page_of(p.cache, row, p.table.columns, base + lane % TILE);
}

// Eight rows of a tile for every lane, 16 lanes to a row: rows 16 (e / 4) + 4 j + e % 4, DIM / 16 values from
// (DIM / 16) m on. Every row is read once and by one load: it takes no place in the caches.
// LARGE: pages of 16 positions and more, so that each half of a tile lies in one page: its place is then the
// same in every lane, and a lane's own offsets (`along`, in bytes, for the rows 4 j + 0 .. 3) the same in
// every tile. page: lane r holds that of row r % 32; a row without one is read from some page that exists, and not used.
template <int DIM, bool LARGE>
__device__ __forceinline__ void load_rows(const DecodeParams &p, const unsigned short *array, int base, int page, int64_t head,
                                          int lane, u32x4_t along, unsigned (&rows)[8][DIM / 32])
{
    typedef unsigned row_t __attribute__((ext_vector_type(DIM / 32)));
    const int known = page < 0 ? 0 : page;
    row_t got[8];
    if constexpr (LARGE) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int64_t at = row_offset(p.cache, __builtin_amdgcn_readlane(known, 16 * half), base + 16 * half) + head;
            const char *from = reinterpret_cast<const char *>(array + at);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                got[4 * half + e] = __builtin_nontemporal_load(reinterpret_cast<const row_t *>(from + along[e]));
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int r = 16 * (e / 4) + 4 * (lane / 16) + e % 4;
            const int64_t at = row_offset(p.cache, __shfl(known, r), base + r) + head + (DIM / 16) * (lane % 16);
            got[e] = __builtin_nontemporal_load(reinterpret_cast<const row_t *>(array + at));
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int i = 0; i < DIM / 32; ++i)
            rows[e][i] = got[e][i];
}

// Where 16-byte chunk `chunk` of key row `row` lies in a wavefront's part of LDS: rows turned so that the
// 16 rows of a fragment lie on different banks.
template <int DIM> __device__ __forceinline__ int key_slot(int row, int chunk)
{
    constexpr int CHUNKS = DIM / 8;
    return row * DIM + (chunk ^ (CHUNKS == 16 ? row & 15 : row >> 1 & 7)) * 8;
}

// Key rows as the lanes loaded them into a wavefront's own part of LDS, whose accesses stay in order without
// a barrier.
template <int DIM>
__device__ __forceinline__ void park_keys(const unsigned (&rows)[8][DIM / 32], int lane, unsigned short *keys)
{
    typedef unsigned row_t __attribute__((ext_vector_type(DIM / 32)));
    const int m = lane % 16, j = lane / 16;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        row_t k;
#pragma unroll
        for (int i = 0; i < DIM / 32; ++i)
            k[i] = rows[e][i];
        *reinterpret_cast<row_t *>(keys + key_slot<DIM>(16 * (e / 4) + 4 * j + e % 4, m * (DIM / 16) / 8) + m * (DIM / 16) % 8) = k;
    }
    asm volatile("" ::: "memory");
}

// The weights of a tile's positions: register r of score[t] is position 16 t + 4 j + r, head m.
template <int DIM>
__device__ __forceinline__ bf16x8_t weigh(float scale, unsigned mask, const bf16x8_t (&q)[DIM / 32], int lane,
                                          const unsigned short *keys, Running<DIM> &run)
{
    const int m = lane % 16, j = lane / 16;
    f32x4_t score[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        score[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < DIM / 32; ++s)
            score[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                *reinterpret_cast<const bf16x8_t *>(keys + key_slot<DIM>(16 * t + m, 4 * s + j)), q[s], score[t], 0, 0, 0);
        score[t] *= scale;
    }
    asm volatile("" ::: "memory");
    if (mask != ~0u) { // (uniform)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                score[t][r] = (mask >> (16 * t + 4 * j + r)) & 1 ? score[t][r] : -INFINITY;
    }
    float top = fmaxf(fmaxf(fmaxf(score[0][0], score[0][1]), fmaxf(score[0][2], score[0][3])),
                      fmaxf(fmaxf(score[1][0], score[1][1]), fmaxf(score[1][2], score[1][3])));
    if (__any(top > run.top + 8.f)) {
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        top = fmaxf(top, run.top);
        const float factor = run.top == top ? 1.f : __builtin_amdgcn_exp2f(run.top - top);
        run.top = top;
        run.total *= factor;
#pragma unroll
        for (int w = 0; w < DIM / 16; ++w)
            run.acc[w] *= factor;
    }
    const float reference = run.top == -INFINITY ? 0.f : run.top;
    u32x4_t weights;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            score[t][r] = __builtin_amdgcn_exp2f(score[t][r] - reference);
            run.total += score[t][r];
        }
        weights[2 * t] = round_pair(score[t][0], score[t][1]);
        weights[2 * t + 1] = round_pair(score[t][2], score[t][3]);
    }
    return __builtin_bit_cast(bf16x8_t, weights);
}

template <int DIM>
__device__ __forceinline__ void add_values(unsigned mask, bf16x8_t weights, unsigned (&v)[8][DIM / 32], int lane, Running<DIM> &run)
{
    if (mask != ~0u) { // (uniform) a weight of zero times what a hidden row may hold, NaN or infinity, would reach the output
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const bool seen = (mask >> (16 * (e / 4) + 4 * (lane / 16) + e % 4)) & 1;
#pragma unroll
            for (int i = 0; i < DIM / 32; ++i)
                v[e][i] = seen ? v[e][i] : 0u;
        }
    }
#pragma unroll
    for (int i = 0; i < DIM / 32; ++i) {
        u32x4_t even, odd;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            even[c] = __builtin_amdgcn_perm(v[2 * c + 1][i], v[2 * c][i], 0x05040100u);
            odd[c] = __builtin_amdgcn_perm(v[2 * c + 1][i], v[2 * c][i], 0x07060302u);
        }
        run.acc[2 * i] =
            __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, even), weights, run.acc[2 * i], 0, 0, 0);
        run.acc[2 * i + 1] =
            __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, odd), weights, run.acc[2 * i + 1], 0, 0, 0);
    }
}

// page: those of the wavefront's first tile (fetch_page). slot < 0: this workgroup holds the whole of it and writes
// the output; otherwise partial `slot`
template <int DIM, bool LARGE, int WAVES>
__device__ __forceinline__ void work_item(const DecodeParams &p, const unsigned short *queries, float scale, const Item item, const TileSpan<TILE> span, int query,
                                          int first, int last, int page, int slot)
{
    // (the outputs of the wavefronts, once they are done with their keys)
    constexpr int KEYS = TILE * DIM * 2, OUTPUTS = HEADS * (DIM + 4) * 4;
    __shared__ __attribute__((aligned(16))) unsigned char room[WAVES * (KEYS > OUTPUTS ? KEYS : OUTPUTS)];
    float(*wave_o)[HEADS][DIM + 4] = reinterpret_cast<float(*)[HEADS][DIM + 4]>(room);
    __shared__ float wave_m[WAVES][HEADS], wave_l[WAVES][HEADS];
    const int thread = threadIdx.x, lane = thread % 64, m = lane % 16, j = lane / 16;
    const int wave = __builtin_amdgcn_readfirstlane(thread / 64);
    unsigned short *keys = reinterpret_cast<unsigned short *>(room + wave * KEYS);
    const int32_t *row = p.table.pages + int64_t(item.sequence) * p.table.stride;
    const int64_t head_at = int64_t(item.kv_head) * p.cache.head_stride;
    u32x4_t along;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        along[e] = LARGE ? (unsigned(4 * j + e) * unsigned(p.cache.slot_stride) + unsigned(DIM / 16 * m)) * 2 : 0;
    bf16x8_t q[DIM / 32];
    {
        const int head = item.head0 + (m < item.heads ? m : item.heads - 1);
        const unsigned short *from = queries + int64_t(item.sequence) * p.q_stride + int64_t(head) * DIM + 8 * j;
#pragma unroll
        for (int s = 0; s < DIM / 32; ++s)
            q[s] = *reinterpret_cast<const bf16x8_t *>(from + 32 * s);
    }
    Running<DIM> run;
    run.top = -INFINITY;
    run.total = 0.f;
#pragma unroll
    for (int w = 0; w < DIM / 16; ++w)
        run.acc[w] = f32x4_t{0.f, 0.f, 0.f, 0.f};

    const int end = min(last * WAVES, span.tiles);
    unsigned met = 0; // whether a position was seen at all
    __syncthreads(); // (outputs of the item before may still be read)
    int tile = __builtin_amdgcn_readfirstlane(first * WAVES + wave);
    if (tile < end) {
        // The next tile's keys are loaded as soon as this one's have gone to LDS, its values as soon as this one's
        // are multiplied: one set of registers each, and one of the two always on its way.
        unsigned k[8][DIM / 32], v[8][DIM / 32];
        const auto seen = [&](int page, int base) { return unsigned(__ballot(page >= 0 && sees(p.see, query, base + lane % TILE))); };
        int base = span.position(tile);
        unsigned mask = seen(page, base);
        load_rows<DIM, LARGE>(p, p.cache.k, base, page, head_at, lane, along, k);
        load_rows<DIM, LARGE>(p, p.cache.v, base, page, head_at, lane, along, v);
        base = span.position(min(tile + WAVES, span.tiles - 1));
        page = fetch_page(p, row, base, lane);
        for (;;) {
            tile += WAVES;
            park_keys<DIM>(k, lane, keys);
            if (tile < end)
                load_rows<DIM, LARGE>(p, p.cache.k, base, page, head_at, lane, along, k);
            met |= mask;
            const bf16x8_t weights = weigh<DIM>(scale, mask, q, lane, keys, run);
            add_values<DIM>(mask, weights, v, lane, run);
            if (tile >= end)
                break;
            mask = seen(page, base);
            load_rows<DIM, LARGE>(p, p.cache.v, base, page, head_at, lane, along, v);
            base = span.position(min(tile + WAVES, span.tiles - 1));
            page = fetch_page(p, row, base, lane);
        }
    }
    if (met && run.top == -INFINITY) // (scores of minus infinity only)
        run.top = -FLT_MAX;
    run.total += __shfl_xor(run.total, 16);
    run.total += __shfl_xor(run.total, 32);
    __syncthreads(); // (keys of other wavefronts may still be read)
    if (j == 0) {
        wave_m[wave][m] = run.top;
        wave_l[wave][m] = run.total;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int w = 0; w < DIM / 16; w += 4)
            *reinterpret_cast<f32x4_t *>(&wave_o[wave][m][(DIM / 16) * (4 * j + r) + w]) =
                f32x4_t{run.acc[w][r], run.acc[w + 1][r], run.acc[w + 2][r], run.acc[w + 3][r]};
    __syncthreads();
    // (four dims a thread, one piece to memory: one by one they made 129 positions 5.9 us of 5.2)
    for (int index = thread; index < item.heads * DIM / 4; index += WAVES * 64) {
        const int h = index / (DIM / 4), d = 4 * (index % (DIM / 4));
        float best = wave_m[0][h];
#pragma unroll
        for (int w = 1; w < WAVES; ++w)
            best = fmaxf(best, wave_m[w][h]);
        const float reference = best == -INFINITY ? 0.f : best;
        f32x4_t numerator = {0.f, 0.f, 0.f, 0.f};
        float denominator = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const float factor = __builtin_amdgcn_exp2f(wave_m[w][h] - reference);
            numerator += factor * *reinterpret_cast<const f32x4_t *>(&wave_o[w][h][d]);
            denominator = fmaf(factor, wave_l[w][h], denominator);
        }
        if (slot < 0) {
            numerator *= normaliser(best, denominator);
            *reinterpret_cast<u32x2_t *>(p.out + int64_t(item.sequence) * p.out_stride + int64_t(item.head0 + h) * DIM + d) =
                u32x2_t{round_pair(numerator[0], numerator[1]), round_pair(numerator[2], numerator[3])};
        } else {
            *reinterpret_cast<f32x4_t *>(p.part_o + (size_t(slot) * HEADS + h) * DIM + d) = numerator;
            if (d == 0) {
                p.part_m[slot * HEADS + h] = best;
                p.part_l[slot * HEADS + h] = denominator;
            }
        }
    }
}

__device__ __forceinline__ TileSpan<TILE> span_of(const DecodeParams &p, int sequence, int &query)
{
    query = live_positions(p.table, p.cache, sequence) - 1;
    return TileSpan<TILE>(p.see, query, query);
}

__device__ __forceinline__ Item item_of(const DecodeParams &p, int sequence, int index)
{
    const int kv_head = index / p.head_tiles, tile = index % p.head_tiles;
    const int first = tile * HEADS;
    return Item{sequence, kv_head, kv_head * p.group + first, min(HEADS, p.group - first)};
}

// The pages of the first tile a wavefront takes from step `first` on.
template <int WAVES>
__device__ __forceinline__ int first_page(const DecodeParams &p, const TileSpan<TILE> span, int sequence, int first)
{
    const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x / 64)), lane = threadIdx.x % 64;
    const int tile = first * WAVES + wave;
    return tile < span.tiles
               ? fetch_page(p, p.table.pages + int64_t(sequence) * p.table.stride, span.position(tile), lane) : -1;
}

// one workgroup per (heads, sequence)
template <int DIM, bool LARGE, int WAVES> __global__ __launch_bounds__(WAVES * 64, 2) void paged_decode_whole_kernel(DecodeParams p)
{
    const int sequence = blockIdx.y;
    int query, page = -1;
    if (p.see.window <= 0) { // the pages travel together with the length that says whether they are needed
        const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x / 64));
        page = fetch_page(p, p.table.pages + int64_t(sequence) * p.table.stride, wave * TILE, threadIdx.x % 64);
    }
    const TileSpan<TILE> span = span_of(p, sequence, query);
    if (p.see.window > 0)
        page = first_page<WAVES>(p, span, sequence, 0);
    work_item<DIM, LARGE, WAVES>(p, p.q, p.scale, item_of(p, sequence, blockIdx.x), span, query, 0, (span.tiles + WAVES - 1) / WAVES, page, -1);
}

// every workgroup an equal run of all steps
template <int DIM, bool LARGE> __global__ __launch_bounds__(SHARE_WAVES * 64, 2) void paged_decode_shares_kernel(DecodeParams p)
{
    constexpr int WAVES = SHARE_WAVES, THREADS = WAVES * 64;
    __shared__ int64_t wave_total[WAVES];
    __shared__ int64_t found_start;
    __shared__ int found_sequence;
    const int thread = threadIdx.x, lane = thread % 64, wave = thread / 64;
    const int items = p.cache.kv_heads * p.head_tiles;
    const unsigned short *queries = p.q;
    const float scale = p.scale;
    // steps before each thread's run of sequences
    const int per = (p.batch + THREADS - 1) / THREADS;
    const int from = min(thread * per, p.batch), to = min(from + per, p.batch);
    int64_t mine = 0;
    for (int b = from; b < to; ++b) {
        int query;
        mine += int64_t((span_of(p, b, query).tiles + WAVES - 1) / WAVES) * items;
    }
    int64_t before = mine;
#pragma unroll
    for (int shift = 1; shift < 64; shift *= 2) {
        const int64_t other = __shfl_up(before, shift);
        before += lane >= shift ? other : 0;
    }
    if (lane == 63)
        wave_total[wave] = before;
    __syncthreads();
    int64_t all = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        before += w < wave ? wave_total[w] : 0;
        all += wave_total[w];
    }
    before -= mine;
    const int64_t workers = min(all, int64_t(gridDim.x)); // each has a step, at least
    if (int64_t(blockIdx.x) >= workers)
        return; // (uniform)
    int64_t step = share_begin(all, workers, blockIdx.x);
    const int64_t stop = share_begin(all, workers, int64_t(blockIdx.x) + 1);
    if (step >= before && step < before + mine) {
        for (int b = from; b < to; ++b) {
            int query;
            const int64_t steps = int64_t((span_of(p, b, query).tiles + WAVES - 1) / WAVES) * items;
            if (step < before + steps) {
                found_sequence = b;
                found_start = before;
                break;
            }
            before += steps;
        }
    }
    __syncthreads();
    int sequence = __builtin_amdgcn_readfirstlane(found_sequence);
    int64_t start = found_start;
    while (step < stop) {
        int query;
        const TileSpan<TILE> span = span_of(p, sequence, query);
        const int steps = (span.tiles + WAVES - 1) / WAVES;
        while (step < stop && step < start + int64_t(steps) * items) {
            const int index = int((step - start) / steps);
            const int64_t begins = start + int64_t(index) * steps;
            const int first = int(step - begins);
            const int last = int(min(int64_t(steps), stop - begins));
            const int slot = first > 0 ? 2 * int(blockIdx.x) : last < steps ? 2 * int(blockIdx.x) + 1 : -1;
            if (first == 0 && thread == 0) {
                p.joins[size_t(sequence) * items + index] =
                    int2{int(blockIdx.x), int(share_of(all, workers, begins + steps - 1))};
            }
            work_item<DIM, LARGE, WAVES>(p, queries, scale, item_of(p, sequence, index), span, query, first, last,
                                  first_page<WAVES>(p, span, sequence, first), slot);
            step = begins + last;
        }
        start += int64_t(steps) * items;
        ++sequence;
    }
}

// Joins the partials of one query head in the order of its positions; zeros where the sequence holds
// nothing. A head that a single workgroup held is written already. DIM / 4 threads take a partial's row and the
// rows are dealt to the groups of threads: an ordered sum, whatever the number of partials (one thread per dim
// walking 64 of them took 140 us). Two trips to memory: what says where the partials lie, and all of them, up to
// AHEAD rows a group (maxima, sums and rows one after the other made five: 131072 positions 97.2 / 96.0 us).
template <int DIM> __global__ __launch_bounds__(JOIN_THREADS) void paged_decode_join_kernel(DecodeParams p)
{
    constexpr int ROW = DIM / 4, GROUPS = JOIN_THREADS / ROW, JOIN_WAVES = JOIN_THREADS / 64, AHEAD = 8;
    __shared__ float weight[MOST_SHARES], group_o[GROUPS][DIM], wave_top[JOIN_WAVES], wave_sums[JOIN_WAVES];
    const int thread = threadIdx.x, lane = thread % 64, wave = thread / 64;
    const int head = blockIdx.x, sequence = blockIdx.y, items = p.cache.kv_heads * p.head_tiles;
    const int within = head % p.group, h = within % HEADS;
    const int2 join = p.joins[size_t(sequence) * items + head / p.group * p.head_tiles + within / HEADS]; // (unset: not used)
    int query;
    const bool empty = span_of(p, sequence, query).tiles == 0;
    unsigned short *out = p.out + int64_t(sequence) * p.out_stride + int64_t(head) * DIM;
    if (empty) {
        if (thread < DIM)
            out[thread] = 0;
        return;
    }
    const int count = join.y - join.x + 1;
    if (count == 1)
        return;
    const auto row_of = [&](int i) { return size_t(2 * (join.x + i) + (i == 0)) * HEADS + h; };
    const int group = thread / ROW, d = 4 * (thread % ROW);
    const auto part = [&](int i) { return *reinterpret_cast<const f32x4_t *>(p.part_o + row_of(i) * DIM + d); };
    // (threads without a partial read the last one)
    const int own = min(thread, count - 1);
    const float own_top = p.part_m[row_of(own)];
    const float own_sum = p.part_l[row_of(own)];
    f32x4_t ahead[AHEAD];
#pragma unroll
    for (int n = 0; n < AHEAD; ++n)
        ahead[n] = part(min(group + n * GROUPS, count - 1));
    float top = own_top;
    for (int i = thread + JOIN_THREADS; i < count; i += JOIN_THREADS)
        top = fmaxf(top, p.part_m[row_of(i)]);
    top = wave_max(top);
    if (lane == 0)
        wave_top[wave] = top;
    __syncthreads();
    top = wave_top[0];
#pragma unroll
    for (int w = 1; w < JOIN_WAVES; ++w)
        top = fmaxf(top, wave_top[w]);
    const float reference = top == -INFINITY ? 0.f : top;
    const float own_factor = __builtin_amdgcn_exp2f(own_top - reference);
    float sum = thread < count ? own_factor * own_sum : 0.f;
    weight[thread] = own_factor;
    for (int i = thread + JOIN_THREADS; i < count; i += JOIN_THREADS) {
        weight[i] = __builtin_amdgcn_exp2f(p.part_m[row_of(i)] - reference);
        sum = fmaf(weight[i], p.part_l[row_of(i)], sum);
    }
    sum = wave_sum(sum);
    if (lane == 0)
        wave_sums[wave] = sum;
    __syncthreads();
    f32x4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int n = 0; n < AHEAD; ++n)
        if (group + n * GROUPS < count)
            o += weight[group + n * GROUPS] * ahead[n];
#pragma unroll 4
    for (int i = group + AHEAD * GROUPS; i < count; i += GROUPS)
        o += weight[i] * part(i);
    *reinterpret_cast<f32x4_t *>(&group_o[group][d]) = o;
    __syncthreads();
    if (thread < DIM) {
        float numerator = 0.f, denominator = 0.f;
#pragma unroll
        for (int g = 0; g < GROUPS; ++g)
            numerator += group_o[g][thread];
#pragma unroll
        for (int w = 0; w < JOIN_WAVES; ++w)
            denominator += wave_sums[w];
        out[thread] = float_to_bf16_bits(denominator != 0.f ? numerator / denominator : numerator * normaliser(top, denominator));
    }
}
} // namespace

// How a call is divided: workgroups that share all steps, or 0 for one workgroup per (heads, sequence). `positions` is what
// the table has room for, or the window: the host does not see the lengths. A table that is wider than its sequences
// are long makes short ones be shared too (64 query and 8 key-value heads of 128, table that fits / of 131072
// positions: 1 sequence of 64 positions 5.2 / 9.0 us, 32 of 64 5.5 / 10.4, 32 of 1024 25.0 / 32.4, 32 of 2048 45.1 / 52.8).
// Sharing costs a second launch and the numbering of the steps, some 4 us, and keeps every compute unit busy
// whatever the lengths; one workgroup each is done when the longest sequence is. Measured, 64 query and 8
// key-value heads of 128, whole / shared: 8 items of 512 positions 9.9 / 11.2 us, of 1024 15.4 / 11.2; 128 items of
// 1024 17.9 / 20.2, of 2048 31.7 / 30.8 (lengths from 1 to that 25 / 20); 256 items of 2048 45 / 52 (35 / 37), of
// 4096 84 / 93 (63 / 49).
static int decode_shares(int64_t items, int64_t positions, int compute_units)
{
    const int64_t busy = items < compute_units ? items : compute_units;
    if (positions <= 512 + 1792 * busy / compute_units)
        return 0;
    return 2 * compute_units < MOST_SHARES ? 2 * compute_units : MOST_SHARES;
}

static int64_t decode_positions(int64_t capacity, const Visibility &see)
{
    return see.window > 0 && int64_t(see.window) + see.sinks < capacity ? int64_t(see.window) + see.sinks : capacity;
}

size_t paged_decode_workspace(int batch, int q_heads, int kv_heads, int dim, int64_t capacity, const Visibility &see,
                              int compute_units)
{
    const int64_t items = int64_t(batch) * kv_heads * ((q_heads / kv_heads + HEADS - 1) / HEADS);
    const size_t shares = size_t(decode_shares(items, decode_positions(capacity, see), compute_units));
    return shares ? 2 * shares * HEADS * (size_t(dim) + 2) * sizeof(float) + size_t(items) * sizeof(int2) : 0;
}

template <int WAVES>
static void launch_whole(hipStream_t stream, int dim, bool large, dim3 grid, const DecodeParams &p)
{
    const auto kernel =
        dim == 128 ? (large ? paged_decode_whole_kernel<128, true, WAVES> : paged_decode_whole_kernel<128, false, WAVES>)
                   : (large ? paged_decode_whole_kernel<64, true, WAVES> : paged_decode_whole_kernel<64, false, WAVES>);
    kernel<<<grid, WAVES * 64, 0, stream>>>(p);
}

hipError_t launch_paged_decode(hipStream_t stream, int batch, int q_heads, int dim, const PagedCache &cache,
                               const PageTable &table, const Visibility &see, float scale, const void *q,
                               int64_t q_stride, void *out, int64_t out_stride, void *workspace, int compute_units)
{
    const int group = q_heads / cache.kv_heads, head_tiles = (group + HEADS - 1) / HEADS;
    const int items = cache.kv_heads * head_tiles;
    const int64_t capacity = int64_t(table.columns) << cache.page_shift;
    const int shares = decode_shares(int64_t(batch) * items, decode_positions(capacity, see), compute_units);
    DecodeParams p = {};
    p.batch = batch;
    p.group = group;
    p.head_tiles = head_tiles;
    p.cache = cache;
    p.table = table;
    p.see = see;
    p.scale = scale * LOG2E;
    p.q = static_cast<const unsigned short *>(q);
    p.out = static_cast<unsigned short *>(out);
    p.q_stride = q_stride;
    p.out_stride = out_stride;
    // (16 rows within the reach of 32-bit offsets)
    const bool large = cache.page_shift >= 4 && cache.slot_stride < (int64_t(1) << 26);
    if (shares == 0) {
        const dim3 grid(items, batch);
        // With less than a workgroup per compute unit eight wavefronts each (8 items of 129 positions, four / eight: 8.0 /
        // 7.3 us); with more workgroups than two per compute unit, as many as fit of four wavefronts, and few positions
        // two each (four / two: 1024 items of 64 positions 11.8 / 9.3 us, of 256 25.9 / 25.1, of 512 46.0 / 46.1; 512 of
        // 64 6.9 / 6.9).
        const int64_t workgroups = int64_t(batch) * items;
        if (workgroups < compute_units)
            launch_whole<8>(stream, dim, large, grid, p);
        else if (workgroups > 2 * compute_units && decode_positions(capacity, see) <= 256)
            launch_whole<2>(stream, dim, large, grid, p);
        else
            launch_whole<4>(stream, dim, large, grid, p);
        return launch_status();
    }
    const size_t rows = 2 * size_t(shares) * HEADS;
    p.part_o = static_cast<float *>(workspace);
    p.part_m = p.part_o + rows * dim;
    p.part_l = p.part_m + rows;
    p.joins = reinterpret_cast<int2 *>(p.part_l + rows);
    const auto kernel = dim == 128 ? (large ? paged_decode_shares_kernel<128, true> : paged_decode_shares_kernel<128, false>)
                                   : (large ? paged_decode_shares_kernel<64, true> : paged_decode_shares_kernel<64, false>);
    kernel<<<shares, SHARE_WAVES * 64, 0, stream>>>(p);
    hipError_t status = launch_status();
    if (status != hipSuccess)
        return status;
    const dim3 grid(q_heads, batch);
    if (dim == 128)
        paged_decode_join_kernel<128><<<grid, JOIN_THREADS, 0, stream>>>(p);
    else
        paged_decode_join_kernel<64><<<grid, JOIN_THREADS, 0, stream>>>(p);
    return launch_status();
}
} // namespace camblas_hip
