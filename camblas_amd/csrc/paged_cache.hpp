// The paged key-value cache as its kernels see it, and which of its rows a query sees.
//
// A cache is two BF16 arrays of pages (keys, values; the same strides), each page holding page_size
// positions of every key-value head. A sequence's positions are found through its row of a page table:
// position p lies in page table[p / page_size], slot p % page_size. An entry outside [0, pages), or a
// position behind the table's last column, holds nothing: it is neither read nor attended to.
#pragma once

#include "common.hpp"
#include "device.hpp"

namespace camblas_hip
{
struct PagedCache {
    unsigned short *k, *v;
    int64_t page_stride, slot_stride, head_stride; // in elements, multiples of eight
    int pages, page_shift, kv_heads;               // page_size = 1 << page_shift
};

struct PageTable {
    const int32_t *pages;   // [sequences][stride]
    const int32_t *lengths; // positions of each sequence that hold a token, clipped to the table
    int64_t stride;
    int columns;
};

// A query at position p sees positions p - window + 1 .. p (window 0: 0 .. p) and those below `sinks`.
struct Visibility {
    int window, sinks;
};

// ---- launchers (each returns a hipError_t); what they ask of their arguments is checked by the entry points
hipError_t launch_qk_norm_rope_append(hipStream_t stream, int tokens, int q_heads, int dim, int rotary, float theta,
                                      float epsilon, const void *q_weight, const void *k_weight, bool weight_bf16,
                                      const int32_t *positions, const int64_t *slots, const void *qkv,
                                      int64_t token_stride, void *q_out, int64_t out_stride, const PagedCache &cache);
size_t paged_decode_workspace(int batch, int q_heads, int kv_heads, int dim, int64_t capacity, int window, int sinks,
                              int compute_units);
hipError_t launch_paged_decode(hipStream_t stream, int batch, int q_heads, int dim, const PagedCache &cache,
                               const PageTable &table, const Visibility &see, float scale, const void *q,
                               int64_t q_stride, void *out, int64_t out_stride, void *workspace, int compute_units);
size_t paged_prefill_workspace(int batch, int tokens, int q_heads, int kv_heads, int dim, int64_t capacity, int window, int sinks,
                               int compute_units);
hipError_t launch_paged_prefill(hipStream_t stream, int batch, int tokens, int q_heads, int dim, const PagedCache &cache,
                                const PageTable &table, const Visibility &see, const int32_t *starts, float scale,
                                const void *q, int64_t q_stride, void *out, int64_t out_stride, void *workspace,
                                int compute_units);

// Two values to BF16 in one word, round to nearest even, NaN stays NaN: one instruction.
__device__ __forceinline__ unsigned round_pair(float lo, float hi)
{
    typedef float pair_f32 __attribute__((ext_vector_type(2)));
    typedef __bf16 pair_bf16 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(unsigned, __builtin_convertvector((pair_f32{lo, hi}), pair_bf16));
}

// The page of `position`, or -1 where the table or the cache has none.
__device__ __forceinline__ int page_of(const PagedCache &cache, const int32_t *row, int columns, int position)
{
    const int column = position >> cache.page_shift;
    if (column >= columns)
        return -1;
    const int page = row[column];
    return unsigned(page) < unsigned(cache.pages) ? page : -1;
}

// Element offset of a position's row of head 0 inside the key or value array (page >= 0).
__device__ __forceinline__ int64_t row_offset(const PagedCache &cache, int page, int position)
{
    return int64_t(page) * cache.page_stride + int64_t(position & ((1 << cache.page_shift) - 1)) * cache.slot_stride;
}

__device__ __forceinline__ int live_positions(const PageTable &table, const PagedCache &cache, int sequence)
{
    const int64_t capacity = int64_t(table.columns) << cache.page_shift;
    const int64_t length = table.lengths[sequence];
    return int(length < 0 ? 0 : length < capacity ? length : capacity);
}

// The positions that queries first .. last of one sequence see between them, in tiles of TILE positions
// that start at multiples of TILE: those of the first tokens, [0, sink_tiles * TILE), then from `begin`
// (a multiple of TILE) to `end`. The two never overlap; a tile may hold positions that some query, or
// none, sees.
template <int TILE> struct TileSpan {
    int sink_tiles, begin, end, tiles;

    __device__ __forceinline__ TileSpan(const Visibility &see, int first, int last)
    {
        end = last + 1;
        begin = 0;
        sink_tiles = 0;
        if (see.window > 0 && first >= see.window) {
            begin = (first - see.window + 1) / TILE * TILE;
            const int sinks = (min(see.sinks, begin) + TILE - 1) / TILE;
            sink_tiles = min(sinks, begin / TILE);
        }
        tiles = end > begin ? sink_tiles + (end - begin + TILE - 1) / TILE : 0;
    }
    __device__ __forceinline__ int position(int tile) const
    {
        return tile < sink_tiles ? tile * TILE : begin + (tile - sink_tiles) * TILE;
    }
};

__device__ __forceinline__ bool sees(const Visibility &see, int query, int position)
{
    return position <= query && (see.window <= 0 || position > query - see.window || position < see.sinks);
}
} // namespace camblas_hip
