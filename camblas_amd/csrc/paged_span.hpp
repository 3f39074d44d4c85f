// The whole-number arithmetic of the paged cache's kernels: where a position's row lies, which positions a
// query sees and in which tiles, how work is numbered and dealt to workgroups. Plain C++, so that it can be
// checked on a CPU as well.
#pragma once

#include <cstdint>
#include <initializer_list>

#if defined(__HIPCC__)
#define PAGED_INLINE __host__ __device__ __forceinline__
#else
#define PAGED_INLINE inline
#endif

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

// The same with numbers no larger than a table's capacity (at most 2^30): a window that reaches all of it is none.
PAGED_INLINE Visibility clipped(int window, int sinks, int64_t capacity)
{
    return Visibility{window < capacity ? window : 0, int(sinks < capacity ? sinks : capacity)};
}

PAGED_INLINE bool sees(const Visibility &see, int query, int position)
{
    return position <= query && (see.window <= 0 || position > query - see.window || position < see.sinks);
}

// The page of `position`, or -1 where the table or the cache has none.
PAGED_INLINE int page_of(const PagedCache &cache, const int32_t *row, int columns, int position)
{
    const int column = position >> cache.page_shift;
    if (column >= columns)
        return -1;
    const int page = row[column];
    return unsigned(page) < unsigned(cache.pages) ? page : -1;
}

// Element offset of a position's row of head 0 inside the key or value array (page >= 0).
PAGED_INLINE int64_t row_offset(const PagedCache &cache, int page, int position)
{
    return int64_t(page) * cache.page_stride + int64_t(position & ((1 << cache.page_shift) - 1)) * cache.slot_stride;
}

PAGED_INLINE int live_positions(const PageTable &table, const PagedCache &cache, int sequence)
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

    PAGED_INLINE TileSpan(const Visibility &see, int first, int last)
    {
        end = last + 1;
        begin = 0;
        sink_tiles = 0;
        if (see.window > 0 && first >= see.window) {
            begin = (first - see.window + 1) / TILE * TILE;
            const int sinks = ((see.sinks < begin ? see.sinks : begin) + TILE - 1) / TILE;
            sink_tiles = sinks < begin / TILE ? sinks : begin / TILE;
        }
        tiles = end > begin ? sink_tiles + (end - begin + TILE - 1) / TILE : 0;
    }
    PAGED_INLINE int position(int tile) const
    {
        return tile < sink_tiles ? tile * TILE : begin + (tile - sink_tiles) * TILE;
    }
};

// Rows of `width` elements, `stride` apart.
struct Rows {
    const unsigned short *first;
    int64_t count, width, stride;
};

// Whether no element of one lies in the other. Rows of one stride may lie between each other (heads of one
// activation); of different strides they may not even interleave.
inline bool rows_apart(const Rows &a, const Rows &b)
{
    if (a.count <= 0 || b.count <= 0)
        return true;
    const uintptr_t a_begin = reinterpret_cast<uintptr_t>(a.first), b_begin = reinterpret_cast<uintptr_t>(b.first);
    const uintptr_t a_end = a_begin + uintptr_t((a.count - 1) * a.stride + a.width) * sizeof(unsigned short);
    const uintptr_t b_end = b_begin + uintptr_t((b.count - 1) * b.stride + b.width) * sizeof(unsigned short);
    if (a_end <= b_begin || b_end <= a_begin)
        return true;
    const int64_t stride = a.count > 1 ? a.stride : b.stride;
    if (stride <= 0 || (a.count > 1 && b.count > 1 && a.stride != b.stride))
        return false;
    const int64_t bytes = stride * int64_t(sizeof(unsigned short));
    int64_t along = (int64_t(b_begin) - int64_t(a_begin)) % bytes; // of b's rows inside a's
    along += along < 0 ? bytes : 0;
    return along >= a.width * int64_t(sizeof(unsigned short)) && along + b.width * int64_t(sizeof(unsigned short)) <= bytes;
}

// `count` places `stride` elements apart.
struct Axis {
    int64_t count, stride;
};

// Whether steps along `axes` (fewer than count either way) can bring `offset` within `width` of zero. An axis whose stride
// is no shorter than what the ones behind it span leaves two steps to try; `tries` bounds the others, and
// running out of them counts as yes.
inline bool steps_reach(const Axis *axes, int rank, int64_t offset, int64_t width, int &tries)
{
    if (--tries < 0)
        return true;
    if (rank == 0)
        return -width < offset && offset < width;
    int64_t span = width - 1; // of what is left to step along, and a row
    for (int i = 1; i < rank; ++i)
        span += (axes[i].count - 1) * axes[i].stride;
    const int64_t most = axes[0].count - 1, stride = axes[0].stride;
    // -span <= offset + step * stride <= span, rounded outwards
    int64_t step = (-span - offset) / stride - 1, last = (span - offset) / stride + 1;
    step = step < -most ? -most : step;
    last = last > most ? most : last;
    for (; step <= last; ++step)
        if (steps_reach(axes + 1, rank - 1, offset + step * stride, width, tries))
            return true;
    return false;
}

// Whether all rows of `width` elements along three axes are apart from each other, and from the same rows `offset`
// elements further (keys and values of a cache). Exact for every layout that slices and transposes of one dense
// tensor can have; of others a few that take more than 4096 tries are taken to overlap.
inline bool places_apart(Axis a, Axis b, Axis c, int64_t width, int64_t offset)
{
    Axis axes[3];
    int rank = 0;
    for (const Axis &axis : {a, b, c}) // in descending order of strides; an axis of one place says nothing
        if (axis.count > 1) {
            int at = rank++;
            for (; at > 0 && axes[at - 1].stride < axis.stride; --at)
                axes[at] = axes[at - 1];
            axes[at] = axis;
        }
    if (rank > 0 && axes[rank - 1].stride <= 0)
        return false;
    int tries = 4096;
    int64_t span = width - 1; // of the axes behind i, and a row
    for (int i = rank - 1; i >= 0; --i) { // two rows whose first different step is along axis i
        for (int64_t step = 1; step < axes[i].count && step * axes[i].stride <= span; ++step)
            if (steps_reach(axes + i + 1, rank - i - 1, step * axes[i].stride, width, tries))
                return false;
        span += (axes[i].count - 1) * axes[i].stride;
    }
    return !steps_reach(axes, rank, offset, width, tries);
}

// `all` steps dealt to `workers` (at most as many) in runs that differ by one step at most: the first step of
// worker g's run, and the worker that holds a step.
PAGED_INLINE int64_t share_begin(int64_t all, int64_t workers, int64_t g) { return all * g / workers; }
PAGED_INLINE int64_t share_of(int64_t all, int64_t workers, int64_t step) { return ((step + 1) * workers - 1) / all; }

// Blocks of `rows` rows (token, query head of a group) of sequence b are numbered from here on: a number that
// needs no sum over the sequences before, leaves room for a last block that is not full, and at most one
// unused number per sequence. (first_token * group is below 2^31.)
PAGED_INLINE int first_block(int first_token, int group, int rows, int sequence)
{
    return first_token * group / rows + sequence;
}
} // namespace camblas_hip
