// The paged cache's whole-number arithmetic compiled for the CPU, behind a C interface for the tests.
#include "paged_span.hpp"

using namespace camblas_hip;

extern "C" int span_tiles(int tile, int window, int sinks, int first, int last, int *positions, int room)
{
    const Visibility see = {window, sinks};
    const auto list = [&](const auto &span) {
        for (int t = 0; t < span.tiles && t < room; ++t)
            positions[t] = span.position(t);
        return span.tiles;
    };
    return tile == 32 ? list(TileSpan<32>(see, first, last)) : list(TileSpan<64>(see, first, last));
}
extern "C" int is_seen(int window, int sinks, int query, int position) { return sees(Visibility{window, sinks}, query, position); }
extern "C" void clip(int window, int sinks, int64_t capacity, int *out)
{
    const Visibility see = clipped(window, sinks, capacity);
    out[0] = see.window;
    out[1] = see.sinks;
}
extern "C" int find_page(const int32_t *row, int columns, int pages, int page_shift, int position)
{
    PagedCache cache = {};
    cache.pages = pages;
    cache.page_shift = page_shift;
    return page_of(cache, row, columns, position);
}
extern "C" int64_t find_row(int64_t page_stride, int64_t slot_stride, int page_shift, int page, int position)
{
    PagedCache cache = {};
    cache.page_stride = page_stride;
    cache.slot_stride = slot_stride;
    cache.page_shift = page_shift;
    return row_offset(cache, page, position);
}
extern "C" int find_length(int32_t length, int columns, int page_shift)
{
    PagedCache cache = {};
    cache.page_shift = page_shift;
    return live_positions(PageTable{nullptr, &length, 0, columns}, cache, 0);
}
extern "C" int64_t find_share_begin(int64_t all, int64_t workers, int64_t g) { return share_begin(all, workers, g); }
extern "C" int64_t find_share(int64_t all, int64_t workers, int64_t step) { return share_of(all, workers, step); }
extern "C" int find_first_block(int token, int group, int rows, int sequence) { return first_block(token, group, rows, sequence); }
extern "C" int find_apart(int64_t a, int64_t a_count, int64_t a_width, int64_t a_stride, int64_t b, int64_t b_count, int64_t b_width,
                          int64_t b_stride)
{
    const auto *memory = reinterpret_cast<const unsigned short *>(uintptr_t(1) << 40);
    return rows_apart(Rows{memory + a, a_count, a_width, a_stride}, Rows{memory + b, b_count, b_width, b_stride});
}
extern "C" int find_places_apart(const int64_t *counts, const int64_t *strides, int64_t width, int64_t offset)
{
    return places_apart({counts[0], strides[0]}, {counts[1], strides[1]}, {counts[2], strides[2]}, width, offset);
}
