// Entry points of the paged key-value cache: append with per-head norm and rotation, decode and prefill
// attention (no counterpart in the reference).
#include "entry.hpp"
#include "paged_cache.hpp"

#include <cfloat>
#include <cmath>
#include <cstdint>

using namespace camblas_hip;

namespace camblas_hip
{
namespace
{
constexpr int64_t FAR = int64_t(1) << 32; // no stride of a row reaches as far (2^33 bytes)

// A cache the kernels can address: whole 16-byte pieces of every head, strides no shorter than a head. Rows may
// still share memory: see writable_cache.
bool valid_cache(const camblas_cuda_paged_cache *cache)
{
    if (!cache || !usable({{cache->k, 16}, {cache->v, 16}}) || cache->k == cache->v)
        return false;
    const bool shaped = (cache->dim == 64 || cache->dim == 128) && cache->pages >= 1 &&
                        (cache->page_size & (cache->page_size - 1)) == 0 &&
                        within({{cache->page_size, 1, 65536, 1}, {cache->kv_heads, 1, 65536, 1}}) &&
                        within({{cache->head_stride, 0, FAR, 8}, {cache->slot_stride, 0, FAR, 8}, {cache->page_stride, 0, FAR, 8}});
    return shaped && (cache->kv_heads == 1 || cache->head_stride >= cache->dim) &&
           (cache->page_size == 1 || cache->slot_stride >= cache->dim) &&
           (cache->pages == 1 ||
            within({{cache->page_stride, cache->dim, (int64_t(1) << 46) / cache->pages, 1}})); // (last byte: 2^47)
}

// No two rows of the cache share memory, those of keys and of values among each other: the append's wavefronts write
// them in no order. (Attention only reads them.)
bool writable_cache(const camblas_cuda_paged_cache *cache)
{
    const int64_t between = int64_t(reinterpret_cast<uintptr_t>(cache->v)) - int64_t(reinterpret_cast<uintptr_t>(cache->k));
    return places_apart({cache->pages, cache->page_stride}, {cache->page_size, cache->slot_stride},
                        {cache->kv_heads, cache->head_stride}, cache->dim, between / int64_t(sizeof(unsigned short)));
}

PagedCache device_cache(const camblas_cuda_paged_cache *cache)
{
    PagedCache to = {};
    to.k = static_cast<unsigned short *>(cache->k);
    to.v = static_cast<unsigned short *>(cache->v);
    to.page_stride = cache->page_stride;
    to.slot_stride = cache->slot_stride;
    to.head_stride = cache->head_stride;
    to.pages = cache->pages;
    while ((1 << to.page_shift) < cache->page_size)
        ++to.page_shift;
    to.kv_heads = cache->kv_heads;
    return to;
}

bool valid_heads(int q_heads, const camblas_cuda_paged_cache *cache)
{
    return q_heads >= 1 && q_heads <= 65536 && q_heads % cache->kv_heads == 0;
}

Visibility visible(const camblas_cuda_paged_cache *cache, int table_columns, int window, int sinks)
{
    return clipped(window, sinks, int64_t(table_columns) * cache->page_size);
}

// What both attentions ask of their arguments, `batch` sequences and `tokens` query rows.
bool valid_attention(int batch, int tokens, int q_heads, const camblas_cuda_paged_cache *cache, int64_t table_stride,
                     int table_columns, int window, int sinks, float scale, int64_t q_stride, int64_t output_stride)
{
    constexpr int64_t MOST = int64_t(1) << 30;
    return valid_heads(q_heads, cache) &&
           within({{batch, 0, 65535, 1}, {tokens, 0, INT32_MAX, 1}, {window, 0, INT32_MAX, 1}, {sinks, 0, INT32_MAX, 1},
                   {int64_t(tokens) * q_heads, 0, MOST, 1}, {int64_t(table_columns) * cache->page_size, 0, MOST, 1}}) &&
           table_columns >= 0 && table_stride >= 0 && std::isfinite(scale) && scale > 0.f && scale < 1e30f &&
           within({{q_stride, 0, FAR, 8}, {output_stride, 0, FAR, 8}}) &&
           (tokens <= 1 || output_stride >= int64_t(q_heads) * cache->dim);
}

// Where the pages of one array lie, first to last element.
Rows extent(const camblas_cuda_paged_cache *cache, const void *array)
{
    const int64_t last = int64_t(cache->pages - 1) * cache->page_stride +
                         int64_t(cache->page_size - 1) * cache->slot_stride +
                         int64_t(cache->kv_heads - 1) * cache->head_stride + cache->dim;
    return Rows{static_cast<const unsigned short *>(array), 1, last, 0};
}

Rows query_rows(const void *first, int rows, int heads, int dim, int64_t stride)
{
    return Rows{static_cast<const unsigned short *>(first), rows, int64_t(heads) * dim, stride};
}

// written rows share nothing with the cache
bool apart_from_cache(const Rows &written, const camblas_cuda_paged_cache *cache)
{
    return rows_apart(written, extent(cache, cache->k)) && rows_apart(written, extent(cache, cache->v));
}
} // namespace
} // namespace camblas_hip

extern "C" int camblas_cuda_qk_norm_rope_append(camblas_cuda_context *context, int tokens, int q_heads, int rotary_dim,
                                                float theta, int weight_dtype, float epsilon, const void *q_weight,
                                                const void *k_weight, const int32_t *positions, const int64_t *slots,
                                                const void *qkv, int64_t token_stride, void *queries,
                                                int64_t queries_stride, const camblas_cuda_paged_cache *cache)
{
    return camblas_cuda_qk_norm_rope_append_wide_theta(context, tokens, q_heads, rotary_dim, theta, weight_dtype, epsilon,
                                                       q_weight, k_weight, positions, slots, qkv, token_stride, queries,
                                                       queries_stride, cache);
}

extern "C" int camblas_cuda_qk_norm_rope_append_wide_theta(camblas_cuda_context *context, int tokens, int q_heads,
                                                           int rotary_dim, double theta, int weight_dtype, float epsilon,
                                                           const void *q_weight, const void *k_weight,
                                                           const int32_t *positions, const int64_t *slots, const void *qkv,
                                                           int64_t token_stride, void *queries, int64_t queries_stride,
                                                           const camblas_cuda_paged_cache *cache)
{
    Entry entry(context);
    return entry.run([&] {
        if (!valid_cache(cache))
            return entry.refuse("invalid paged cache");
        const int64_t width = (int64_t(q_heads) + 2 * int64_t(cache->kv_heads)) * cache->dim;
        const bool shaped = q_heads >= 1 && q_heads <= 65536 &&
                            within({{tokens, 0, 1 << 25, 1}, {rotary_dim, 0, cache->dim, 16}}) &&
                            theta >= 0x1p-149 && theta <= FLT_MAX && storage_in(weight_dtype, {0, 2}) && std::isfinite(epsilon) && epsilon >= 0 &&
                            within({{token_stride, 0, FAR, 8}, {queries_stride, 0, FAR, 8}}) &&
                            (tokens <= 1 || queries_stride >= int64_t(q_heads) * cache->dim);
        if (!shaped)
            return entry.refuse("invalid paged append arguments");
        if (!writable_cache(cache))
            return entry.refuse("paged append into a cache whose rows share memory");
        if (tokens == 0)
            return 0;
        // (the queries may replace their own un-rotated rows, which a workgroup reads before it writes them)
        const Rows in = {static_cast<const unsigned short *>(qkv), tokens, width, token_stride};
        const Rows out = query_rows(queries, tokens, q_heads, cache->dim, queries_stride);
        const bool in_place = queries == qkv && (tokens <= 1 || queries_stride == token_stride);
        if (!usable({{q_weight, 16, true}, {k_weight, 16, true}, {positions, 4}, {slots, 8}, {qkv, 16}, {queries, 16}}) ||
            !q_weight != !k_weight || !(in_place || rows_apart(in, out)) || !apart_from_cache(in, cache) ||
            !apart_from_cache(out, cache))
            return entry.refuse("invalid paged append buffers");
        return entry.finish(launch_qk_norm_rope_append(entry.stream(), tokens, q_heads, cache->dim, rotary_dim, theta, epsilon,
                                                       q_weight, k_weight, weight_dtype == 2, positions, slots, qkv,
                                                       token_stride, queries, queries_stride, device_cache(cache)),
                            "paged append");
    });
}

extern "C" size_t camblas_cuda_paged_decode_workspace_size(const camblas_cuda_context *context, int batch, int q_heads,
                                                           const camblas_cuda_paged_cache *cache, int table_columns,
                                                           int window, int sinks)
{
    if (!context || !valid_cache(cache) ||
        !valid_attention(batch, batch, q_heads, cache, table_columns, table_columns, window, sinks, 1.f,
                         int64_t(q_heads) * cache->dim, int64_t(q_heads) * cache->dim))
        return 0;
    return paged_decode_workspace(batch, q_heads, cache->kv_heads, cache->dim, int64_t(table_columns) * cache->page_size,
    visible(cache, table_columns, window, sinks), context->compute_units);
}

extern "C" int camblas_cuda_paged_decode_attention(camblas_cuda_context *context, int batch, int q_heads,
                                                   const camblas_cuda_paged_cache *cache, const int32_t *page_table,
                                                   int64_t table_stride, int table_columns, const int32_t *lengths,
                                                   int window, int sinks, float scale, const void *q, int64_t q_stride,
                                                   void *workspace, size_t workspace_bytes, void *output,
                                                   int64_t output_stride)
{
    Entry entry(context);
    return entry.run([&] {
        if (!valid_cache(cache))
            return entry.refuse("invalid paged cache");
        if (!valid_attention(batch, batch, q_heads, cache, table_stride, table_columns, window, sinks, scale, q_stride,
                             output_stride))
            return entry.refuse("invalid paged attention arguments");
        if (batch == 0)
            return 0;
        if (!usable({{page_table, 4, table_columns == 0}, {lengths, 4}, {q, 16}, {output, 16}}) ||
            !rows_apart(query_rows(output, batch, q_heads, cache->dim, output_stride),
                        query_rows(q, batch, q_heads, cache->dim, q_stride)) ||
            !apart_from_cache(query_rows(output, batch, q_heads, cache->dim, output_stride), cache))
            return entry.refuse("invalid paged attention buffers");
        const size_t bytes = paged_decode_workspace(batch, q_heads, cache->kv_heads, cache->dim,
                                                    int64_t(table_columns) * cache->page_size,
                                                    visible(cache, table_columns, window, sinks), context->compute_units);
        if (bytes && (!usable({{workspace, 16}}) || workspace_bytes < bytes))
            return entry.refuse("paged attention workspace is missing, misaligned or too small");
        context->counts[6]++;
        return entry.finish(launch_paged_decode(entry.stream(), batch, q_heads, cache->dim, device_cache(cache),
                                                PageTable{page_table, lengths, table_stride, table_columns},
                                                visible(cache, table_columns, window, sinks), scale, q, q_stride, output,
                                                output_stride, workspace, context->compute_units),
                            "paged decode attention");
    });
}

extern "C" size_t camblas_cuda_paged_prefill_workspace_size(const camblas_cuda_context *context, int batch, int tokens,
                                                            int q_heads, const camblas_cuda_paged_cache *cache,
                                                            int table_columns, int window, int sinks)
{
    if (!context || !valid_cache(cache) ||
        !valid_attention(batch, tokens, q_heads, cache, table_columns, table_columns, window, sinks, 1.f,
                         int64_t(q_heads) * cache->dim, int64_t(q_heads) * cache->dim))
        return 0;
    return paged_prefill_workspace(batch, tokens, q_heads, cache->kv_heads, cache->dim,
                                   int64_t(table_columns) * cache->page_size,
                                   visible(cache, table_columns, window, sinks), context->compute_units);
}

extern "C" int camblas_cuda_paged_prefill_attention(camblas_cuda_context *context, int batch, int tokens, int q_heads,
                                                    const camblas_cuda_paged_cache *cache, const int32_t *page_table,
                                                    int64_t table_stride, int table_columns, const int32_t *lengths,
                                                    const int32_t *query_starts, int window, int sinks, float scale,
                                                    const void *q, int64_t q_stride, void *workspace,
                                                    size_t workspace_bytes, void *output, int64_t output_stride)
{
    Entry entry(context);
    return entry.run([&] {
        if (!valid_cache(cache))
            return entry.refuse("invalid paged cache");
        if (!valid_attention(batch, tokens, q_heads, cache, table_stride, table_columns, window, sinks, scale, q_stride,
                             output_stride))
            return entry.refuse("invalid paged attention arguments");
        if (batch == 0 || tokens == 0)
            return 0;
        if (!usable({{page_table, 4, table_columns == 0}, {lengths, 4}, {query_starts, 4}, {q, 16}, {output, 16}}) ||
            !rows_apart(query_rows(output, tokens, q_heads, cache->dim, output_stride),
                        query_rows(q, tokens, q_heads, cache->dim, q_stride)) ||
            !apart_from_cache(query_rows(output, tokens, q_heads, cache->dim, output_stride), cache))
            return entry.refuse("invalid paged attention buffers");
        const size_t bytes = paged_prefill_workspace(batch, tokens, q_heads, cache->kv_heads, cache->dim,
                                                     int64_t(table_columns) * cache->page_size,
                                                     visible(cache, table_columns, window, sinks), context->compute_units);
        if (bytes && (!usable({{workspace, 16}}) || workspace_bytes < bytes))
            return entry.refuse("paged attention workspace is missing, misaligned or too small");
        context->counts[6]++;
        return entry.finish(launch_paged_prefill(entry.stream(), batch, tokens, q_heads, cache->dim, device_cache(cache),
                                                 PageTable{page_table, lengths, table_stride, table_columns},
                                                 visible(cache, table_columns, window, sinks), query_starts, scale, q, q_stride,
                                                 output, output_stride, workspace, context->compute_units),
                            "paged prefill attention");
    });
}
