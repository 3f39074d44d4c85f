// The paged key-value cache as its kernels see it, and which of its rows a query sees.
//
// A cache is two BF16 arrays of pages (keys, values; the same strides), each page holding page_size
// positions of every key-value head. A sequence's positions are found through its row of a page table:
// position p lies in page table[p / page_size], slot p % page_size. An entry outside [0, pages), or a
// position behind the table's last column, holds nothing: it is neither read nor attended to.
#pragma once

#include "common.hpp"
#include "device.hpp"
#include "paged_span.hpp"

#include <cfloat>
#include <cmath>

namespace camblas_hip
{
// ---- launchers (each returns a hipError_t); what they ask of their arguments is checked by the entry points
hipError_t launch_qk_norm_rope_append(hipStream_t stream, int tokens, int q_heads, int dim, int rotary, double theta,
                                      float epsilon, const void *q_weight, const void *k_weight, bool weight_bf16,
                                      const int32_t *positions, const int64_t *slots, const void *qkv,
                                      int64_t token_stride, void *q_out, int64_t out_stride, const PagedCache &cache);
size_t paged_decode_workspace(int batch, int q_heads, int kv_heads, int dim, int64_t capacity, const Visibility &see,
                              int compute_units);
hipError_t launch_paged_decode(hipStream_t stream, int batch, int q_heads, int dim, const PagedCache &cache,
                               const PageTable &table, const Visibility &see, float scale, const void *q,
                               int64_t q_stride, void *out, int64_t out_stride, void *workspace, int compute_units);
size_t paged_prefill_workspace(int batch, int tokens, int q_heads, int kv_heads, int dim, int64_t capacity,
                               const Visibility &see, int compute_units);
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

// What the weighted sum of a head is multiplied by at the end, from the running maximum and the sum of weights. A head
// that has seen no position keeps a maximum of minus infinity and gives zeros. One whose scores were all minus
// infinity has a finite maximum (no score is below it) and a sum of zero: 0 / 0, NaN. A sum that is NaN stays NaN.
__device__ __forceinline__ float normaliser(float top, float sum)
{
    return sum != 0.f ? 1.f / sum : top == -INFINITY ? 0.f : __builtin_nanf("");
}
} // namespace camblas_hip
