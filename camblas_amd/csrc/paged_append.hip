// What a decoder layer does with a fused QKV activation before attention over a paged cache, in one
// launch: the RMS norm of every query and key head (optional), the rotary embedding, the queries into
// their output, keys and values into their slots.
//
//   y = x * rsqrt(mean(x^2) + epsilon) * weight          over one head's dims
//   (lo, hi) -> (lo cos a - hi sin a, hi cos a + lo sin a)   lo = y[i], hi = y[i + rotary / 2],
//                                                        a = position * theta^(-2 i / rotary)
//
// All of it in FP32 with one rounding to BF16 at the end. The angle is formed in FP64, from a base in FP64, as a
// number of turns, of which the whole ones are dropped before the FP32 sine and cosine: at position 2^20 an angle
// in FP32 is off by up to 2^-4 of a radian, and one whose base is rounded to FP32 by up to 2^-8.
//
// A lane owns eight pairs of a head: dims 8 j .. 8 j + 7 and rotary / 2 further (dims that are not
// rotated are dealt in the same way: two runs of eight), so dim / 16 lanes hold a head, the sum of squares
// stays within them and the angles of a lane are the same for every head of a token. A wavefront takes
// some or all heads of one token. Bound by the copy of the rows (4096 tokens of 80 heads of 128: 32.4 us, 5.2 TB/s,
// where a large copy reaches 4.9), small calls by the launch.
#include "common.hpp"
#include "device.hpp"
#include "paged_cache.hpp"

#include <cmath>

namespace camblas_hip
{
namespace
{
constexpr int APPEND_WAVES = 4;

struct AppendParams {
    int tokens, q_heads, parts, groups_per_part;
    int half; // rotary / 2
    float epsilon;
    const void *q_weight, *k_weight; // null: no norm
    int weight_bf16;
    const int32_t *positions;
    const int64_t *slots;
    const unsigned short *qkv;
    unsigned short *q_out;
    int64_t token_stride, out_stride;
    PagedCache cache;
    double powers[6]; // theta^(-2 i / rotary) for i = 1, 2, 4, .. 32
};

__device__ __forceinline__ void load_weights(const void *weight, int bf16, int at, float (&w)[8])
{
    if (bf16) {
        const u32x4_t packed = *reinterpret_cast<const u32x4_t *>(static_cast<const unsigned short *>(weight) + at);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            w[2 * e] = __uint_as_float(packed[e] << 16);
            w[2 * e + 1] = __uint_as_float(packed[e] & 0xffff0000u);
        }
    } else {
        const float *from = static_cast<const float *>(weight) + at;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            w[e] = from[e];
    }
}

__device__ __forceinline__ void unpack(const u32x4_t &packed, float (&x)[8])
{
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        x[2 * e] = __uint_as_float(packed[e] << 16);
        x[2 * e + 1] = __uint_as_float(packed[e] & 0xffff0000u);
    }
}

__device__ __forceinline__ u32x4_t pack(const float (&x)[8])
{
    return u32x4_t{round_pair(x[0], x[1]), round_pair(x[2], x[3]), round_pair(x[4], x[5]), round_pair(x[6], x[7])};
}

// Un-rotated rows are not read again: past the caches (4096 tokens of 80 heads of 128 in a loop over fresh rows 37.8 / 32.4
// us). Stores stay ordinary: written past the caches as well the same call takes 29.7 us, but the attention that reads
// them next loses more than that (4096 tokens, both together 321 / 332 us).
__device__ __forceinline__ u32x4_t load_once(const unsigned short *from)
{
    return __builtin_nontemporal_load(reinterpret_cast<const u32x4_t *>(from));
}

template <int DIM> __global__ __launch_bounds__(APPEND_WAVES * 64) void qk_norm_rope_append_kernel(AppendParams p)
{
    constexpr int LANES = DIM / 16, HEADS = 64 / LANES; // lanes of a head, heads a wavefront takes at once
    const int lane = threadIdx.x % 64;
    const int64_t index = int64_t(blockIdx.x) * APPEND_WAVES + threadIdx.x / 64;
    const int token = int(index / p.parts), part = int(index % p.parts);
    if (token >= p.tokens)
        return;
    const int j = lane % LANES, rotating = p.half / 8; // lanes of a head whose dims are rotated
    const bool rotates = j < rotating;
    const int low = rotates ? 8 * j : 2 * p.half + 16 * (j - rotating);
    const int high = rotates ? low + p.half : low + 8;
    const int kv_heads = p.cache.kv_heads, heads = p.q_heads + 2 * kv_heads;

    // One angle a lane, handed round through a wavefront's own part of LDS (every lane working out its own eight
    // was half of the time of heads of 64: 4096 tokens of 30 heads 11.6 us).
    __shared__ __attribute__((aligned(16))) float sines[APPEND_WAVES][64], cosines[APPEND_WAVES][64];
    const int wave = threadIdx.x / 64;
    {
        // theta^(-2 lane / rotary) as a product over the bits of the lane (64 values worked out on the host were 2 of
        // the 6 us of a small call). A square doubles the relative error of its power and rounds once, so that lane i is
        // off by (3 i + 8) 2^-53 of its turn at most; turns get shorter faster than that grows: under 2^-18 of a radian
        // at position 2^31 and a base of 10^4 or more.
        double turn = double(p.positions[token]) * (1 / 6.283185307179586476925);
#pragma unroll
        for (int bit = 0; bit < 6; ++bit)
            turn *= lane >> bit & 1 ? p.powers[bit] : 1.0;
        float s, c;
        sincospif(2.f * float(turn - rint(turn)), &s, &c);
        sines[wave][lane] = s;
        cosines[wave][lane] = c;
    }
    asm volatile("" ::: "memory");
    float s[8], c[8];
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
        const f32x4_t four_s = *reinterpret_cast<const f32x4_t *>(&sines[wave][rotates ? 8 * j + e : 0]);
        const f32x4_t four_c = *reinterpret_cast<const f32x4_t *>(&cosines[wave][rotates ? 8 * j + e : 0]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s[e + i] = four_s[i];
            c[e + i] = four_c[i];
        }
    }
    float q_low[8], q_high[8], k_low[8], k_high[8];
    if (p.q_weight) {
        load_weights(p.q_weight, p.weight_bf16, low, q_low);
        load_weights(p.q_weight, p.weight_bf16, high, q_high);
        load_weights(p.k_weight, p.weight_bf16, low, k_low);
        load_weights(p.k_weight, p.weight_bf16, high, k_high);
    }
    const int64_t slot = p.slots[token];
    const int64_t page = slot >> p.cache.page_shift;
    const bool stored = slot >= 0 && page < p.cache.pages;
    const int64_t row = stored ? row_offset(p.cache, int(page), int(slot & ((int64_t(1) << p.cache.page_shift) - 1))) : 0;

    const unsigned short *from = p.qkv + int64_t(token) * p.token_stride;
    const int first = part * p.groups_per_part * HEADS + lane / LANES;
    const int last = min(heads, (part + 1) * p.groups_per_part * HEADS);
    u32x4_t next_lo = {0, 0, 0, 0}, next_hi = next_lo;
    if (first < last) {
        next_lo = load_once(from + int64_t(first) * DIM + low);
        next_hi = load_once(from + int64_t(first) * DIM + high);
    }
    for (int head = first; head < last; head += HEADS) {
        u32x4_t lo = next_lo, hi = next_hi;
        if (head + HEADS < last) { // (travels while this one is worked on)
            next_lo = load_once(from + int64_t(head + HEADS) * DIM + low);
            next_hi = load_once(from + int64_t(head + HEADS) * DIM + high);
        }
        const bool is_query = head < p.q_heads, is_value = head >= p.q_heads + kv_heads;
        float x[8], y[8];
        unpack(lo, x);
        unpack(hi, y);
        if (p.q_weight) {
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                sum = fmaf(x[e], x[e], fmaf(y[e], y[e], sum));
            sum += dpp_move<0xB1>(sum);
            sum += dpp_move<0x4E>(sum);
            if (LANES == 8)
                sum += dpp_move<0x141>(sum);
            const float inverse = 1.f / sqrtf(sum * (1.f / DIM) + p.epsilon);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] *= inverse * (is_query ? q_low[e] : k_low[e]);
                y[e] *= inverse * (is_query ? q_high[e] : k_high[e]);
            }
        }
        if (!is_value) {
            float a[8], b[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                a[e] = x[e] * c[e] - y[e] * s[e];
                b[e] = y[e] * c[e] + x[e] * s[e];
            }
            // (dims that are not rotated and not normalised pass bit for bit, NaN payloads and infinities too)
            if (rotates || p.q_weight) {
                lo = pack(rotates ? a : x);
                hi = pack(rotates ? b : y);
            }
        }
        if (is_query) {
            unsigned short *to = p.q_out + int64_t(token) * p.out_stride + int64_t(head) * DIM;
            *reinterpret_cast<u32x4_t *>(to + low) = lo;
            *reinterpret_cast<u32x4_t *>(to + high) = hi;
        } else if (stored) {
            const int kv = head - p.q_heads - (is_value ? kv_heads : 0);
            unsigned short *to = (is_value ? p.cache.v : p.cache.k) + row + int64_t(kv) * p.cache.head_stride;
            *reinterpret_cast<u32x4_t *>(to + low) = lo;
            *reinterpret_cast<u32x4_t *>(to + high) = hi;
        }
    }
}
} // namespace

hipError_t launch_qk_norm_rope_append(hipStream_t stream, int tokens, int q_heads, int dim, int rotary, double theta,
                                      float epsilon, const void *q_weight, const void *k_weight, bool weight_bf16,
                                      const int32_t *positions, const int64_t *slots, const void *qkv,
                                      int64_t token_stride, void *q_out, int64_t out_stride, const PagedCache &cache)
{
    AppendParams p = {};
    p.tokens = tokens;
    p.q_heads = q_heads;
    p.half = rotary / 2;
    p.epsilon = epsilon;
    p.q_weight = q_weight;
    p.k_weight = k_weight;
    p.weight_bf16 = weight_bf16;
    p.positions = positions;
    p.slots = slots;
    p.qkv = static_cast<const unsigned short *>(qkv);
    p.q_out = static_cast<unsigned short *>(q_out);
    p.token_stride = token_stride;
    p.out_stride = out_stride;
    p.cache = cache;
    double power = rotary ? std::pow(theta, -2.0 / rotary) : 1;
    for (double &of : p.powers) {
        of = power;
        power *= power;
    }
    const int heads = q_heads + 2 * cache.kv_heads, at_once = 1024 / dim;
    const int groups = (heads + at_once - 1) / at_once;
    // some 4096 wavefronts, four a SIMD, if there are as many groups of heads (2048 / 4096 / 8192 wavefronts: 256 tokens of 80
    // heads of 128 6.3 / 5.7 / 5.7 us, 1500 16.4 / 14.6 / 15.8, 883 of 45 8.0 / 8.0 / 9.2)
    const int wanted = 4096 / tokens;
    p.parts = wanted < 1 ? 1 : wanted < groups ? wanted : groups;
    p.groups_per_part = (groups + p.parts - 1) / p.parts;
    const int64_t waves = int64_t(tokens) * p.parts;
    const unsigned blocks = unsigned((waves + APPEND_WAVES - 1) / APPEND_WAVES);
    if (dim == 128)
        qk_norm_rope_append_kernel<128><<<blocks, APPEND_WAVES * 64, 0, stream>>>(p);
    else
        qk_norm_rope_append_kernel<64><<<blocks, APPEND_WAVES * 64, 0, stream>>>(p);
    return launch_status();
}
} // namespace camblas_hip
