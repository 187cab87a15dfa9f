// New rows into a cache in pages, and rows back out of it (gptoss_attn_paged_write, gptoss_attn_paged_read).
//
// Eight lanes take a row of 64, eight numbers each.  What bounds both: a decoding step's write is one launch's latency; prompts and
// reads move bytes, K and V by the same thread so that both rows are under way together.
#pragma once
#include "paged_common.h"

namespace gptoss {

// The row's power of two from its largest finite number (over the eight lanes of the row), see gptoss_attn.h.
__device__ __forceinline__ int row_exponent(const float (&x)[8]) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t u = __float_as_uint(x[i]) & 0x7fffffffu;      // finite magnitudes compare as their bits do
        top = max(top, u < 0x7f800000u ? u : 0u);
    }
    top = max(top, (uint32_t)__shfl_xor((int)top, 1));
    top = max(top, (uint32_t)__shfl_xor((int)top, 2));
    top = max(top, (uint32_t)__shfl_xor((int)top, 4));
    // 448 = 1.75 * 2^8 (numbers below 2^-126 have no leading one: their exponent is under the smallest one in any case)
    return max((int)(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0), kMinExp);
}

__device__ __forceinline__ uint2 e4m3_codes(const float (&x)[8], int s) {
    const float inv = exp_of_byte((uint32_t)(kExpBias - s));         // 2^-s: the products are exact, but for numbers that round to 0
    // next to 2^128 the nearest code would come back as infinity: 240 * 2^120 instead (still within 2^-4)
    const float most = s == kMaxExp ? 240.0f : 448.0f;
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
        y[i] = (__float_as_uint(x[i]) & 0x7fffffffu) < 0x7f800000u ? __builtin_amdgcn_fmed3f(x[i] * inv, -most, most) : __uint_as_float(0x7fc00000u);
    int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false), hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], 0, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], hi, true);
    return make_uint2((uint32_t)lo, (uint32_t)hi);
}

template <typename T>
__device__ __forceinline__ void store_quantised(char *row, char *exp, int c8, const T *src) {
    float x[8];
    load8(src + c8, x);
    const int s = row_exponent(x);
    *reinterpret_cast<uint2 *>(row + c8) = e4m3_codes(x, s);
    if (c8 == 0) *exp = (char)(s + kExpBias);
}

template <typename T>
__device__ __forceinline__ void copy8(T *dst, const T *src) {
#pragma unroll
    for (int i = 0; i < (int)(8 * sizeof(T) / 16); ++i) reinterpret_cast<u32x4 *>(dst)[i] = reinterpret_cast<const u32x4 *>(src)[i];
}

// Rows (token, KV head) of a batch row, the KV head fastest: the model's keys and values have a token's heads side by side.
template <typename T, bool E4M3>
__global__ __launch_bounds__(256) void paged_write_kernel(const PagedArgs a) {
    const int b = blockIdx.x / a.blocks, row = (blockIdx.x % a.blocks) * 32 + (threadIdx.x >> 3), c8 = (threadIdx.x & 7) * 8;
    const int i = row / a.G, g = row % a.G;
    const int n = a.seqlens ? min(a.seqlens[b], a.Sq) : a.Sq;
    if (i >= n) return;                                              // (all eight lanes of the row)
    const int64_t pos = (int64_t)a.start[b] + i;
    const int page = pos < 0 || pos > 0x7fffffff ? -1 : paged_page(a, b, (int)pos);
    if (page < 0) return;
    const T *k = reinterpret_cast<const T *>(a.k) + b * a.ks.b + g * a.ks.h + i * a.ks.s;
    const T *v = reinterpret_cast<const T *>(a.v) + b * a.vs.b + g * a.vs.h + i * a.vs.s;
    const int at = (int)pos & ((1 << a.page_shift) - 1);
    char *kr = a.kp.head(g) + a.kp.at(page, at), *vr = a.vp.head(g) + a.vp.at(page, at);
    if constexpr (E4M3) {
        store_quantised(kr, a.ke.head(g) + a.ke.at(page, at), c8, k);
        store_quantised(vr, a.ve.head(g) + a.ve.at(page, at), c8, v);
    } else {
        copy8(reinterpret_cast<T *>(kr) + c8, k + c8);
        copy8(reinterpret_cast<T *>(vr) + c8, v + c8);
    }
}

template <typename T, typename ST>
__device__ __forceinline__ void read8(T *dst, const char *row, const char *exp, int c8, bool there) {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = 0.0f;
    if (there) {
        load8(reinterpret_cast<const ST *>(row) + c8, x);
        if constexpr (sizeof(ST) == 1) {
            const float f = exp_of_byte(*reinterpret_cast<const uint8_t *>(exp));
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] *= f;
        }
    }
    store8(dst + c8, x);
}

// Rows of a (batch row, KV head), which lie side by side in the result.
template <typename T, typename ST>
__global__ __launch_bounds__(256) void paged_read_kernel(const PagedArgs a) {
    int bid = blockIdx.x;
    const int i = (bid % a.blocks) * 32 + (threadIdx.x >> 3), c8 = (threadIdx.x & 7) * 8;
    bid /= a.blocks;
    const int g = bid % a.G, b = bid / a.G;
    if (i >= a.Sq) return;
    const int64_t pos = (a.start ? (int64_t)a.start[b] : 0) + i;
    const int page = pos >= 0 && pos < paged_length(a, b) ? paged_page(a, b, (int)pos) : -1;
    const bool there = page >= 0;
    const int at = (int)pos & ((1 << a.page_shift) - 1), p = there ? page : 0;
    read8<T, ST>(reinterpret_cast<T *>(a.k) + b * a.ks.b + g * a.ks.h + i * a.ks.s, a.kp.head(g) + a.kp.at(p, at), a.ke.head(g) + a.ke.at(p, at), c8, there);
    read8<T, ST>(reinterpret_cast<T *>(a.v) + b * a.vs.b + g * a.vs.h + i * a.vs.s, a.vp.head(g) + a.vp.at(p, at), a.ve.head(g) + a.ve.at(p, at), c8, there);
}

}  // namespace gptoss
