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

// Eight numbers of a row as they travel.
template <typename T> struct Piece { u32x4 u[sizeof(T) / 2]; };
template <typename T>
__device__ __forceinline__ Piece<T> load_piece(const T *p) {
    Piece<T> x;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); ++i) x.u[i] = reinterpret_cast<const u32x4 *>(p)[i];
    return x;
}
template <typename T>
__device__ __forceinline__ void numbers_of(const Piece<T> &p, float (&x)[8]) {
    if constexpr (sizeof(T) == 2) {
        const bf16x8 v = as_bf16x8(p.u[0]);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (float)v[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(p.u[i >> 2][i & 3]);
    }
}

template <typename T, bool E4M3>
__device__ __forceinline__ void write_piece(const PagedPool &rows, const PagedPool &exps, int page, int at, int g, int c8, const Piece<T> &p) {
    char *row = rows.head(g) + rows.at(page, at);
    if constexpr (E4M3) {
        float x[8];
        numbers_of(p, x);
        const int s = row_exponent(x);
        *reinterpret_cast<uint2 *>(row + c8) = e4m3_codes(x, s);
        if (c8 == 0) *(exps.head(g) + exps.at(page, at)) = (char)(s + kExpBias);
    } else {
#pragma unroll
        for (int i = 0; i < (int)(sizeof(T) / 2); ++i) reinterpret_cast<u32x4 *>(row + c8 * sizeof(T))[i] = p.u[i];
    }
}

// Rows (token, KV head) of a batch row, the KV head fastest: the model's keys and values have a token's heads side by side.  The rows are under
// way while their page is looked up.  One row to a lane: with two, 8 x 4096 tokens of 8 KV heads took 27.9 us and not 26.2 (134 MB moved).
template <typename T, bool E4M3>
__global__ __launch_bounds__(256) void paged_write_kernel(const PagedArgs a) {
    const int b = a.by_blocks.quotient(blockIdx.x), row = (blockIdx.x - b * a.blocks) * 32 + (threadIdx.x >> 3), c8 = (threadIdx.x & 7) * 8;
    const int n = a.seqlens ? min(a.seqlens[b], a.Sq) : a.Sq;
    const int i = a.by_g.quotient(row), g = row - i * a.G;
    if (i >= n) return;                                              // (all eight lanes of the row)
    const Piece<T> k = load_piece(reinterpret_cast<const T *>(a.k) + b * a.ks.b + g * a.ks.h + i * a.ks.s + c8);
    const Piece<T> v = load_piece(reinterpret_cast<const T *>(a.v) + b * a.vs.b + g * a.vs.h + i * a.vs.s + c8);
    const int64_t pos = (int64_t)a.start[b] + i;
    const int page = pos < 0 || pos > 0x7fffffff ? -1 : paged_page(a, b, (int)pos);
    if (page < 0) return;
    const int at = (int)pos & ((1 << a.page_shift) - 1);
    write_piece<T, E4M3>(a.kp, a.ke, page, at, g, c8, k);
    write_piece<T, E4M3>(a.vp, a.ve, page, at, g, c8, v);
}

// Rows of a (batch row, KV head), which lie side by side in the result; one to a lane (two: eight prompts of up to 12000 tokens in e4m3, and their
// last chunks written, 58 us and not 52).  The result is streamed past the caches' retention (the same 56.7 us without that), as are rows of whole
// cache lines on their way in (16000 tokens of eight rows in bfloat16 106 us with neither, 97 with the first, 90 with both; codes 46 and 56).
template <typename T, typename ST>
__global__ __launch_bounds__(256) void paged_read_kernel(const PagedArgs a) {
    const int bg = a.by_blocks.quotient(blockIdx.x), i = (blockIdx.x - bg * a.blocks) * 32 + (threadIdx.x >> 3), c8 = (threadIdx.x & 7) * 8;
    const int b = a.by_g.quotient(bg), g = bg - b * a.G;
    if (i >= a.Sq) return;
    const int64_t pos = (a.start ? (int64_t)a.start[b] : 0) + i;
    const int page = pos >= 0 && pos < paged_length(a, b) ? paged_page(a, b, (int)pos) : -1;
    float k[8], v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) k[e] = v[e] = 0.0f;
    if (page >= 0) {
        const int at = (int)pos & ((1 << a.page_shift) - 1);
        load8<true>(reinterpret_cast<const ST *>(a.kp.head(g) + a.kp.at(page, at)) + c8, k);
        load8<true>(reinterpret_cast<const ST *>(a.vp.head(g) + a.vp.at(page, at)) + c8, v);
        if constexpr (sizeof(ST) == 1) {
            const float ke = factor_of_byte(*reinterpret_cast<const uint8_t *>(a.ke.head(g) + a.ke.at(page, at)));
            const float ve = factor_of_byte(*reinterpret_cast<const uint8_t *>(a.ve.head(g) + a.ve.at(page, at)));
#pragma unroll
            for (int e = 0; e < 8; ++e) { k[e] *= ke; v[e] *= ve; }
        }
    }
    store8<true>(reinterpret_cast<T *>(a.k) + b * a.ks.b + g * a.ks.h + i * a.ks.s + c8, k);
    store8<true>(reinterpret_cast<T *>(a.v) + b * a.vs.b + g * a.vs.h + i * a.vs.s + c8, v);
}

}  // namespace gptoss
