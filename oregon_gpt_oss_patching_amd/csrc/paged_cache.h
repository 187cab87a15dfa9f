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

// The power of two of 32 numbers (over the four lanes that hold them): the smallest 2^s with the largest at most 7 * 2^s, which is where rounding to the format's next
// number, 8, would begin; s = 128, the byte that means NaN, where one of them is not finite.
__device__ __forceinline__ int block_exponent(const float (&x)[8]) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);      // magnitudes compare as their bits do
    top = max(top, (uint32_t)__shfl_xor((int)top, 1));
    top = max(top, (uint32_t)__shfl_xor((int)top, 2));
    if (top >= 0x7f800000u) return 128;
    // 7 = 1.75 * 2^2 (numbers below 2^-126: as in row_exponent)
    return min(max((int)(top >> 23) - 127 - 2 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0), kMinExp), kMaxExp4);
}

__device__ __forceinline__ uint32_t e2m1_codes(const float (&x)[8], int s) {
    const float inv = exp_of_byte((uint32_t)(kExpBias - min(s, kMaxExp4)));      // 2^-s: as in e4m3_codes
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = __builtin_amdgcn_fmed3f(x[i] * inv, -6.0f, 6.0f);
    uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, y[0], y[1], 1.0f, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[2], y[3], 1.0f, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[4], y[5], 1.0f, 2);
    return s == 128 ? 0u : __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[6], y[7], 1.0f, 3);
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

template <typename T, typename ST>
__device__ __forceinline__ void write_piece(const PagedPool &rows, const PagedPool &exps, int page, int at, int g, int c8, const Piece<T> &p) {
    char *row = rows.head(g) + rows.at(page, at);
    if constexpr (is_e2m1<ST>) {
        float x[8];
        numbers_of(p, x);
        const int s = block_exponent(x);
        *reinterpret_cast<uint32_t *>(row + (c8 >> 1)) = e2m1_codes(x, s);
        if ((c8 & 31) == 0) *(exps.head(g) + exps.at(page, at) + (c8 >> 5)) = (char)(s + kExpBias);
    } else if constexpr (sizeof(ST) == 1) {
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

// Which 32 rows a workgroup writes.  Workgroups go to the eight XCDs in turn; of 4-bit rows each XCD has a run, so that its L2 has whole lines of them and of their exponents to write back (the grid is a multiple of
// eight).  us, in the order of the workgroups / so: 8 x 4096 tokens of 8 KV heads 24.1 / 22.4, 4 x 3001 9.8 / 9.5, by slots 7666 tokens 7.0 / 6.6, 30000 20.6 / 20.3; but in e4m3 8 x 4096 27.3 / 27.8, in bfloat16 27.9 / 28.8.
template <typename ST>
__device__ __forceinline__ int write_group() {
    return is_e2m1<ST> ? (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3) : blockIdx.x;
}

// Rows (token, KV head) of a batch row, the KV head fastest: the model's keys and values have a token's heads side by side.  The rows are under
// way while their page is looked up.  One row to a lane: with two, 8 x 4096 tokens of 8 KV heads took 27.9 us and not 26.2 (134 MB moved).
template <typename T, typename ST>
__global__ __launch_bounds__(256) void paged_write_kernel(const PagedArgs a) {
    const int wg = write_group<ST>(), b = a.by_blocks.quotient(wg), row = (wg - b * a.blocks) * 32 + (threadIdx.x >> 3), c8 = (threadIdx.x & 7) * 8;
    if (is_e2m1<ST> && b >= a.B) return;
    const int n = a.seqlens ? min(a.seqlens[b], a.Sq) : a.Sq;
    const int i = a.by_g.quotient(row), g = row - i * a.G;
    if (i >= n) return;                                              // (all eight lanes of the row)
    const Piece<T> k = load_piece(reinterpret_cast<const T *>(a.k) + b * a.ks.b + g * a.ks.h + i * a.ks.s + c8);
    const Piece<T> v = load_piece(reinterpret_cast<const T *>(a.v) + b * a.vs.b + g * a.vs.h + i * a.vs.s + c8);
    const int64_t pos = (int64_t)a.start[b] + i;
    const int page = pos < 0 || pos > 0x7fffffff ? -1 : paged_page(a, b, (int)pos);
    if (page < 0) return;
    const int at = (int)pos & ((1 << a.page_shift) - 1);
    write_piece<T, ST>(a.kp, a.ke, page, at, g, c8, k);
    write_piece<T, ST>(a.vp, a.ve, page, at, g, c8, v);
}

// The same of one batch row whose tokens have slots of their own.
template <typename T, typename ST>
__global__ __launch_bounds__(256) void paged_write_slots_kernel(const PagedArgs a, const int64_t *slots) {
    const int row = write_group<ST>() * 32 + (threadIdx.x >> 3), c8 = (threadIdx.x & 7) * 8;
    const int i = a.by_g.quotient(row), g = row - i * a.G;
    if (i >= a.Sq) return;                                           // (all eight lanes of the row)
    const Piece<T> k = load_piece(reinterpret_cast<const T *>(a.k) + g * a.ks.h + i * a.ks.s + c8);
    const Piece<T> v = load_piece(reinterpret_cast<const T *>(a.v) + g * a.vs.h + i * a.vs.s + c8);
    const int64_t slot = slots[i], page = slot >> a.page_shift;
    if (slot < 0 || page >= a.pages) return;
    const int at = (int)slot & ((1 << a.page_shift) - 1);
    write_piece<T, ST>(a.kp, a.ke, (int)page, at, g, c8, k);
    write_piece<T, ST>(a.vp, a.ve, (int)page, at, g, c8, v);
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
        load8<true>(reinterpret_cast<const ST *>(a.kp.head(g) + a.kp.at(page, at)), c8, k);
        load8<true>(reinterpret_cast<const ST *>(a.vp.head(g) + a.vp.at(page, at)), c8, v);
        if constexpr (sizeof(ST) == 1) {
            const int half = is_e2m1<ST> ? c8 >> 5 : 0;              // which of a row's bytes
            const float ke = factor_of_byte(*reinterpret_cast<const uint8_t *>(a.ke.head(g) + a.ke.at(page, at) + half));
            const float ve = factor_of_byte(*reinterpret_cast<const uint8_t *>(a.ve.head(g) + a.ve.at(page, at) + half));
#pragma unroll
            for (int e = 0; e < 8; ++e) { k[e] *= ke; v[e] *= ve; }
        }
    }
    store8<true>(reinterpret_cast<T *>(a.k) + b * a.ks.b + g * a.ks.h + i * a.ks.s + c8, k);
    store8<true>(reinterpret_cast<T *>(a.v) + b * a.vs.b + g * a.vs.h + i * a.vs.s + c8, v);
}

}  // namespace gptoss
