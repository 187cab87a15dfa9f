// A key / value cache in pages: what its kernels share (the arguments, the page of a token, rows of 64 as they are stored).
//
// A stored row is 64 numbers of the model's type, or 64 e4m3 codes and a byte e: the row is code * 2^(e - 127).  A power of two
// makes both directions exact but for the one rounding to e4m3: codes widen to bf16 (four significant bits), and so do their
// products with 2^s.  A divisor of largest / 448, which fills the format's range, would save at most one bit in the numbers below
// 2^-15 of the row's largest, and cost a rounding in each direction.
#pragma once
#include "attn_common.h"

namespace gptoss {

// Quotients of numbers below 2^31 by a number that the host knows: one multiplication.  With s = ceil(log2 d) and mul = ceil(2^(31 + s) / d) the
// product is too large by less than x * 2^s / d, which is less than 2^(31 + s) / d: never by a whole quotient.
struct Div {
    uint32_t mul, shift;
    __host__ __device__ __forceinline__ int quotient(int x) const { return (int)(((uint64_t)(uint32_t)x * mul) >> shift); }
};
inline Div div_by(int64_t d) {
    uint32_t s = 0;
    while (((int64_t)1 << s) < d) ++s;
    return Div{(uint32_t)((((uint64_t)1 << (31 + s)) + (uint64_t)d - 1) / (uint64_t)d), 31 + s};
}

// A pool of pages: strides in bytes, of pages and tokens below 2^32.
struct PagedPool {
    char *base;
    int64_t h;
    uint32_t b, s;
    __device__ __forceinline__ char *head(int g) const { return base + g * h; }
    __device__ __forceinline__ int64_t at(int page, int slot) const { return (int64_t)((uint64_t)(uint32_t)page * b + (uint64_t)(uint32_t)slot * s); }
};

struct PagedArgs {
    const void *q, *sinks;
    void *o;
    float *lse;
    PagedPool kp, vp;            // rows in bytes
    PagedPool ke, ve;            // their exponents
    const int32_t *table, *seqlens, *start;
    char *k, *v;                 // rows to write, or the result of reading
    Strides qs, os, ks, vs;      // elements
    int64_t table_stride;
    int B, H, G, r, Sq;
    int pages, page_shift, width, window;
    int blocks;                  // workgroups of a batch row (write), of a row and KV head (read); blocks of pairs of a row (attention)
    // attention: (row, block of pairs) units, into how many shares their work is cut (0: not), of how many tiles at least; the shares'
    // partial results and, for each unit, its first share and their number
    int units, shares;
    bool across;                 // eight slots of workgroups next to each other, not the heads of one
    Div by_r, by_g, by_blocks, by_wgs;          // by r, G, blocks, and a row and KV head's workgroups of the sum over shares
    float *partial;
    int *plan;
    float scale_log2;
    bool sinks_bf16;
};

constexpr int kExpBias = 127, kMinExp = -64, kMaxExp = 120;       // exponent bytes; the powers of two of rows
constexpr float kLowest = -3.0e38f;                // start of a running maximum: finite, so that -inf - (it) is -inf and not NaN

__device__ __forceinline__ float paged_sink(const PagedArgs &a, int head) {
    if (!a.sinks) return 0.0f;
    return a.sinks_bf16 ? (float)static_cast<const bf16 *>(a.sinks)[head] : static_cast<const float *>(a.sinks)[head];
}

// Page of token t of a row, -1 where there is none (t outside the table, an entry outside the pool).
__device__ __forceinline__ int paged_page(const PagedArgs &a, int b, int t) {
    if (t < 0 || (t >> a.page_shift) >= a.width) return -1;
    const int page = a.table[(int64_t)b * a.table_stride + (t >> a.page_shift)];
    return (unsigned)page < (unsigned)a.pages ? page : -1;
}

// Tokens of a row in the cache.
__device__ __forceinline__ int paged_length(const PagedArgs &a, int b) {
    return min(max(a.seqlens[b], 0), a.width << a.page_shift);
}

__device__ __forceinline__ float exp_of_byte(uint32_t e) { return __uint_as_float(e << 23); }        // 2^(e - 127), 1 <= e <= 254

// 2^(e - 127) as a factor of any byte e, NaN for 255: what the scaling conversions take exp_of_byte(e) for.  (2^-127 is half of 32 bits' smallest normal number.)
__device__ __forceinline__ float factor_of_byte(uint32_t e) { return __uint_as_float(e == 0 ? 0x00400000u : e == 255 ? 0x7fc00000u : e << 23); }

struct e4m3 { uint8_t code; };

// A number of a row (of a code: without its power of two).
__device__ __forceinline__ float stored_number(const bf16 *p) { return (float)*p; }
__device__ __forceinline__ float stored_number(const float *p) { return *p; }
__device__ __forceinline__ float stored_number(const e4m3 *p) { return __builtin_amdgcn_cvt_f32_fp8((int)p->code, 0); }

// 16 bytes; ONCE: past the caches' retention, for what a kernel streams through.
template <bool ONCE>
__device__ __forceinline__ u32x4 load16(const void *p) {
    if constexpr (ONCE) return __builtin_nontemporal_load(static_cast<const u32x4 *>(p));
    else return *static_cast<const u32x4 *>(p);
}
template <bool ONCE>
__device__ __forceinline__ void store16(void *p, const u32x4 x) {
    if constexpr (ONCE) __builtin_nontemporal_store(x, static_cast<u32x4 *>(p));
    else *static_cast<u32x4 *>(p) = x;
}

// Eight numbers of a row.
template <bool ONCE = false>
__device__ __forceinline__ void load8(const bf16 *p, float (&x)[8]) {
    const bf16x8 v = as_bf16x8(load16<ONCE>(p));
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)v[i];
}
template <bool ONCE = false>
__device__ __forceinline__ void load8(const float *p, float (&x)[8]) {
    const u32x4 u = load16<ONCE>(p), w = load16<ONCE>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[i] = __uint_as_float(u[i]); x[4 + i] = __uint_as_float(w[i]); }
}
template <bool ONCE = false>
__device__ __forceinline__ void load8(const e4m3 *p, float (&x)[8]) {
    const uint2 w = *reinterpret_cast<const uint2 *>(p);
    x[0] = __builtin_amdgcn_cvt_f32_fp8((int)w.x, 0);
    x[1] = __builtin_amdgcn_cvt_f32_fp8((int)w.x, 1);
    x[2] = __builtin_amdgcn_cvt_f32_fp8((int)w.x, 2);
    x[3] = __builtin_amdgcn_cvt_f32_fp8((int)w.x, 3);
    x[4] = __builtin_amdgcn_cvt_f32_fp8((int)w.y, 0);
    x[5] = __builtin_amdgcn_cvt_f32_fp8((int)w.y, 1);
    x[6] = __builtin_amdgcn_cvt_f32_fp8((int)w.y, 2);
    x[7] = __builtin_amdgcn_cvt_f32_fp8((int)w.y, 3);
}
template <bool ONCE = false>
__device__ __forceinline__ void store8(bf16 *p, const float (&x)[8]) {
    union { bf16x8 v; u32x4 u; } out;
#pragma unroll
    for (int i = 0; i < 8; ++i) out.v[i] = (bf16)x[i];
    store16<ONCE>(p, out.u);
}
template <bool ONCE = false>
__device__ __forceinline__ void store8(float *p, const float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i += 4) store16<ONCE>(p + i, u32x4{__float_as_uint(x[i]), __float_as_uint(x[i + 1]), __float_as_uint(x[i + 2]), __float_as_uint(x[i + 3])});
}

}  // namespace gptoss
