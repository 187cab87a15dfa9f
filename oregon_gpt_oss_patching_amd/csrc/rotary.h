// Rotary positions (gptoss_attn_rotary): pairs (x1, x2) of a head's first R numbers turned by their token's angle,
//   y1 = c x1 - s x2,  y2 = c x2 + s x1,  c = scale cos(p f_i), s = scale sin(p f_i),
// and the other way round (-s) for gradients; the other D - R numbers go through as they are.
//
// What bounds it: moving q and k once in and once out; a decoding step's call, one launch.  A thread has V pairs of a token and walks some of its
// heads, so that the angles, which all heads share, cost little: V pairs are one or two 16-byte accesses each way.
// Results are stored so that caches keep them: the attention reads them next (past the caches' retention 2 x 4096 tokens take 33.6 us and not 34.4, with the attention over a window of 128 behind it
// 79.2 and not 72.9).
#pragma once
#include "paged_common.h"

namespace gptoss {

// Threads of a workgroup, which share nothing: one wavefront each (with four 32 x 1 token 3.35 us and not 3.13, and inputs that no cache holds: 1000 tokens 8.1 / 7.8, 4096 21.2 / 20.4, 2 x 4096
// 35.2 / 33.9, 16384 62.0 / 62.4).
constexpr int kRotaryThreads = 64;

struct RotaryArgs {
    const void *q, *k;
    void *q_out, *k_out;
    const void *positions;               // int32 or int64 (wide)
    const double *frequencies;
    const void *cos, *sin;               // instead of the two above
    Strides qs, ks, qo, ko;              // elements
    int64_t pos_b, pos_s, cos_b, cos_s, sin_b, sin_s;
    int64_t items;                       // threads with work: (token, slot, chunk), chunks fastest
    int H, heads, D, R, pairs, chunks;   // heads: H + G; pairs: chunks that are turned, the others are copied
    int slots;                           // threads that share a token's heads
    int inner;                           // what runs behind the chunks: the slots of a token, or (along_tokens) the tokens of a slot
    Div by_chunks, by_inner, by_s;
    int S;
    float scale;                         // of the angles' cosine and sine; of tables 1
    bool wide, f32_tables, whole_tables, inverse, along_tokens;
};

// c = cos(u pi / 2), s = sin(u pi / 2).  The whole quarters come off in 64 bits, what is left is at most half of one: polynomials (the Taylor series, whose
// first term left out is below 2^-29 there) in 32 bits.  Off by at most 4 * 2^-24: the argument's rounding, the leading constant's and the last
// multiplication's and addition's.  u itself, a position times (a frequency times 2 / pi), has been rounded three times in 64 bits: the angle is off by up to 3 * 2^-53 of itself, which
// is 2^-24 more at 2^27 radians and grows with them (and positions beyond 2^53 are not held exactly).
__device__ __forceinline__ void quarter_turns(double u, float &c, float &s) {
    const double n = __builtin_rint(u);
    const float f = (float)(u - n), f2 = f * f;
    const int quarter = (int)(n - 4.0 * __builtin_floor(n * 0.25));
    // (pi/2)^i / i!
    const float sn = f * fmaf(f2, fmaf(f2, fmaf(f2, fmaf(f2, 1.6044118e-4f, -4.6817541e-3f), 7.9692626e-2f), -6.4596410e-1f), 1.5707963e+0f);
    const float cn = fmaf(f2, fmaf(f2, fmaf(f2, fmaf(f2, fmaf(f2, -2.5202042e-5f, 9.1926030e-4f), -2.0863481e-2f), 2.5366951e-1f), -1.2337005e+0f), 1.0f);
    const float a = quarter & 1 ? sn : cn, b = quarter & 1 ? cn : sn;
    c = quarter == 1 || quarter == 2 ? -a : a;
    s = quarter >= 2 ? -b : b;
}

// V numbers as they lie in memory, in 4, 8 or 16 bytes (V = 1: as they are).
template <typename T, int V> struct RotaryPiece;
template <typename T> struct RotaryPiece<T, 1> {
    T x;
    __device__ __forceinline__ float get(int) const { return (float)x; }
    __device__ __forceinline__ void set(int, float v) { x = (T)v; }
};
template <int V> struct RotaryPiece<float, V> {
    typedef __attribute__((ext_vector_type(V))) float vec;
    vec x;
    __device__ __forceinline__ float get(int i) const { return x[i]; }
    __device__ __forceinline__ void set(int i, float v) { x[i] = v; }
};
template <int V> struct RotaryPiece<bf16, V> {
    typedef __attribute__((ext_vector_type(V))) __bf16 vec;
    vec x;
    __device__ __forceinline__ float get(int i) const { return (float)x[i]; }
    __device__ __forceinline__ void set(int i, float v) { x[i] = (bf16)v; }
};
template <> struct RotaryPiece<float, 1> {
    float x;
    __device__ __forceinline__ float get(int) const { return x; }
    __device__ __forceinline__ void set(int, float v) { x = v; }
};
template <> struct RotaryPiece<bf16, 1> {
    bf16 x;
    __device__ __forceinline__ float get(int) const { return (float)x; }
    __device__ __forceinline__ void set(int, float v) { x = (bf16)v; }
};

// V numbers of a table row of either type; `whole`: its pieces of V lie on boundaries of their own size (of 16 bytes at most).
template <int V>
__device__ __forceinline__ void table_numbers(const void *p, int64_t at, bool f32, bool whole, float (&x)[V]) {
    if constexpr (V > 1) {
        if (whole) {
            if (f32) {
                constexpr int n = V < 4 ? V : 4;
#pragma unroll
                for (int i = 0; i < V; i += n) {
                    const auto y = *reinterpret_cast<const RotaryPiece<float, n> *>(static_cast<const float *>(p) + at + i);
#pragma unroll
                    for (int e = 0; e < n; ++e) x[i + e] = y.get(e);
                }
            } else {
                const auto y = *reinterpret_cast<const RotaryPiece<bf16, V> *>(static_cast<const bf16 *>(p) + at);
#pragma unroll
                for (int e = 0; e < V; ++e) x[e] = y.get(e);
            }
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = f32 ? static_cast<const float *>(p)[at + i] : (float)static_cast<const bf16 *>(p)[at + i];
}

// PAIRED: numbers 2i and 2i + 1 are a pair, otherwise i and i + R/2.
template <typename T, int V, bool PAIRED, bool TABLES>
__global__ __launch_bounds__(kRotaryThreads) void rotary_kernel(const RotaryArgs a) {
    using Piece = RotaryPiece<T, V>;
    constexpr int kAtOnce = 4;           // heads whose numbers are under way together
    const int64_t item = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (item >= a.items) return;
    const int line = a.by_chunks.quotient((int)item), chunk = (int)item - line * a.chunks;
    const int quotient = a.by_inner.quotient(line), inner = line - quotient * a.inner;
    const int token = a.along_tokens ? inner : quotient, slot = a.along_tokens ? quotient : inner;
    const int b = a.by_s.quotient(token), s = token - b * a.S;
    const bool turned = chunk < a.pairs;
    // the two pieces of a head's row (of what is copied: one)
    const int at0 = turned ? (PAIRED ? 2 * V * chunk : V * chunk) : a.R + V * (chunk - a.pairs);
    const int at1 = turned ? (PAIRED ? at0 + V : at0 + a.R / 2) : at0;
    const T *q = static_cast<const T *>(a.q) + b * a.qs.b + s * a.qs.s, *k = static_cast<const T *>(a.k) + b * a.ks.b + s * a.ks.s;
    T *qo = static_cast<T *>(a.q_out) + b * a.qo.b + s * a.qo.s, *ko = static_cast<T *>(a.k_out) + b * a.ko.b + s * a.ko.s;
    Piece x0[kAtOnce], x1[kAtOnce];
    auto load = [&](int h0) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            // (behind the last head that one once more)
            const int h = min(h0 + i * a.slots, a.heads - 1);
            const T *row = h < a.H ? q + h * a.qs.h : k + (h - a.H) * a.ks.h;
            x0[i] = *reinterpret_cast<const Piece *>(row + at0);
            x1[i] = *reinterpret_cast<const Piece *>(row + at1);
        }
    };
    load(slot);
    float c[V], sn[V];
    if (turned) {
        if constexpr (TABLES) {
            table_numbers<V>(a.cos, b * a.cos_b + s * a.cos_s + V * chunk, a.f32_tables, a.whole_tables, c);
            table_numbers<V>(a.sin, b * a.sin_b + s * a.sin_s + V * chunk, a.f32_tables, a.whole_tables, sn);
        } else {
            const int64_t at = b * a.pos_b + s * a.pos_s;
            const double p = a.wide ? (double)static_cast<const int64_t *>(a.positions)[at] : (double)static_cast<const int32_t *>(a.positions)[at];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                quarter_turns(p * (a.frequencies[V * chunk + i] * 0.63661977236758134308), c[i], sn[i]);
                c[i] *= a.scale;
                sn[i] *= a.scale;
            }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) sn[i] = a.inverse ? -sn[i] : sn[i];
    }
    for (int h0 = slot;;) {
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const int h = h0 + i * a.slots;
            if (h >= a.heads) break;
            T *row = h < a.H ? qo + h * a.qo.h : ko + (h - a.H) * a.ko.h;
            Piece y0 = x0[i], y1 = x1[i];
            if (turned) {
                // pair j of the piece: PAIRED: its numbers 2j, 2j + 1, over both pieces
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const Piece &p0 = PAIRED && 2 * j >= V ? x1[i] : x0[i], &p1 = !PAIRED || 2 * j >= V || V == 1 ? x1[i] : x0[i];
                    const int i0 = PAIRED ? 2 * j % V : j, i1 = PAIRED ? (2 * j + 1) % V : j;
                    const float u = p0.get(i0), w = p1.get(i1);
                    const float yu = fmaf(u, c[j], -(w * sn[j])), yw = fmaf(w, c[j], u * sn[j]);
                    if (PAIRED && 2 * j >= V) y1.set(i0, yu);
                    else y0.set(i0, yu);
                    if (!PAIRED || 2 * j >= V || V == 1) y1.set(i1, yw);
                    else y0.set(i1, yw);
                }
                *reinterpret_cast<Piece *>(row + at1) = y1;
            }
            *reinterpret_cast<Piece *>(row + at0) = y0;
        }
        h0 += kAtOnce * a.slots;
        if (h0 >= a.heads) break;
        load(h0);
    }
}

}  // namespace gptoss
