// Attention of new queries over a key / value cache in pages (gptoss_attn_paged_fwd).
//
// What bounds it: reading the rows that the queries see once from HBM, or, for short rows, the latency of a launch or two.
//
// Work.  The Sq * r (query, head of the group) pairs of a KV head are the columns of S^T, up to 16 NB of them to a workgroup (a unit), so that
// K and V are read once.  The host does not see the lengths: a fixed number of workgroups finds, from all lengths, how long equal shares of
// all units' 32-key tiles are and which share is its own (PagedShare); a unit with one share writes its results, the others leave fp32
// partials that attn_paged_combine_kernel adds in the order of the shares.  So one long row among many short ones is spread over the chip,
// and a table that is wider than the rows costs nothing.
//
// In a workgroup four wavefronts take tiles in turn, each for itself (no barrier in the loop), and merge their (m, l, O) at the end.
//  * K goes from the pages straight into the MFMA's A operand: a lane holds pieces of one key's row, and which number of the row stands in
//    which slot of the contraction is free as long as Q has the same order.
//  * V has to be turned (the contraction runs over keys): bf16 rows go through a stage of LDS and are read back transposed; in 32 bits each
//    lane loads four columns of its own four keys, which is what the fp32 MFMA takes.
//  * P leaves the S product in the layout of the PV product's B operand.
//  * Entries of the page table are loaded 64 tiles at a time, one per lane; a tile's page is a readlane and its addresses are scalar.
//  * e4m3 rows widen on the way into the operand: to bf16 by the instruction that takes a power of two along (exact), K's with one
//    power per lane, V's before they are staged.
// The running maximum is raised only when a logit passes it by more than 2^8 (the sums are in 32 bits and the weights keep their relative
// precision): the reduction over the lanes and the rescaling are then rare.
#pragma once
#include <type_traits>

#include "paged_common.h"

namespace gptoss {

constexpr int kPagedKeys = 32, kPagedWaves = 4, kPagedMaxUnits = 1024;
constexpr int kPagedRow = kD + 2;               // floats of a merged row: O, m, l
constexpr float kRaise = 8.0f;                  // in the exponent of two

// Pairs (query, head of the group) that one workgroup may take.
template <typename T> __host__ __device__ constexpr int paged_pairs() { return sizeof(T) == 2 ? 64 : 32; }
// floats of a share's partial result: rows of O, then (m, l) of each
__host__ __device__ constexpr int64_t paged_partial_floats(int nb) { return (int64_t)16 * nb * kPagedRow; }

// The queries of a unit (a row's block of pairs) and the keys that they see.
struct PagedSpan {
    int b, pair0, n, base;       // batch row, first pair, tokens in the cache, position of the row's query 0
    int pos0, pos1;              // first and last position of queries that exist
    int lo, hi, t_first, tiles;  // keys lo .. hi - 1, in tiles
};
__device__ __forceinline__ PagedSpan paged_span(const PagedArgs &a, int unit, int pairs) {
    PagedSpan s;
    s.b = unit / a.blocks;
    s.pair0 = (unit - s.b * a.blocks) * pairs;
    s.n = paged_length(a, s.b);
    // (positions beyond +-2^30 exist in no row)
    s.base = a.start ? min(max(a.start[s.b], -(1 << 30)), (1 << 30) - 1) : s.n - a.Sq;
    const int i0 = s.pair0 / a.r, i1 = min(a.Sq - 1, (s.pair0 + pairs - 1) / a.r);
    s.pos0 = max(s.base + i0, 0);
    s.pos1 = min(s.base + i1, s.n - 1);
    const bool any = s.pos0 <= s.pos1;
    s.lo = any && a.window ? max(0, s.pos0 - a.window + 1) : 0;
    s.hi = any ? s.pos1 + 1 : 0;
    s.t_first = s.lo / kPagedKeys;
    s.tiles = any ? (s.hi + kPagedKeys - 1) / kPagedKeys - s.t_first : 0;
    return s;
}

// Which share of which unit a workgroup takes.  All units' tiles are cut into shares of `chunk`, the smallest length of at least
// a.min_tiles with which they number no more than a.shares and one for each unit, which is what the grid and the scratch hold.
struct PagedShare { int unit, index, count, first; };     // first: number of the unit's first share; unit < 0: nothing left
__device__ __forceinline__ PagedShare paged_share(const PagedArgs &a, int slot, int pairs) {
    if (!a.shares) return PagedShare{slot, 0, 1, slot};
    const int lane = threadIdx.x & 63;
    int64_t all = 0;
    if (a.units <= 64) {
        uint32_t x = lane < a.units ? (uint32_t)paged_span(a, lane, pairs).tiles : 0u;      // at most 2^25 each
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) x += (uint32_t)__shfl_xor((int)x, d);
        all = x;
    } else {
        for (int u = lane; u < a.units; u += 64) all += paged_span(a, u, pairs).tiles;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) all += __shfl_xor((long long)all, d);
    }
    const int64_t even = (all + a.shares - 1) / a.shares;
    const int chunk = max(a.min_tiles, (int)(even < (1 << 30) ? even : (1 << 30)));      // (more tiles than a unit can have)
    int before = 0;
    for (int u0 = 0; u0 < a.units; u0 += 64) {
        const int u = u0 + lane;
        const int mine = u < a.units ? max(1, (paged_span(a, u, pairs).tiles + chunk - 1) / chunk) : 0;
        int incl = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int y = __shfl_up(incl, d);
            if (lane >= d) incl += y;
        }
        const int first = before + incl - mine;
        const unsigned long long who = __builtin_amdgcn_ballot_w64(slot >= first && slot < first + mine);
        if (who) {
            const int l = __builtin_ctzll(who);
            const int f = __builtin_amdgcn_readlane(first, l);
            return PagedShare{u0 + l, slot - f, __builtin_amdgcn_readlane(mine, l), f};
        }
        before += __builtin_amdgcn_readlane(incl, 63);
    }
    return PagedShare{-1, 0, 0, 0};
}

// max / sum over the four lanes that hold a column (lane ^ 16, lane ^ 32)
__device__ __forceinline__ float quad_max(float x) {
    typedef __attribute__((ext_vector_type(2))) unsigned u32x2_t;
    const unsigned u = __float_as_uint(x);
    const u32x2_t r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const unsigned p = r.x, q = r.y;
    return xhalf_max(fast_max(__uint_as_float(p), __uint_as_float(q)));
}
__device__ __forceinline__ float quad_sum(float x) {
    typedef __attribute__((ext_vector_type(2))) unsigned u32x2_t;
    const unsigned u = __float_as_uint(x);
    const u32x2_t r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const unsigned p = r.x, q = r.y;
    return xhalf_sum(__uint_as_float(p) + __uint_as_float(q));
}

typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;

// Eight codes as bf16 numbers times the power of two `f`: exact (four significant bits).
__device__ __forceinline__ bf16x8 widen8(uint32_t w0, uint32_t w1, float f) {
    union { bf16x2 p[4]; bf16x8 v; } x;
    x.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, f, false);
    x.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, f, true);
    x.p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, f, false);
    x.p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, f, true);
    return x.v;
}

// A tile's K and V as they are loaded, and what is done with them.  `kb` / `vb`: scalar addresses of the first row of a block of 16 keys;
// lanes: l16 = lane % 16, quad = lane / 16.
template <typename T, typename ST, int NB> struct PagedTile;

// ---- bfloat16 products -----------------------------------------------------------------------------------------------
template <typename ST, int NB>
struct PagedTile<bf16, ST, NB> {
    static constexpr bool kCodes = sizeof(ST) == 1;
    static constexpr int kStage = kPagedKeys * kRowBytes;        // LDS bytes of a wavefront
    static constexpr int kVecs = kCodes ? 1 : 2;                 // 16-byte loads per lane and block
    u32x4 k[2][kVecs], v[2][kVecs];
    uint32_t ke[2], ve[2];
    bf16x8 q[NB][2];
    f32x4 o[NB][4];
    uint32_t tr[4], wr[2];

    __device__ __forceinline__ static int v_row(int lane, int i) { return kCodes ? lane >> 2 : (lane >> 3) + 8 * i; }

    __device__ __forceinline__ void init(uint32_t stage, int lane) {
        const int i = lane & 15, row = 4 * (lane >> 4) + (i >> 2);
#pragma unroll
        for (int d = 0; d < 4; ++d) tr[d] = stage + row * kRowBytes + (((2 * d + ((i & 3) >> 1)) ^ swz(row)) * 16) + (i & 1) * 8;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = v_row(lane, e), c = kCodes ? 2 * (lane & 3) + e : lane & 7;
            wr[e] = stage + r * kRowBytes + ((c ^ swz(r)) * 16);
        }
    }
    __device__ __forceinline__ void load_q(int nb, const bf16 *row, bool there, int quad) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const u32x4 x = *reinterpret_cast<const u32x4 *>(row + (kCodes ? 16 * quad + 8 * s : 32 * s + 8 * quad));
            q[nb][s] = as_bf16x8(there ? x : u32x4{0, 0, 0, 0});
        }
#pragma unroll
        for (int d = 0; d < 4; ++d) o[nb][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    __device__ __forceinline__ void load_k(int blk, const char *kb, const uint8_t *eb, const PagedArgs &a, int lane) {
        const int l16 = lane & 15, quad = lane >> 4;
        const uint32_t at = (uint32_t)(l16 * (int)a.kps.s * (kCodes ? 1 : 2) + 16 * quad);
#pragma unroll
        for (int s = 0; s < kVecs; ++s) k[blk][s] = *reinterpret_cast<const u32x4 *>(kb + at + 64 * s);
        if constexpr (kCodes) ke[blk] = eb[(uint32_t)(l16 * (int)a.kes.s)];
    }
    __device__ __forceinline__ void load_v(int blk, const char *vb, const uint8_t *eb, const PagedArgs &a, int lane) {
#pragma unroll
        for (int i = 0; i < kVecs; ++i)
            v[blk][i] = *reinterpret_cast<const u32x4 *>(vb + (uint32_t)(v_row(lane, i) * (int)a.vps.s * (kCodes ? 1 : 2) + 16 * (kCodes ? lane & 3 : lane & 7)));
        if constexpr (kCodes) ve[blk] = eb[(uint32_t)(v_row(lane, 0) * (int)a.ves.s)];
    }
    __device__ __forceinline__ void logits(f32x4 (&s)[NB][2]) const {
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) {
            bf16x8 f[2];
            if constexpr (kCodes) {
                const float p = exp_of_byte(ke[blk]);
                f[0] = widen8(k[blk][0][0], k[blk][0][1], p);
                f[1] = widen8(k[blk][0][2], k[blk][0][3], p);
            } else {
                f[0] = as_bf16x8(k[blk][0]);
                f[1] = as_bf16x8(k[blk][1]);
            }
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                const f32x4 z = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f[0], q[nb][0], f32x4{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
                s[nb][blk] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f[1], q[nb][1], z, 0, 0, 0);
            }
        }
    }
    // V into the stage; rows outside first .. last - 1 of the tile as zeros where `edge`, and whether a row inside holds no finite number
    __device__ __forceinline__ bool stage_v(bool edge, int first, int last, unsigned there, int lane) {
        bool odd = false;
#pragma unroll
        for (int blk = 0; blk < 2; ++blk)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                u32x4 x;
                if constexpr (kCodes) {
                    union { bf16x8 b; u32x4 u; } w;
                    w.b = widen8(v[blk][0][2 * i], v[blk][0][2 * i + 1], exp_of_byte(ve[blk]));
                    x = w.u;
                } else {
                    x = v[blk][i];
                }
                if (edge) {
                    const int r = 16 * blk + v_row(lane, i);
                    const bool in = r >= first && r < last && (there >> blk & 1);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x[e] = in ? x[e] : 0u;
                        odd = odd || (x[e] & 0x7f80u) == 0x7f80u || (x[e] & 0x7f800000u) == 0x7f800000u;
                    }
                }
                *reinterpret_cast<__attribute__((address_space(3))) u32x4 *>((uintptr_t)(wr[i] + 16 * blk * kRowBytes)) = x;
            }
        return odd;
    }
    __device__ __forceinline__ void product(const f32x4 (&s)[NB][2]) {
        bf16x8 p[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int e = 0; e < 4; ++e) { p[nb][e] = (bf16)s[nb][0][e]; p[nb][4 + e] = (bf16)s[nb][1][e]; }
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            union { struct { s16x4 a, b; } s; bf16x8 v; } x;
            x.s.a = lds_load_tr64(tr[d], 0);
            x.s.b = lds_load_tr64(tr[d], 16 * kRowBytes);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) o[nb][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.v, p[nb], o[nb][d], 0, 0, 0);
        }
    }
    // column of o[.][d][e] in the lane's row
    __device__ __forceinline__ static int column(int d, int e, int quad) { return 16 * d + 4 * quad + e; }
    // V of row `key` and that column, out of the stage
    __device__ __forceinline__ static float staged(uint32_t stage, int key, int col) {
        const uint32_t at = stage + key * kRowBytes + (((col >> 3) ^ swz(key)) * 16) + (col & 7) * 2;
        return (float)*reinterpret_cast<const __attribute__((address_space(3))) bf16 *>((uintptr_t)at);
    }
};

// ---- float32 products ------------------------------------------------------------------------------------------------
template <typename ST, int NB>
struct PagedTile<float, ST, NB> {
    static constexpr bool kCodes = sizeof(ST) == 1;
    static constexpr int kStage = kPagedKeys * kD * 4;           // used where V holds infinities or NaN only
    static constexpr int kVecs = kCodes ? 1 : 4;
    typedef typename std::conditional<kCodes, uint32_t, f32x4>::type vec;       // four numbers of a row of V
    u32x4 k[2][kVecs];
    vec v[2][4];
    uint32_t ke[2], ve[2][4];
    float q[NB][16];
    f32x4 o[NB][4];
    uint32_t stage;

    __device__ __forceinline__ void init(uint32_t stage_, int) { stage = stage_; }
    __device__ __forceinline__ static int q_index(int t, int quad) { return kCodes ? 16 * quad + t : 16 * (t >> 2) + 4 * quad + (t & 3); }
    __device__ __forceinline__ void load_q(int nb, const float *row, bool there, int quad) {
#pragma unroll
        for (int t = 0; t < 16; t += 4) {
            const f32x4 x = *reinterpret_cast<const f32x4 *>(row + q_index(t, quad));
#pragma unroll
            for (int e = 0; e < 4; ++e) q[nb][t + e] = there ? x[e] : 0.0f;
        }
#pragma unroll
        for (int d = 0; d < 4; ++d) o[nb][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    __device__ __forceinline__ void load_k(int blk, const char *kb, const uint8_t *eb, const PagedArgs &a, int lane) {
        const int l16 = lane & 15, quad = lane >> 4;
        const uint32_t at = (uint32_t)(l16 * (int)a.kps.s * (kCodes ? 1 : 4) + 16 * quad);
#pragma unroll
        for (int s = 0; s < kVecs; ++s) k[blk][s] = *reinterpret_cast<const u32x4 *>(kb + at + 64 * s);
        if constexpr (kCodes) ke[blk] = eb[(uint32_t)(l16 * (int)a.kes.s)];
    }
    __device__ __forceinline__ void load_v(int blk, const char *vb, const uint8_t *eb, const PagedArgs &a, int lane) {
        const int l16 = lane & 15, quad = lane >> 4;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[blk][e] = *reinterpret_cast<const vec *>(vb + (uint32_t)((4 * quad + e) * (int)a.vps.s * (kCodes ? 1 : 4) + (kCodes ? 4 : 16) * l16));
            if constexpr (kCodes) ve[blk][e] = eb[(uint32_t)((4 * quad + e) * (int)a.ves.s)];
        }
    }
    __device__ __forceinline__ void logits(f32x4 (&s)[NB][2]) const {
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) s[nb][blk] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            float p = 1.0f;
            if constexpr (kCodes) p = exp_of_byte(ke[blk]);
#pragma unroll
            for (int t = 0; t < 16; ++t) {
                float x;
                if constexpr (kCodes) x = p * code(k[blk][0][t >> 2], t & 3);
                else x = __uint_as_float(k[blk][t >> 2][t & 3]);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) s[nb][blk] = __builtin_amdgcn_mfma_f32_16x16x4f32(x, q[nb][t], s[nb][blk], 0, 0, 0);
            }
        }
    }
    __device__ __forceinline__ static float code(uint32_t w, int i) {
        return i == 0 ? __builtin_amdgcn_cvt_f32_fp8((int)w, 0) : i == 1 ? __builtin_amdgcn_cvt_f32_fp8((int)w, 1)
               : i == 2 ? __builtin_amdgcn_cvt_f32_fp8((int)w, 2) : __builtin_amdgcn_cvt_f32_fp8((int)w, 3);
    }
    f32x4 w[2][4];       // V as numbers
    __device__ __forceinline__ bool stage_v(bool edge, int first, int last, unsigned there, int lane) {
        bool odd = false;
        const int l16 = lane & 15, quad = lane >> 4;
#pragma unroll
        for (int blk = 0; blk < 2; ++blk)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (kCodes) {
                    const float p = exp_of_byte(ve[blk][e]);
#pragma unroll
                    for (int d = 0; d < 4; ++d) w[blk][e][d] = p * code(v[blk][e], d);
                } else {
                    w[blk][e] = v[blk][e];
                }
                if (edge) {
                    const int r = 16 * blk + 4 * quad + e;
                    const bool in = r >= first && r < last && (there >> blk & 1);
#pragma unroll
                    for (int d = 0; d < 4; ++d) {
                        w[blk][e][d] = in ? w[blk][e][d] : 0.0f;
                        odd = odd || (__float_as_uint(w[blk][e][d]) & 0x7f800000u) == 0x7f800000u;
                    }
                    *reinterpret_cast<__attribute__((address_space(3))) f32x4 *>((uintptr_t)(stage + (r * kD + 4 * l16) * 4)) = w[blk][e];
                }
            }
        return odd;
    }
    __device__ __forceinline__ void product(const f32x4 (&s)[NB][2]) {
#pragma unroll
        for (int blk = 0; blk < 2; ++blk)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int d = 0; d < 4; ++d)
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) o[nb][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[blk][e][d], s[nb][blk][e], o[nb][d], 0, 0, 0);
    }
    __device__ __forceinline__ static int column(int d, int e, int quad) { return 16 * quad + 4 * e + d; }
    __device__ __forceinline__ static float staged(uint32_t stage, int key, int col) {
        return *reinterpret_cast<const __attribute__((address_space(3))) float *>((uintptr_t)(stage + (key * kD + col) * 4));
    }
};

template <typename T, typename ST, int NB>
constexpr int paged_lds_bytes() {
    constexpr int merge = kPagedWaves * 16 * (NB > 2 ? 2 : NB) * kPagedRow * 4, stages = kPagedWaves * PagedTile<T, ST, NB>::kStage;
    return stages > merge ? stages : merge;
}

// Eight columns of a finished row: weights' sum l and products `acc` relative to the maximum `top`, the sink not yet among them.
template <typename T>
__device__ __forceinline__ void paged_finish(const PagedArgs &a, const PagedSpan &sp, int row, int head, int c8, float top, float l, const float (&acc)[8]) {
    const float sink = paged_sink(a, head), sink2 = sink * kLog2e;
    // (the larger one's weight is 1 and not the power of a difference with itself, which a fused multiply-add of the logit would not make 0)
    const bool by_sink = sink2 >= top;
    const float ref = by_sink ? sink2 : top, f = by_sink ? fast_exp2(top - sink2) : 1.0f;
    const float z = l * f + (by_sink ? 1.0f : fast_exp2(sink2 - top));
    const int pos = sp.base + row;
    const bool none = pos < 0 || pos >= sp.n || l == 0.0f;          // no query, or no key that it sees
    const float mul = none ? 0.0f : f / z;
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = none ? 0.0f : acc[e] * mul;
    store8(static_cast<T *>(a.o) + sp.b * a.os.b + head * a.os.h + row * a.os.s + c8, x);
    if (c8 == 0) a.lse[((int64_t)sp.b * a.H + head) * a.Sq + row] = none ? sink : (ref + fast_log2(z)) * kLn2;
}

template <typename T, typename ST, int NB>
__global__ __launch_bounds__(64 * kPagedWaves, NB == 1 && sizeof(T) == 2 ? 4 : 2) void attn_paged_kernel(const PagedArgs a) {
    using Tile = PagedTile<T, ST, NB>;
    constexpr int NW = kPagedWaves, kPairs = 16 * NB;
    __shared__ __attribute__((aligned(128))) char smem[paged_lds_bytes<T, ST, NB>()];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, quad = lane >> 4;
    const int g = blockIdx.x % a.G;
    const PagedShare share = paged_share(a, blockIdx.x / a.G, kPairs);
    const int unit = __builtin_amdgcn_readfirstlane(share.unit);
    if (unit < 0) return;
    const PagedSpan sp = paged_span(a, unit, kPairs);
    const int t_lo = sp.t_first + (int)((int64_t)sp.tiles * share.index / share.count);
    const int n_wg = sp.t_first + (int)((int64_t)sp.tiles * (share.index + 1) / share.count) - t_lo;
    const int n_it = n_wg > w ? (n_wg - w + NW - 1) / NW : 0;       // this wavefront's tiles: t_lo + w + NW j
    const int pairs = min(a.Sq * a.r - sp.pair0, kPairs);

    Tile tile;
    const uint32_t stage = lds_addr(smem) + w * Tile::kStage;
    tile.init(stage, lane);
    int pq[NB];                // position of the column's query
    float m[NB], l[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        const bool ok = 16 * nb + l16 < pairs;
        const int pair = sp.pair0 + (ok ? 16 * nb + l16 : 0), row = pair / a.r, head = g * a.r + pair % a.r;
        pq[nb] = sp.base + row;
        tile.load_q(nb, static_cast<const T *>(a.q) + sp.b * a.qs.b + head * a.qs.h + row * a.qs.s, ok, quad);
        m[nb] = kLowest;
        l[nb] = 0.0f;
    }

    const int32_t *table = a.table + sp.b * a.table_stride;
    const int in_page = (1 << a.page_shift) - 1, weff = a.window ? a.window : 0x3fffffff;
    int entry0 = 0, entry1 = 0;              // pages of the wavefront's next 64 tiles, one a lane: their first and second 16 keys
    unsigned there = 0;                      // of the tile under way: which of the two exist
    auto entry = [&](int token) {
        const int i = token >> a.page_shift;
        const int page = i < a.width ? table[i] : -1;
        return (unsigned)page < (unsigned)a.pages ? page : -1;
    };
    auto entries = [&](int j) __attribute__((always_inline)) {
        if ((j & 63) == 0) {
            const int n0 = (t_lo + w + NW * (j + lane)) * kPagedKeys;
            const bool mine = j + lane < n_it;
            entry0 = mine ? entry(n0) : -1;
            entry1 = mine ? (a.page_shift > 4 ? entry0 : entry(n0 + 16)) : -1;
        }
    };
    auto page_of = [&](int j, int blk) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(blk ? entry1 : entry0, j & 63); };
    auto fetch_k = [&](int j) __attribute__((always_inline)) {
        const int n0 = (t_lo + w + NW * j) * kPagedKeys;
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) {
            const int page = max(page_of(j, blk), 0), slot = (n0 + 16 * blk) & in_page;
            tile.load_k(blk, a.k_pages + (page * a.kps.b + g * a.kps.h + slot * a.kps.s) * (int)sizeof(ST),
                        Tile::kCodes ? a.k_exp + page * a.kes.b + g * a.kes.h + slot * a.kes.s : nullptr, a, lane);
        }
    };
    auto fetch_v = [&](int j) __attribute__((always_inline)) {
        const int n0 = (t_lo + w + NW * j) * kPagedKeys;
#pragma unroll
        for (int blk = 0; blk < 2; ++blk) {
            const int page = max(page_of(j, blk), 0), slot = (n0 + 16 * blk) & in_page;
            tile.load_v(blk, a.v_pages + (page * a.vps.b + g * a.vps.h + slot * a.vps.s) * (int)sizeof(ST),
                        Tile::kCodes ? a.v_exp + page * a.ves.b + g * a.ves.h + slot * a.ves.s : nullptr, a, lane);
        }
    };

    if (n_it > 0) {
        entries(0);
        fetch_k(0);
        fetch_v(0);
    }
    for (int j = 0; j < n_it; ++j) {
        const int n0 = (t_lo + w + NW * j) * kPagedKeys;
        there = (page_of(j, 0) >= 0 ? 1u : 0u) | (page_of(j, 1) >= 0 ? 2u : 0u);
        const bool edge = !(n0 + kPagedKeys - 1 <= sp.pos0 && n0 > sp.pos1 - weff && there == 3u);
        f32x4 s[NB][2];
        tile.logits(s);
        const bool more = j + 1 < n_it;
        if (more) {
            entries(j + 1);
            fetch_k(j + 1);
        }
        const bool odd = tile.stage_v(edge, sp.lo - n0, sp.hi - n0, there, lane);
        if (more) fetch_v(j + 1);
        // (a key that one query sees and another does not: only where there are several)
        const bool by_hand = edge && sp.pos0 != sp.pos1 && __builtin_amdgcn_ballot_w64(odd) != 0ull;

#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            if (edge) {
#pragma unroll
                for (int blk = 0; blk < 2; ++blk)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int key = n0 + 16 * blk + 4 * quad + e;
                        s[nb][blk][e] = key <= pq[nb] && key > pq[nb] - weff && (there >> blk & 1) ? s[nb][blk][e] : -INFINITY;
                    }
            }
            float mx = s[nb][0][0];
#pragma unroll
            for (int e = 1; e < 8; ++e) mx = fast_max(mx, s[nb][e >> 2][e & 3]);
            mx *= a.scale_log2;
            if (__builtin_amdgcn_ballot_w64(mx > m[nb] + kRaise) != 0ull) {
                const float m_new = fast_max(m[nb], quad_max(mx)), alpha = fast_exp2(m[nb] - m_new);
                l[nb] *= alpha;
#pragma unroll
                for (int d = 0; d < 4; ++d) tile.o[nb][d] *= alpha;
                m[nb] = m_new;
            }
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float p = fast_exp2(fmaf(s[nb][e >> 2][e & 3], a.scale_log2, -m[nb]));
                s[nb][e >> 2][e & 3] = p;
                sum += p;
            }
            l[nb] += sum;
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        if (!by_hand) {
            tile.product(s);
        } else {
            // infinities or NaN in V: key by key, and only for the queries that see it (0 times infinity is NaN)
#pragma unroll 1
            for (int key = 0; key < kPagedKeys; ++key) {
                const int from = ((key >> 2 & 3) << 4) | l16, reg = (key >> 4) * 4 + (key & 3);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    float p = s[nb][0][0];
#pragma unroll
                    for (int e = 1; e < 8; ++e) p = reg == e ? s[nb][e >> 2][e & 3] : p;
                    p = __shfl(p, from);
                    if (n0 + key <= pq[nb] && n0 + key > pq[nb] - weff && (there >> (key >> 4) & 1)) {
#pragma unroll
                        for (int d = 0; d < 4; ++d)
#pragma unroll
                            for (int e = 0; e < 4; ++e) tile.o[nb][d][e] += p * Tile::staged(stage, key, Tile::column(d, e, quad));
                    }
                }
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }

    // ---- merge the wavefronts, up to 32 pairs at a time: rows [wavefront][pair][64 + (m, l)] in LDS ----
    constexpr int kHalf = NB > 2 ? 2 : NB;
    float *red = reinterpret_cast<float *>(smem);
    float *part = a.partial + ((int64_t)(share.first + share.index) * a.G + g) * paged_partial_floats(NB);
#pragma unroll
    for (int h = 0; h < NB / kHalf; ++h) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kHalf; ++i) {
            const int nb = h * kHalf + i;
            float *row = red + (w * 16 * kHalf + 16 * i + l16) * kPagedRow;
            const float l_tot = quad_sum(l[nb]);
#pragma unroll
            for (int d = 0; d < 4; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) row[Tile::column(d, e, quad)] = tile.o[nb][d][e];
            if (quad == 0) { row[kD] = m[nb]; row[kD + 1] = l_tot; }
        }
        __syncthreads();
        // eight lanes per row, eight columns each
        const int c8 = (tid & 7) * 8, local = tid >> 3;
        const int slot = h * 16 * kHalf + local;
        if (local < 16 * kHalf && slot < pairs) {
            float top = kLowest, l_all = 0.0f, acc[8];
#pragma unroll
            for (int k = 0; k < NW; ++k) top = fast_max(top, red[(k * 16 * kHalf + local) * kPagedRow + kD]);
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] = 0.0f;
#pragma unroll
            for (int k = 0; k < NW; ++k) {
                const float *row = red + (k * 16 * kHalf + local) * kPagedRow;
                const float f = fast_exp2(row[kD] - top);
                l_all += f * row[kD + 1];
#pragma unroll
                for (int e = 0; e < 8; ++e) acc[e] += f * row[c8 + e];
            }
            if (share.count > 1) {
                *reinterpret_cast<f32x4 *>(part + slot * kD + c8) = f32x4{acc[0], acc[1], acc[2], acc[3]};
                *reinterpret_cast<f32x4 *>(part + slot * kD + c8 + 4) = f32x4{acc[4], acc[5], acc[6], acc[7]};
                if (c8 == 0) { part[kPairs * kD + 2 * slot] = top; part[kPairs * kD + 2 * slot + 1] = l_all; }
            } else {
                const int pair = sp.pair0 + slot, row = pair / a.r, head = g * a.r + pair % a.r;
                paged_finish<T>(a, sp, row, head, c8, top, l_all, acc);
            }
        }
    }
    if (a.plan && share.index == 0 && g == 0 && tid == 0) {
        a.plan[2 * unit] = share.first;
        a.plan[2 * unit + 1] = share.count;
    }
}

// Shares of one (batch row, head, query) row, one wavefront per row: lane = (group of shares, 8 columns), added in an order that
// depends on their number only.
template <typename T, int NB>
__global__ __launch_bounds__(256) void attn_paged_combine_kernel(const PagedArgs a) {
    constexpr int kPairs = 16 * NB;
    const int lane = threadIdx.x & 63, c8 = (lane & 7) * 8, sg = lane >> 3;
    const int64_t idx = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int64_t per_head = (int64_t)a.Sq * a.r;
    if (idx >= (int64_t)a.B * a.G * per_head) return;
    const int pair = (int)(idx % per_head), g = (int)(idx / per_head % a.G), b = (int)(idx / per_head / a.G);
    const int unit = b * a.blocks + pair / kPairs, slot = pair % kPairs;
    const int first = a.plan[2 * unit], count = a.plan[2 * unit + 1];
    if (count == 1) return;
    const float *part = a.partial + ((int64_t)first * a.G + g) * paged_partial_floats(NB);
    const int64_t step = a.G * paged_partial_floats(NB);
    float m = kLowest, l = 0.0f, acc[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = 0.0f;
    for (int s = sg; s < count; s += 8) {
        const float *p = part + s * step;
        const float ms = p[kPairs * kD + 2 * slot], ls = p[kPairs * kD + 2 * slot + 1];
        const f32x4 x = *reinterpret_cast<const f32x4 *>(p + slot * kD + c8), y = *reinterpret_cast<const f32x4 *>(p + slot * kD + c8 + 4);
        const float mn = fast_max(m, ms), fo = fast_exp2(m - mn), f = fast_exp2(ms - mn);
        l = l * fo + f * ls;
#pragma unroll
        for (int e = 0; e < 4; ++e) { acc[e] = acc[e] * fo + f * x[e]; acc[4 + e] = acc[4 + e] * fo + f * y[e]; }
        m = mn;
    }
    float top = m;
    top = fast_max(top, __shfl_xor(top, 8));
    top = fast_max(top, __shfl_xor(top, 16));
    top = fast_max(top, __shfl_xor(top, 32));
    const float f = fast_exp2(m - top);
    l *= f;
    l += __shfl_xor(l, 8); l += __shfl_xor(l, 16); l += __shfl_xor(l, 32);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        acc[e] *= f;
        acc[e] += __shfl_xor(acc[e], 8); acc[e] += __shfl_xor(acc[e], 16); acc[e] += __shfl_xor(acc[e], 32);
    }
    if (sg == 0) paged_finish<T>(a, paged_span(a, unit, kPairs), pair / a.r, g * a.r + pair % a.r, c8, top, l, acc);
}

}  // namespace gptoss
