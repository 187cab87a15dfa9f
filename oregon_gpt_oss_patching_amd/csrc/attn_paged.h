// Attention of new queries over a key / value cache in pages (gptoss_attn_paged_fwd).
//
// What bounds it: reading the rows that the queries see once from HBM, or, for short rows, the latency of a launch or two.
//
// Work.  The Sq * r (query, head of the group) pairs of a KV head are the columns of S^T, up to 16 NB of them to a workgroup (a unit), so that
// K and V are read once.  The host does not see the lengths: a fixed number of workgroups finds, from all lengths, how long equal shares of
// all units' tiles (of 16, 32 or 64 keys) are and which share is its own (PagedShare); a unit with one share writes its results, the others leave fp32
// partials that attn_paged_combine_kernel adds in the order of the shares.  So one long row among many short ones is spread over the chip,
// and rows are divided alike in a table that fits them and in a wider one (but for the shortest, which the host sends to a workgroup each where the table says that they are:
// gptoss_paged.hip).
//
// In a workgroup four wavefronts take tiles in turn, each for itself (no barrier in the loop), and merge their (m, l, O) at the end.
//  * Loads take whole cache lines.  The MFMA's A operand wants a lane to hold pieces of one key's row, 16 rows of 64 bytes to a load: codes come so,
//    but rows of more bytes loaded that way keep a compute unit at 37 GB/s (one workgroup of 16 wavefronts; with whole rows 131), so K goes
//    through a stage of LDS first.  Which number of the row stands in which slot of the contraction is free as long as Q has the same order.
//  * V has to be turned (the contraction runs over keys): for bf16 products it goes through the same stage, after K, and is read back transposed;
//    from float32 pages each lane loads four columns of its own four keys, which is what the fp32 MFMA takes.
//  * P leaves the S product in the layout of the PV product's B operand.
//  * Entries of the page table are loaded 64 tiles at a time, one per lane; a tile's page is a readlane and its addresses are scalar.
//  * e4m3 rows widen on the way into the operand: to bf16 by the instruction that takes a power of two along (exact), K's with one
//    power per lane, V's before they are staged; float32 queries then go in as three bf16 terms.
// The running maximum is raised only when a logit passes it by more than 2^8 (the sums are in 32 bits and the weights keep their relative
// precision): the reduction over the lanes and the rescaling are then rare.
#pragma once
#include <type_traits>

#include "paged_common.h"

namespace gptoss {

constexpr int kPagedMaxUnits = 1024;
constexpr int kPagedRow = kD + 2;               // floats of a merged row: O, m, l
constexpr float kRaise = 8.0f;                  // in the exponent of two

// Wavefronts of a workgroup: four, or (NW) up to as many as a compute unit runs where one workgroup walks a unit alone.
constexpr int kPagedWaves = 4;
// Blocks of 16 keys in a tile: what a wavefront has under way is a tile, so rows of fewer bytes come more at a time; two columns' worth of
// float32 numbers leave registers for one block.
template <typename T, typename ST, int NB, int NW> __host__ __device__ constexpr int paged_tile_blocks() {
    return sizeof(ST) == 4 ? (NB > 1 ? 1 : 2) : sizeof(ST) == 1 && NB == 1 && NW == kPagedWaves ? 4 : 2;
}
// Wavefronts per SIMD, of what the registers leave.
template <typename T, typename ST, int NB, int NW> __host__ __device__ constexpr int paged_occupancy() {
    return sizeof(ST) == 4 ? (NB == 2 && NW == kPagedWaves ? 3 : 2) : sizeof(T) == 4 ? 3 : NB == 1 ? 4 : NB == 2 || (NB == 3 && sizeof(ST) == 1) ? 3 : 2;
}
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
__device__ __forceinline__ int paged_base(const PagedArgs &a, int b, int n) {
    // (positions of 2^30 and more exist in no row; below -2^30 no query reaches one that does)
    return a.start ? min(max(a.start[b], -(1 << 30)), 1 << 30) : n - a.Sq;
}
template <int PAIRS, int KEYS>
__device__ __forceinline__ PagedSpan paged_span(const PagedArgs &a, int b, int block, int n, int base) {
    PagedSpan s;
    s.b = b;
    s.pair0 = block * PAIRS;
    s.n = n;
    s.base = base;
    const int i0 = a.by_r.quotient(s.pair0), i1 = min(a.Sq - 1, a.by_r.quotient(s.pair0 + PAIRS - 1));
    s.pos0 = max(base + i0, 0);
    s.pos1 = min(base + i1, n - 1);
    const bool any = s.pos0 <= s.pos1;
    s.lo = any && a.window ? max(0, s.pos0 - a.window + 1) : 0;
    s.hi = any ? s.pos1 + 1 : 0;
    s.t_first = s.lo / KEYS;
    s.tiles = any ? (s.hi + KEYS - 1) / KEYS - s.t_first : 0;
    return s;
}

// x + (x of all lanes below), over the wavefront, without LDS: within rows of 16 lanes, then over the rows
__device__ __forceinline__ int wave_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);        // row_shr:1
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);        // row_bcast:15 into rows 1 and 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);        // row_bcast:31 into rows 2 and 3
    return x;
}

// The sum of the lanes' numbers, each at most 2^30 / KEYS: 64 times 2^26 (tiles of 16 keys) does not fit 32 bits.
template <int KEYS>
__device__ __forceinline__ uint64_t wave_total(int x) {
    if constexpr (KEYS >= 32) return (uint32_t)__builtin_amdgcn_readlane(wave_scan(x), 63);
    const uint32_t lo = __builtin_amdgcn_readlane(wave_scan(x & 0xffff), 63), hi = __builtin_amdgcn_readlane(wave_scan(x >> 16), 63);
    return ((uint64_t)hi << 16) + lo;
}

// Length of the shares that `tiles` are cut into: the smallest of at least `least` with which units that have so many in all have no more than `shares`, and
// one for each unit, which is what the grid and the scratch hold.
__host__ __device__ __forceinline__ int paged_chunk(uint64_t tiles, int shares, int least) {
    const uint64_t up = tiles + (uint32_t)shares - 1u;
    const uint64_t even = up >> 32 ? up / (uint32_t)shares : (uint32_t)up / (uint32_t)shares;     // (32 bits: a quotient in a tenth of the instructions)
    const int chunk = even < (1u << 30) ? (int)even : 1 << 30;                                    // (more tiles than a unit can have)
    return chunk > least ? chunk : least;
}

// The least length of a share, in 128 keys, from how many workgroups (shares of all units for all KV heads) there are with shares of one, two, three and six times that,
// for 256 compute units: 128, 256 or 384 keys, the first with which each workgroup has a compute unit to itself; where none has, 768 if that fills the compute units evenly,
// four fifths of whole rounds, and 384 if not.  us at 128 / 256 / 384 / 768, workgroups in brackets:
//   1 x 2049 tokens 8.8 [136] / 9.2 / 9.8 / -, 1 x 5000 10.6 [320] / 9.6 [160] / 10.3 / -, 2 x 4000 11.5 / 10.1 [256] / 10.8 / 12.3, 1 x 10000 13.1 / 12.0 [320] / 10.7 [216] / 12.3, in
//   32 bits 16.6 / 17.7 / 14.9 / 18.5, 20 of 100 to 6000 on two KV heads, five queries, 17.6 / 15.6 [258] / 14.7 [180] / 17.0;
//   8 of 700 to 6000 - / 14.9 / 14.5 [464] / 14.4 [248], under five queries - / 20.3 / 20.0 / 18.7, in 32 bits - / 23.1 / 22.6 / 22.3, 16 of 500 to 6000 20.4 [824] / 19.1 [440], in e4m3
//   17.7 / 16.0, 32 of 100 to 3000 17.4 [712] / 17.0 [440];
//   but 24 of 100 to 2500 14.2 [480] / 15.2 [304], 4 x 8193 17.9 [704] / 18.9 [352], 12 of 700 to 6000 under five queries 22.7 [512] / 24.0 [360], under eight 24.8 / 26.5.
__host__ __device__ __forceinline__ int paged_least(int of1, int of2, int of3, int of6) {
    constexpr int kUnits = 256;
    if (of1 <= kUnits) return 1;
    if (of2 <= kUnits) return 2;
    if (of3 <= kUnits) return 3;
    const int rounds = (of6 + kUnits - 1) / kUnits;
    return (int64_t)5 * of6 >= (int64_t)4 * kUnits * rounds ? 6 : 3;
}

// Which share of which unit a workgroup takes.
struct PagedShare { int unit, index, count, first; };     // first: number of the unit's first share; unit < 0: nothing left
template <int PAIRS, int KEYS>
__device__ __forceinline__ PagedShare paged_share(const PagedArgs &a, int slot, PagedSpan &sp) {
    const int lane = threadIdx.x & 63;
    if (!a.shares) {
        const int b = a.by_blocks.quotient(slot), n = paged_length(a, b);
        sp = paged_span<PAIRS, KEYS>(a, b, slot - b * a.blocks, n, paged_base(a, b, n));
        return PagedShare{slot, 0, 1, slot};
    }
    // a lane's unit, the first 64 of them kept
    auto mine = [&](int u, int &n, int &base) __attribute__((always_inline)) {
        n = base = 0;
        if (u >= a.units) return 0;
        const int b = a.by_blocks.quotient(u);
        n = paged_length(a, b);
        base = paged_base(a, b, n);
        return paged_span<PAIRS, KEYS>(a, b, u - b * a.blocks, n, base).tiles;
    };
    int n, base;
    const int tiles0 = mine(lane, n, base);
    uint64_t all = wave_total<KEYS>(tiles0);
    // numbers of shares of n times 128 keys, two at a time in 16 bits (which they fit wherever they are used: at most six times a.shares, and one for each unit)
    constexpr int k128 = 128 / KEYS;
    auto numbers = [&](int u, int tiles, int n, int m) __attribute__((always_inline)) {
        const uint32_t x = max(1, (tiles + n * k128 - 1) / (n * k128)), y = max(1, (tiles + m * k128 - 1) / (m * k128));
        return (uint32_t)__builtin_amdgcn_readlane(wave_scan(u < a.units ? (int)(x + (y << 16)) : 0), 63);
    };
    uint32_t of12 = numbers(lane, tiles0, 1, 2), of36 = numbers(lane, tiles0, 3, 6);
    for (int u0 = 64; u0 < a.units; u0 += 64) {
        int x, y;
        const int tiles = mine(u0 + lane, x, y);
        all += wave_total<KEYS>(tiles);
        of12 += numbers(u0 + lane, tiles, 1, 2);
        of36 += numbers(u0 + lane, tiles, 3, 6);
    }
    int chunk = paged_chunk(all, a.shares, 1);
    if (chunk < 6 * k128)
        chunk = max(chunk, k128 * paged_least((of12 & 0xffff) * a.G, (of12 >> 16) * a.G, (of36 & 0xffff) * a.G, (of36 >> 16) * a.G));
    int before = 0;
    for (int u0 = 0; u0 < a.units; u0 += 64) {
        const int tiles = u0 ? mine(u0 + lane, n, base) : tiles0;
        const int shares = u0 + lane < a.units ? max(1, (int)((uint32_t)(tiles + chunk - 1) / (uint32_t)chunk)) : 0;
        const int incl = wave_scan(shares), first = before + incl - shares;
        const unsigned long long who = __builtin_amdgcn_ballot_w64(slot >= first && slot < first + shares);
        if (who) {
            const int l = __builtin_ctzll(who), f = __builtin_amdgcn_readlane(first, l), b = a.by_blocks.quotient(u0 + l);
            sp = paged_span<PAIRS, KEYS>(a, b, u0 + l - b * a.blocks, __builtin_amdgcn_readlane(n, l), __builtin_amdgcn_readlane(base, l));
            return PagedShare{u0 + l, slot - f, __builtin_amdgcn_readlane(shares, l), f};
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

// A lane's 32-bit offset from a scalar address.  Hidden, as the compiler widens it once in front of the loop otherwise, and then adds 64 bits per load.
__device__ __forceinline__ uint32_t lane_offset(uint32_t at, uint32_t mask) {
    at &= mask;
    asm volatile("" : "+v"(at));
    return at;
}

// kOnce: rows that no other workgroup reads bypass the caches' retention, us without / with: 16 x 8192 tokens 54.6 / 47.3, 4 x 65536 101 / 87.2 (6.2 TB/s), 64 rows of 150
// to 16384 96.7 / 84.8, 32 of 6000 to 16384 in e4m3 74.8 / 66.2.  A row of more pairs than a workgroup takes is read again by the next one (NB = 4, and two
// blocks in 32 bits).
// A tile's K and V as they are loaded, and what is done with them.  `kb` / `vb`: scalar addresses of the first row of a block of 16 keys;
// lanes: l16 = lane % 16, quad = lane / 16.
template <typename T, typename ST, int NB, int KB> struct PagedTile;

// Eight numbers as their upper 16 bits, and what is left of them.
__device__ __forceinline__ bf16x8 take_upper(float (&x)[8]) {
    u32x4 u;
#pragma unroll
    for (int e = 0; e < 4; ++e) u[e] = __builtin_amdgcn_perm(__float_as_uint(x[2 * e + 1]), __float_as_uint(x[2 * e]), 0x07060302u);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] -= __uint_as_float(__float_as_uint(x[e]) & 0xffff0000u);
    return as_bf16x8(u);
}

// Eight weights as two bfloat16 terms each: the upper 16 bits, and what is left, which is less than 2^-7 of the weight and rounded by 2^-8 of itself, so that
// their sum is off by 2^-15 of the weight at most.  2^-20 of the weight is added to what is left, as 0 times an infinity in V would be NaN, where a weight times
// infinity is infinity (for weights above 2^-110, as below 2^-126 for a single term).
__device__ __forceinline__ void split_weights(const float (&x)[8], bf16x8 &hi, bf16x8 &lo) {
    u32x4 u;
#pragma unroll
    for (int e = 0; e < 4; ++e) u[e] = __builtin_amdgcn_perm(__float_as_uint(x[2 * e + 1]), __float_as_uint(x[2 * e]), 0x07060302u);
    hi = as_bf16x8(u);
#pragma unroll
    for (int e = 0; e < 8; ++e) lo[e] = (bf16)fmaf(x[e], 1.0f + 0x1p-20f, -__uint_as_float(__float_as_uint(x[e]) & 0xffff0000u));
}

// ---- bfloat16 products -----------------------------------------------------------------------------------------------
// Of float32 queries over codes too: a code times its power of two is a bfloat16 number, and a float32 number is the sum of three (its 24 bits, eight
// at a time), so three products of each kind take the place of the fp32 MFMA's, in a fifth of their time: 32 rows of 6000 to 16384 tokens 69 us, and 135 with those.
// The smaller terms are added first, to 0: their roundings are then 2^-8 of the sum's.
template <typename T, typename ST, int NB, int KB>
struct PagedTile16 {
    static constexpr bool kCodes = sizeof(ST) == 1, kOnce = NB < (sizeof(T) == 4 ? 2 : 4), kStagedK = !kCodes;
    static constexpr int kTerms = sizeof(T) == 4 ? 3 : 1;
    static constexpr int kStage = 16 * KB * kRowBytes;           // LDS bytes of a wavefront
    static constexpr int kVecs = kCodes ? 1 : 2;                 // 16-byte loads per lane and block
    u32x4 k[KB][kVecs], v[KB][kVecs];
    uint32_t ke[KB], ve[KB];
    bf16x8 q[NB][kTerms][2];     // the largest term first
    f32x4 o[NB][4];
    uint32_t tr[4], wr[2], nat[2], k_at[kVecs], v_at[kVecs], ke_at, ve_at;

    // (codes: rows 0, 1, 4, 5 and so on for each 16 lanes, which then write to distinct banks)
    __device__ __forceinline__ static int v_row(int lane, int i) {
        const int q = lane >> 2;
        return kCodes ? (q & 9) | (q & 2) << 1 | (q & 4) >> 1 : (lane >> 3) + 8 * i;
    }

    __device__ __forceinline__ void init(const PagedArgs &a, uint32_t stage, int lane) {
        const int i = lane & 15, quad = lane >> 4, row = 4 * quad + (i >> 2);
#pragma unroll
        for (int d = 0; d < 4; ++d) tr[d] = stage + row * kRowBytes + (((2 * d + ((i & 3) >> 1)) ^ swz(row)) * 16) + (i & 1) * 8;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = v_row(lane, e), c = kCodes ? 2 * (lane & 3) + e : lane & 7;
            wr[e] = stage + r * kRowBytes + ((c ^ swz(r)) * 16);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) nat[e] = stage + i * kRowBytes + (((4 * e + quad) ^ swz(i)) * 16);
#pragma unroll
        for (int e = 0; e < kVecs; ++e) k_at[e] = kCodes ? i * a.kp.s + 16 * quad : v_row(lane, e) * a.kp.s + 16 * (lane & 7);
#pragma unroll
        for (int e = 0; e < kVecs; ++e) v_at[e] = v_row(lane, e) * a.vp.s + 16 * (kCodes ? lane & 3 : lane & 7);
        ke_at = i * a.ke.s;
        ve_at = v_row(lane, 0) * a.ve.s;
    }
    __device__ __forceinline__ void load_q(int nb, const T *row, bool there, int quad) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const T *at = row + (kCodes ? 16 * quad + 8 * s : 32 * s + 8 * quad);
            if constexpr (kTerms == 1) {
                const u32x4 x = *reinterpret_cast<const u32x4 *>(at);
                q[nb][0][s] = as_bf16x8(there ? x : u32x4{0, 0, 0, 0});
            } else {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = there ? at[e] : 0.0f;
#pragma unroll
                for (int t = 0; t < kTerms; ++t) {
                    q[nb][t][s] = take_upper(x);
                    // (an infinity less itself is not what is left of it)
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = isinf(at[e]) ? 0.0f : x[e];
                }
            }
        }
#pragma unroll
        for (int d = 0; d < 4; ++d) o[nb][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    // `mask`: all ones, or 0 where there is no next tile (one address instead of a branch)
    __device__ __forceinline__ void load_k(int blk, const char *kb, const char *eb, uint32_t mask) {
#pragma unroll
        for (int s = 0; s < kVecs; ++s) k[blk][s] = load16<kOnce>(kb + lane_offset(k_at[s], mask));
        if constexpr (kCodes) ke[blk] = (uint8_t)eb[lane_offset(ke_at, mask)];
    }
    __device__ __forceinline__ void load_v(int blk, const char *vb, const char *eb, uint32_t mask) {
#pragma unroll
        for (int i = 0; i < kVecs; ++i) v[blk][i] = load16<kOnce>(vb + lane_offset(v_at[i], mask));
        if constexpr (kCodes) ve[blk] = (uint8_t)eb[lane_offset(ve_at, mask)];
    }
    __device__ __forceinline__ void stage_k() const {
#pragma unroll
        for (int blk = 0; blk < KB; ++blk)
#pragma unroll
            for (int i = 0; i < kVecs; ++i) *reinterpret_cast<__attribute__((address_space(3))) u32x4 *>((uintptr_t)(wr[i] + 16 * blk * kRowBytes)) = k[blk][i];
    }
    __device__ __forceinline__ void logits(f32x4 (&s)[NB][KB]) const {
#pragma unroll
        for (int blk = 0; blk < KB; ++blk) {
            bf16x8 f[2];
            if constexpr (kCodes) {
                const float p = exp_of_byte(ke[blk]);
                f[0] = widen8(k[blk][0][0], k[blk][0][1], p);
                f[1] = widen8(k[blk][0][2], k[blk][0][3], p);
            } else {
                f[0] = as_bf16x8(lds_load128(nat[0], 16 * blk * kRowBytes));
                f[1] = as_bf16x8(lds_load128(nat[1], 16 * blk * kRowBytes));
            }
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                f32x4 z = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int t = kTerms - 1; t >= 0; --t) {
                    z = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f[0], q[nb][t][0], z, 0, 0, 0);
                    z = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f[1], q[nb][t][1], z, 0, 0, 0);
                }
                s[nb][blk] = z;
            }
        }
    }
    // V into the stage.  Where `edge`: rows outside first .. last - 1 of the tile as zeros; with `several` queries, what is not finite in the
    // others as zeros too, and the answer is whether there was such a thing.
    __device__ __forceinline__ bool stage_v(bool edge, bool several, int first, int last, unsigned there, int lane) {
        bool odd = false;
        if (edge) {
#pragma unroll
            for (int blk = 0; blk < KB; ++blk)
#pragma unroll
                for (int i = 0; i < kVecs; ++i) {
                    const int r = 16 * blk + v_row(lane, i);
                    const bool in = r >= first && r < last && (there >> blk & 1);
                    if constexpr (kCodes) ve[blk] = in ? ve[blk] : (uint32_t)kExpBias;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[blk][i][e] = in ? v[blk][i][e] : 0u;
                }
            if (several) {
#pragma unroll
                for (int blk = 0; blk < KB; ++blk) {
                    // Added to the magnitudes of codes, what carries those that are not finite into the sign's bit: NaN, 0x7f; under 2^120 and more what comes to 2^128, from 0x78
                    // down by 8 for each power; under the byte 255 all of them.
                    uint32_t carry = 0x01010101u;
                    if constexpr (kCodes) {
                        carry = ve[blk] < 247u ? carry : ve[blk] == 255u ? 0x80808080u : 0x08080808u * (ve[blk] - 246u);
                        ve[blk] = ve[blk] == 255u ? (uint32_t)kExpBias : ve[blk];
                    }
#pragma unroll
                    for (int i = 0; i < kVecs; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t x = v[blk][i][e];
                            uint32_t bad;
                            if constexpr (kCodes) bad = ((((x & 0x7f7f7f7fu) + carry) & 0x80808080u) >> 7) * 0xffu;
                            else bad = ((x & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) | ((x & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u);
                            odd = odd || bad != 0u;
                            v[blk][i][e] = x & ~bad;
                        }
                }
            }
        }
#pragma unroll
        for (int blk = 0; blk < KB; ++blk)
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
                *reinterpret_cast<__attribute__((address_space(3))) u32x4 *>((uintptr_t)(wr[i] + 16 * blk * kRowBytes)) = x;
            }
        return odd;
    }
    __device__ __forceinline__ void product(const f32x4 (&s)[NB][KB]) {
#pragma unroll
        for (int h = 0; h < KB / 2; ++h) {
            // A bfloat16 query's weights go in as two terms: one alone, half a step of bfloat16 of each weight, adds as much to the result's error as
            // rounding it does (relative, 2-norm: 2.2e-3 in all and not 1.7e-3).  us, one term / two: 16 x 8192 tokens 48.7 / 48.9, in e4m3 30.7 / 31.1, one row of 2049 8.5 / 8.6,
            // five queries on eight rows of 700 to 6000 17.6 / 18.3; where the arithmetic counts, eight queries on 16 x 8192 in e4m3, 43.0 / 49.5.
            constexpr int kWeightTerms = kTerms == 1 ? 2 : kTerms;
            bf16x8 p[NB][kWeightTerms];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = s[nb][2 * h + (e >> 2)][e & 3];
                if constexpr (kTerms == 1) {
                    split_weights(x, p[nb][0], p[nb][1]);
                } else {
#pragma unroll
                    for (int t = 0; t < kTerms; ++t) p[nb][t] = take_upper(x);
                }
            }
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                union { struct { s16x4 a, b; } s; bf16x8 v; } x;
                x.s.a = lds_load_tr64(tr[d], 32 * h * kRowBytes);
                x.s.b = lds_load_tr64(tr[d], (32 * h + 16) * kRowBytes);
                if constexpr (kTerms == 1) {
#pragma unroll
                    for (int t = kWeightTerms - 1; t >= 0; --t)
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) o[nb][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.v, p[nb][t], o[nb][d], 0, 0, 0);
                } else {
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        f32x4 z = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int t = kTerms - 1; t >= 0; --t) z = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.v, p[nb][t], z, 0, 0, 0);
                        o[nb][d] += z;
                    }
                }
            }
        }
    }
    // column of o[.][d][e] in the lane's row
    __device__ __forceinline__ static int column(int d, int e, int quad) { return 16 * d + 4 * quad + e; }
};
template <typename ST, int NB, int KB> struct PagedTile<bf16, ST, NB, KB> : PagedTile16<bf16, ST, NB, KB> {};
template <int NB, int KB> struct PagedTile<float, e4m3, NB, KB> : PagedTile16<float, e4m3, NB, KB> {};

// ---- float32 products ------------------------------------------------------------------------------------------------
template <int NB, int KB>
struct PagedTile<float, float, NB, KB> {
    static constexpr bool kCodes = false, kOnce = NB < 2, kStagedK = true;
    static constexpr int kStage = 16 * KB * kD * 4;
    static constexpr int kVecs = 4;
    u32x4 k[KB][kVecs];
    f32x4 v[KB][4];              // four numbers of a row of V
    float q[NB][16];
    f32x4 o[NB][4];
    f32x4 w[KB][4];              // V without what is masked
    uint32_t k_at[kVecs], wr[kVecs], nat[kVecs], v_at[4];

    __device__ __forceinline__ void init(const PagedArgs &a, uint32_t stage, int lane) {
        const int l16 = lane & 15, quad = lane >> 4;
#pragma unroll
        for (int e = 0; e < kVecs; ++e) {
            // rows quad + 4 e in 16 pieces, piece c of row r at c ^ r: what 16 lanes write or read is in distinct banks
            const int r = quad + 4 * e;
            k_at[e] = r * a.kp.s + 16 * l16;
            wr[e] = stage + r * kD * 4 + ((l16 ^ r) * 16);
            nat[e] = stage + l16 * kD * 4 + (((4 * e + quad) ^ l16) * 16);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) v_at[e] = (4 * quad + e) * a.vp.s + 16 * l16;
    }
    __device__ __forceinline__ void load_q(int nb, const float *row, bool there, int quad) {
#pragma unroll
        for (int t = 0; t < 16; t += 4) {
            const f32x4 x = *reinterpret_cast<const f32x4 *>(row + 4 * t + 4 * quad);
#pragma unroll
            for (int e = 0; e < 4; ++e) q[nb][t + e] = there ? x[e] : 0.0f;
        }
#pragma unroll
        for (int d = 0; d < 4; ++d) o[nb][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    __device__ __forceinline__ void load_k(int blk, const char *kb, const char *, uint32_t mask) {
#pragma unroll
        for (int s = 0; s < kVecs; ++s) k[blk][s] = load16<kOnce>(kb + lane_offset(k_at[s], mask));
    }
    __device__ __forceinline__ void load_v(int blk, const char *vb, const char *, uint32_t mask) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[blk][e] = __builtin_bit_cast(f32x4, load16<kOnce>(vb + lane_offset(v_at[e], mask)));
    }
    __device__ __forceinline__ void stage_k() const {
#pragma unroll
        for (int blk = 0; blk < KB; ++blk)
#pragma unroll
            for (int i = 0; i < kVecs; ++i) *reinterpret_cast<__attribute__((address_space(3))) u32x4 *>((uintptr_t)(wr[i] + 16 * blk * kD * 4)) = k[blk][i];
    }
    __device__ __forceinline__ void logits(f32x4 (&s)[NB][KB]) const {
#pragma unroll
        for (int blk = 0; blk < KB; ++blk) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) s[nb][blk] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            u32x4 f[kVecs];
#pragma unroll
            for (int t = 0; t < kVecs; ++t) f[t] = lds_load128(nat[t], 16 * blk * kD * 4);
#pragma unroll
            for (int t = 0; t < 16; ++t)
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
                    s[nb][blk] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(f[t >> 2][t & 3]), q[nb][t], s[nb][blk], 0, 0, 0);
        }
    }
    __device__ __forceinline__ bool stage_v(bool edge, bool several, int first, int last, unsigned there, int lane) {
        bool odd = false;
#pragma unroll
        for (int blk = 0; blk < KB; ++blk)
#pragma unroll
            for (int e = 0; e < 4; ++e) w[blk][e] = v[blk][e];
        if (edge) {
#pragma unroll
            for (int blk = 0; blk < KB; ++blk)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = 16 * blk + 4 * (lane >> 4) + e;
                    const bool in = r >= first && r < last && (there >> blk & 1);
#pragma unroll
                    for (int d = 0; d < 4; ++d) {
                        const float x = in ? w[blk][e][d] : 0.0f;
                        const bool bad = several && (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u;
                        odd = odd || bad;
                        w[blk][e][d] = bad ? 0.0f : x;
                    }
                }
        }
        return odd;
    }
    __device__ __forceinline__ void product(const f32x4 (&s)[NB][KB]) {
#pragma unroll
        for (int blk = 0; blk < KB; ++blk)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int d = 0; d < 4; ++d)
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) o[nb][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[blk][e][d], s[nb][blk][e], o[nb][d], 0, 0, 0);
    }
    __device__ __forceinline__ static int column(int d, int e, int quad) { return 16 * quad + 4 * e + d; }
};

// Eight columns of a finished row: weights' sum l and products `acc` relative to the maximum `top`, the sink not yet among them.  `none`: no
// query, or no key that it sees.
template <typename T>
__device__ __forceinline__ void paged_finish(const PagedArgs &a, int b, int row, int head, int c8, float sink, bool none, float top, float l, const float (&acc)[8]) {
    const float sink2 = sink * kLog2e;
    // (the larger one's weight is 1 and not the power of a difference with itself, which a fused multiply-add of the logit would not make 0)
    const bool by_sink = sink2 >= top;
    const float ref = by_sink ? sink2 : top, f = by_sink ? fast_exp2(top - sink2) : 1.0f;
    const float z = l * f + (by_sink ? 1.0f : fast_exp2(sink2 - top));
    const float mul = none ? 0.0f : f / z;
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = none ? 0.0f : acc[e] * mul;
    store8(static_cast<T *>(a.o) + b * a.os.b + head * a.os.h + row * a.os.s + c8, x);
    if (c8 == 0 && a.lse) a.lse[((int64_t)b * a.H + head) * a.Sq + row] = none ? sink : (ref + fast_log2(z)) * kLn2;
}

// column blocks and wavefronts that are merged at a time
template <int NB> constexpr int paged_merge_blocks() { return NB == 4 ? 2 : NB; }
template <int NW> constexpr int paged_merge_waves() { return NW < 8 ? NW : 8; }
template <typename T, typename ST, int NB, int NW>
constexpr int paged_lds_bytes() {
    constexpr int merge = paged_merge_waves<NW>() * 16 * paged_merge_blocks<NB>() * kPagedRow * 4;
    constexpr int stages = NW * PagedTile<T, ST, NB, paged_tile_blocks<T, ST, NB, NW>()>::kStage;
    return stages > merge ? stages : merge;
}

// LDS written and read by lanes of one wavefront, which executes these in order: the compiler has to keep that order too.
__device__ __forceinline__ void wave_lds_order() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <typename T, typename ST, int NB, int NW>
__global__ __launch_bounds__(64 * NW, (paged_occupancy<T, ST, NB, NW>())) void attn_paged_kernel(const PagedArgs a) {
    constexpr int kPairs = 16 * NB, KB = paged_tile_blocks<T, ST, NB, NW>(), kKeys = 16 * KB;
    using Tile = PagedTile<T, ST, NB, KB>;
    __shared__ __attribute__((aligned(128))) char smem[paged_lds_bytes<T, ST, NB, NW>()];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, quad = lane >> 4;
    // workgroup -> (slot, KV head), heads next to each other or eight slots (a.across: the heads of a slot then run on one XCD)
    const int line = a.across ? blockIdx.x >> 3 : blockIdx.x, line_slot = a.by_g.quotient(line), g = line - line_slot * a.G;
    const int slot = a.across ? 8 * line_slot + (blockIdx.x & 7) : line_slot;
    PagedSpan sp;
    const PagedShare share = paged_share<kPairs, kKeys>(a, slot, sp);
    if (share.unit < 0) return;
    // the unit's tiles in even parts, the first ones a tile longer where it does not come out even
    const int part_tiles = (int)((uint32_t)sp.tiles / (uint32_t)share.count), longer = sp.tiles - part_tiles * share.count;
    const int t_lo = sp.t_first + part_tiles * share.index + min(share.index, longer), n_wg = part_tiles + (share.index < longer ? 1 : 0);
    const int n_it = n_wg > w ? (n_wg - w + NW - 1) / NW : 0;       // this wavefront's tiles: t_lo + w + NW j
    const int pairs = min(a.Sq * a.r - sp.pair0, kPairs);

    const int32_t *table = a.table + sp.b * a.table_stride;
    const int in_page = (1 << a.page_shift) - 1, weff = a.window ? a.window : 1 << 30;
    int entry[KB];                           // pages of the wavefront's next 64 tiles, one a lane, for each 16 keys of a tile
    auto entries = [&](int j) __attribute__((always_inline)) {
        const int n0 = (t_lo + w + NW * (j + lane)) * kKeys;
#pragma unroll
        for (int blk = 0; blk < KB; ++blk) {
            if (blk && (16 * blk & in_page)) {
                entry[blk] = entry[blk - 1];
            } else {
                const int i = (n0 + 16 * blk) >> a.page_shift;
                int page = -1;
                if (j + lane < n_it && i < a.width) page = table[i];
                entry[blk] = (unsigned)page < (unsigned)a.pages ? page : -1;
            }
        }
    };
    if (n_it > 0) entries(0);

    Tile tile;
    const uint32_t stage = lds_addr(smem) + w * Tile::kStage;
    tile.init(a, stage, lane);
    int pq[NB];                // position of the column's query
    float m[NB], l[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        const bool ok = 16 * nb + l16 < pairs;
        const int pair = sp.pair0 + (ok ? 16 * nb + l16 : 0), row = a.by_r.quotient(pair), head = g * a.r + pair - row * a.r;
        pq[nb] = sp.base + row;
        tile.load_q(nb, static_cast<const T *>(a.q) + sp.b * a.qs.b + head * a.qs.h + row * a.qs.s, ok, quad);
        m[nb] = kLowest;
        l[nb] = 0.0f;
    }

    const char *k_base = a.kp.head(g), *v_base = a.vp.head(g), *ke_base = a.ke.head(g), *ve_base = a.ve.head(g);
    auto page_of = [&](int j, int blk) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(entry[blk], j & 63); };
    // (page, slot) -> load(block, address of the rows, of their exponents); blocks behind the first of a page follow it
    auto fetch = [&](int j, const char *base, const PagedPool &rows, const char *ebase, const PagedPool &exps, auto load) __attribute__((always_inline)) {
        const int n0 = (t_lo + w + NW * j) * kKeys;
        const char *p = nullptr, *e = nullptr;
#pragma unroll
        for (int blk = 0; blk < KB; ++blk) {
            if (blk && (16 * blk & in_page)) {
                p += 16 * (uint64_t)rows.s;
                if constexpr (Tile::kCodes) e += 16 * exps.s;
            } else {
                const int page = max(page_of(j, blk), 0), at = (n0 + 16 * blk) & in_page;
                p = base + rows.at(page, at);
                if constexpr (Tile::kCodes) e = ebase + exps.at(page, at);
            }
            load(blk, p, e);
        }
    };
    auto fetch_k = [&](int j, uint32_t mask) __attribute__((always_inline)) { fetch(j, k_base, a.kp, ke_base, a.ke, [&](int blk, const char *p, const char *e) { tile.load_k(blk, p, e, mask); }); };
    auto fetch_v = [&](int j, uint32_t mask) __attribute__((always_inline)) { fetch(j, v_base, a.vp, ve_base, a.ve, [&](int blk, const char *p, const char *e) { tile.load_v(blk, p, e, mask); }); };

    if (n_it > 0) {
        fetch_k(0, ~0u);
        fetch_v(0, ~0u);
    }
    const bool several = sp.pos0 != sp.pos1;
    bool odd = false;
    for (int j = 0; j < n_it; ++j) {
        const int n0 = (t_lo + w + NW * j) * kKeys;
        int pages = 0;                       // negative where a block of the tile has no page
        unsigned there = 0;                  // which of them have one
#pragma unroll
        for (int blk = 0; blk < KB; ++blk) {
            pages |= page_of(j, blk);
            there |= page_of(j, blk) >= 0 ? 1u << blk : 0u;
        }
        const bool edge = n0 + kKeys - 1 > sp.pos0 || n0 <= sp.pos1 - weff || pages < 0;
        // The next tile; behind the last one the same loads from one line of it, so that the waits for what is under way can be counted: with a branch
        // around them every tile began with a wait for all of it.
        const int next = min(j + 1, n_it - 1);
        const uint32_t mask = next > j ? ~0u : 0u;
        if ((next & 63) == 0) entries(next);
        f32x4 s[NB][KB];
        if constexpr (Tile::kStagedK) {
            tile.stage_k();
            fetch_k(next, mask);
            wave_lds_order();
            tile.logits(s);
            wave_lds_order();
        } else {
            tile.logits(s);
            fetch_k(next, mask);
        }
        odd = tile.stage_v(edge, several, sp.lo - n0, sp.hi - n0, there, lane) || odd;
        fetch_v(next, mask);
        if (edge) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int blk = 0; blk < KB; ++blk)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int key = n0 + 16 * blk + 4 * quad + e;
                        s[nb][blk][e] = key <= pq[nb] && key > pq[nb] - weff && (there >> blk & 1) ? s[nb][blk][e] : -INFINITY;
                    }
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            float mx = s[nb][0][0];
#pragma unroll
            for (int e = 1; e < 4 * KB; ++e) mx = fast_max(mx, s[nb][e >> 2][e & 3]);
            mx *= a.scale_log2;
            if (__builtin_amdgcn_ballot_w64(mx > m[nb] + kRaise) != 0ull) {
                const float m_new = fast_max(m[nb], quad_max(mx)), alpha = fast_exp2(m[nb] - m_new);
                l[nb] *= alpha;
#pragma unroll
                for (int d = 0; d < 4; ++d) tile.o[nb][d] *= alpha;
                m[nb] = m_new;
            }
            float sum0 = 0.0f, sum1 = 0.0f;
#pragma unroll
            for (int e = 0; e < 4 * KB; ++e) {
                const float p = fast_exp2(fmaf(s[nb][e >> 2][e & 3], a.scale_log2, -m[nb]));
                s[nb][e >> 2][e & 3] = p;
                if (e & 1) sum1 += p;
                else sum0 += p;
            }
            l[nb] += sum0 + sum1;
        }
        wave_lds_order();
        tile.product(s);
        wave_lds_order();
    }

    // Infinities and NaN in a row of V that one query sees and another does not (0 times them is NaN) have been left out of the product.  A weight times
    // infinity is infinity, so they are what is missing: added here to the columns that see them, from the pages, key by key.  (In the loop,
    // whatever form it has, this costs the kernels 15 registers and more.)
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(odd) != 0ull, 0)) {
#pragma unroll 1
        for (int j = 0; j < n_it; ++j) {
            const int n0 = (t_lo + w + NW * j) * kKeys;
            // (in a tile whose keys all queries see nothing has been left out)
            if (n0 + kKeys - 1 <= sp.pos0 && n0 > sp.pos1 - weff && paged_page(a, sp.b, n0) >= 0 && paged_page(a, sp.b, n0 + kKeys - 16) >= 0 &&
                (KB < 4 || (paged_page(a, sp.b, n0 + 16) >= 0 && paged_page(a, sp.b, n0 + 32) >= 0)))
                continue;
#pragma unroll 1
            for (int key = max(n0, sp.lo); key < min(n0 + kKeys, sp.hi); ++key) {
                const int page = paged_page(a, sp.b, key);
                if (page < 0) continue;
                const char *row = v_base + a.vp.at(page, key & in_page);
                float power = 1.0f;
                if constexpr (Tile::kCodes) power = factor_of_byte((uint8_t)ve_base[a.ve.at(page, key & in_page)]);
#pragma unroll
                for (int d = 0; d < 4; ++d)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float x = stored_number(reinterpret_cast<const ST *>(row) + Tile::column(d, e, quad));
                        if constexpr (Tile::kCodes) x *= power;
                        if ((__float_as_uint(x) & 0x7f800000u) != 0x7f800000u) continue;
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb)
                            if (key <= pq[nb] && key > pq[nb] - weff) tile.o[nb][d][e] += x;
                    }
            }
        }
    }

    // ---- merge the wavefronts: rows [wavefront][pair][64 + (m, l)] in LDS ----
    constexpr int kMerge = paged_merge_blocks<NB>(), MW = paged_merge_waves<NW>();
    float *red = reinterpret_cast<float *>(smem);
    if constexpr (NW > MW) {
        // LDS holds half of them: the upper ones hand theirs over first
        static_assert(NW == 2 * MW && NB == 1, "one block of columns, two halves");
        float *row = red + ((w % MW) * 16 + l16) * kPagedRow;
        const float l_tot = quad_sum(l[0]);
        __syncthreads();
        if (w >= MW) {
#pragma unroll
            for (int d = 0; d < 4; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) row[Tile::column(d, e, quad)] = tile.o[0][d][e];
            if (quad == 0) { row[kD] = m[0]; row[kD + 1] = l_tot; }
        }
        __syncthreads();
        if (w < MW) {
            const float top = fast_max(m[0], row[kD]), f = fast_exp2(m[0] - top), f2 = fast_exp2(row[kD] - top);
            l[0] = l[0] * f + (quad == 0 ? f2 * row[kD + 1] : 0.0f);
#pragma unroll
            for (int d = 0; d < 4; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) tile.o[0][d][e] = tile.o[0][d][e] * f + f2 * row[Tile::column(d, e, quad)];
            m[0] = top;
        }
    }
    float *part = a.partial + ((int64_t)(share.first + share.index) * a.G + g) * paged_partial_floats(NB);
#pragma unroll
    for (int h = 0; h < NB / kMerge; ++h) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kMerge; ++i) {
            const int nb = h * kMerge + i;
            float *row = red + (w * 16 * kMerge + 16 * i + l16) * kPagedRow;
            const float l_tot = quad_sum(l[nb]);
            if (NW > MW && w >= MW) continue;
#pragma unroll
            for (int d = 0; d < 4; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) row[Tile::column(d, e, quad)] = tile.o[nb][d][e];
            if (quad == 0) { row[kD] = m[nb]; row[kD + 1] = l_tot; }
        }
        __syncthreads();
        // eight lanes per row, eight columns each
        const int c8 = (tid & 7) * 8;
#pragma unroll
        for (int local = tid >> 3; local < 16 * kMerge; local += 8 * NW) {
            const int mine = h * 16 * kMerge + local;
            if (mine >= pairs) break;
            float top = kLowest, l_all = 0.0f, acc[8];
#pragma unroll
            for (int k = 0; k < MW; ++k) top = fast_max(top, red[(k * 16 * kMerge + local) * kPagedRow + kD]);
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] = 0.0f;
#pragma unroll
            for (int k = 0; k < MW; ++k) {
                const float *row = red + (k * 16 * kMerge + local) * kPagedRow;
                const float f = fast_exp2(row[kD] - top);
                l_all += f * row[kD + 1];
#pragma unroll
                for (int e = 0; e < 8; ++e) acc[e] += f * row[c8 + e];
            }
            if (share.count > 1) {
                *reinterpret_cast<f32x4 *>(part + mine * kD + c8) = f32x4{acc[0], acc[1], acc[2], acc[3]};
                *reinterpret_cast<f32x4 *>(part + mine * kD + c8 + 4) = f32x4{acc[4], acc[5], acc[6], acc[7]};
                if (c8 == 0) { part[kPairs * kD + 2 * mine] = top; part[kPairs * kD + 2 * mine + 1] = l_all; }
            } else {
                const int pair = sp.pair0 + mine, row = a.by_r.quotient(pair), head = g * a.r + pair - row * a.r, pos = sp.base + row;
                paged_finish<T>(a, sp.b, row, head, c8, paged_sink(a, head), pos < 0 || pos >= sp.n || l_all == 0.0f, top, l_all, acc);
            }
        }
    }
    if (a.shares && share.index == 0 && g == 0 && tid == 0) {
        a.plan[2 * share.unit] = share.first;
        a.plan[2 * share.unit + 1] = share.count;
    }
}

// Shares of one (batch row, KV head, pair) row, WR wavefronts per row (one: four rows to a workgroup): lane = (group of shares, 8 columns),
// added in an order that depends on their number only.
template <typename T, int NB, int WR>
__global__ __launch_bounds__(256) void attn_paged_combine_kernel(const PagedArgs a) {
    constexpr int kPairs = 16 * NB, kRows = 4 / WR, kGroups = 8 * WR;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c8 = (lane & 7) * 8;
    // workgroups: kRows pairs of a (batch row, KV head)
    const int per_head = a.Sq * a.r, wgs = (per_head + kRows - 1) / kRows;
    const int bid = a.by_wgs.quotient(blockIdx.x);
    const int pair = (blockIdx.x - bid * wgs) * kRows + (WR == 1 ? w : 0);
    const int b = a.by_g.quotient(bid), g = bid - b * a.G;
    if (pair >= per_head) return;
    const int block = pair / kPairs, slot = pair % kPairs, row = a.by_r.quotient(pair), head = g * a.r + pair - row * a.r;
    const int unit = b * a.blocks + block;
    const int first = a.plan[2 * unit], count = a.plan[2 * unit + 1];
    const float sink = paged_sink(a, head);
    const int n = paged_length(a, b), pos = paged_base(a, b, n) + row;
    if (count == 1) return;
    const float *part = a.partial + ((int64_t)first * a.G + g) * paged_partial_floats(NB);
    const int64_t step = a.G * paged_partial_floats(NB);
    float m = kLowest, l = 0.0f, acc[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = 0.0f;
    for (int s = (WR == 1 ? 0 : 8 * w) + (lane >> 3); s < count; s += kGroups) {
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
    float f = fast_exp2(m - top);
    l *= f;
    l += __shfl_xor(l, 8); l += __shfl_xor(l, 16); l += __shfl_xor(l, 32);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        acc[e] *= f;
        acc[e] += __shfl_xor(acc[e], 8); acc[e] += __shfl_xor(acc[e], 16); acc[e] += __shfl_xor(acc[e], 32);
    }
    if constexpr (WR > 1) {
        __shared__ float red[WR][kPagedRow];
        if (lane < 8) {
#pragma unroll
            for (int e = 0; e < 8; ++e) red[w][c8 + e] = acc[e];
            if (lane == 0) { red[w][kD] = top; red[w][kD + 1] = l; }
        }
        __syncthreads();
        if (w != 0) return;
        float all = kLowest;
#pragma unroll
        for (int k = 0; k < WR; ++k) all = fast_max(all, red[k][kD]);
        l = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = 0.0f;
#pragma unroll
        for (int k = 0; k < WR; ++k) {
            f = fast_exp2(red[k][kD] - all);
            l += f * red[k][kD + 1];
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] += f * red[k][c8 + e];
        }
        top = all;
    }
    if (lane < 8) paged_finish<T>(a, b, row, head, c8, sink, pos < 0 || pos >= n || l == 0.0f, top, l, acc);
}

}  // namespace gptoss
