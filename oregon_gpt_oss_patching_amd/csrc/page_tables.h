// Whose page is whose (gptoss_attn_page_table_update) and where the tokens of a call go (gptoss_attn_token_map): whole numbers only.
//
// No list of free pages is kept from call to call: a page is free iff no row's kept entry names it, so each update reads all of them.  What bounds it is not their bytes but latencies, and the
// LDS atomics that set a bit for each (some 1.3 a cycle).  A workgroup has all counts and the pool's bits in LDS; where a table may be large, others set the bits first, each of its
// share of the entries, in a launch of its own.  What is given out goes to sixteen workgroups, 1024 pages at a time, each of which makes the same counts: they read kept entries, lengths and bits,
// and write others.  us: 256 rows of 40 to 9000 tokens 10.6, 3 of them the first launch; 96 of up to 16384 of which 32 begin (8284 pages) 11.3, by one workgroup 28.6; 4096 of 500
// 18.4; 8 of 1000, in one launch, 4.9.
#pragma once
#include "paged_common.h"

namespace gptoss {

constexpr int kTableRows = 16384;                  // rows of a call: a number of 32 bits each in LDS
constexpr int kTableThreads = 1024;
constexpr int kMarkers = 16;                       // workgroups that set bits in a launch of their own
constexpr int kGivers = 16;                        // workgroups that give pages out (4, 8, 32 for the 8284 above: 15.3, 13.3, 11.3 us)
constexpr int kPoolBits = 1 << 19;                 // pages that are looked at together: 64 KB of LDS
constexpr int kPoolGroup = 64 * 32;                // pages of a wavefront's word each
constexpr uint32_t kMany = (1u << 30) + 1;         // sums stay here: more than there are pages or tokens

struct TableArgs {
    int32_t *table;
    const int32_t *have, *want;                    // update; start and counts of the map
    int32_t *seqlens, *left;
    int32_t *row, *position, *first, *used;        // map
    int64_t *slot;
    uint32_t *marks;                               // update: the bits that page_table_mark_kernel has set, or NULL
    int64_t stride;
    int B, width, pages, page_shift, total;
};

__device__ __forceinline__ uint32_t add_up(uint32_t x, uint32_t y) { return min(x + y, kMany); }      // (2 kMany is below 2^32)

// add_up over the lanes up to this one
__device__ __forceinline__ uint32_t wave_scan_up(uint32_t x) {
    x = add_up(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xf, 0xf, false));      // row_shr:1
    x = add_up(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xf, 0xf, false));
    x = add_up(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xf, 0xf, false));
    x = add_up(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xf, 0xf, false));
    x = add_up(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xa, 0xf, false));      // row_bcast:15 into rows 1 and 3
    x = add_up(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xc, 0xf, false));      // row_bcast:31 into rows 2 and 3
    return x;
}

// ends[i] = value(0) + ... + value(i) for i < n, by all THREADS, EACH numbers a thread at a time; `part`: a number for each wavefront.  Ends with a barrier.
template <int THREADS, int EACH, typename F>
__device__ __forceinline__ void sums_of(uint32_t *ends, uint32_t *part, int n, F value) {
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    uint32_t before = 0;
    for (int i0 = 0; i0 < n; i0 += EACH * THREADS) {
        uint32_t x[EACH];
#pragma unroll
        for (int k = 0; k < EACH; ++k) x[k] = i0 + EACH * tid + k < n ? min(value(i0 + EACH * tid + k), kMany) : 0u;
#pragma unroll
        for (int k = 1; k < EACH; ++k) x[k] = add_up(x[k], x[k - 1]);
        const uint32_t incl = wave_scan_up(x[EACH - 1]);
        if (lane == 63) part[w] = incl;
        __syncthreads();
        // what stands in front of the thread's: earlier rounds, wavefronts and lanes (sums that stay at kMany come to kMany here too)
        uint32_t mine = before;
        for (int k = 0; k < THREADS / 64; ++k) {
            const uint32_t p = part[k];
            mine = k < w ? add_up(mine, p) : mine;
            before = add_up(before, p);
        }
        const uint32_t lower = (uint32_t)__shfl_up((int)incl, 1);
        mine = add_up(mine, lane ? lower : 0u);
#pragma unroll
        for (int k = 0; k < EACH; ++k)
            if (i0 + EACH * tid + k < n) ends[i0 + EACH * tid + k] = add_up(mine, x[k]);
        __syncthreads();
    }
}
// (four at a time where one each would take several rounds: 4096 rows 4.5 us, so 2.9; one round 1.0 and 1.5)
template <int THREADS, typename F>
__device__ __forceinline__ void block_sums(uint32_t *ends, uint32_t *part, int n, F value) {
    if (n <= THREADS) sums_of<THREADS, 1>(ends, part, n, value);
    else sums_of<THREADS, 4>(ends, part, n, value);
}

// The first i < n with ends[i] > x, n where there is none.
__device__ __forceinline__ int first_above(const uint32_t *ends, int n, uint32_t x) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (ends[mid] > x) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

struct RowPages { int has, wants; bool fits; };     // entries now and then, 0 .. width; fits: what it wants is not more than the table holds
__device__ __forceinline__ RowPages row_pages(const TableArgs &a, int b) {
    const int64_t up = (1 << a.page_shift) - 1;
    const int64_t has = (max(a.have[b], 0) + up) >> a.page_shift, wants = (max(a.want[b], 0) + up) >> a.page_shift;
    return RowPages{(int)min(has, (int64_t)a.width), (int)min(wants, (int64_t)a.width), wants <= a.width};
}

// Lanes that read a run of a row's entries, sixteen each, and how many runs rows of a table have: where they have one of sixteen lanes at most, four rows to a wavefront.
constexpr int kMarkEach = 16;
__host__ __device__ __forceinline__ int mark_lanes(int width) { return width <= 16 * kMarkEach ? 16 : 64; }
__host__ __device__ __forceinline__ int mark_runs(int width) { return (width + kMarkEach * mark_lanes(width) - 1) / (kMarkEach * mark_lanes(width)); }

// Bits of the pages lo .. lo + kPoolBits - 1 that rows keep: runs in turn among the `waves` of which this is number `wave` (4096 rows
// of 500 tokens with a wavefront each 34.6 us in all, so 18.6).  `bits` of LDS, zeros already; ends with a barrier.
__device__ __forceinline__ void mark_kept(const TableArgs &a, uint32_t *bits, int lo, int wave, int waves) {
    constexpr int kEach = kMarkEach;
    const int lanes = mark_lanes(a.width), lane = threadIdx.x & (lanes - 1), per_wave = 64 / lanes;
    const int runs = mark_runs(a.width), groups = waves * per_wave, group = wave * per_wave + (threadIdx.x & 63) / lanes;
    int b = group / runs, run = group - b * runs;
    const int rows_on = groups / runs, runs_on = groups - rows_on * runs;
    while (b < a.B) {
        const RowPages r = row_pages(a, b);
        const int first = run * kEach * lanes + lane, kept = min(r.has, r.wants);
        const int32_t *row = a.table + b * a.stride;
        int page[kEach];
#pragma unroll
        for (int k = 0; k < kEach; ++k) page[k] = first + k * lanes < kept ? row[first + k * lanes] : -1;
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            const uint32_t at = (uint32_t)page[k] - (uint32_t)lo;                // (pages in front of lo come to 2^31 and more)
            if (page[k] >= 0 && page[k] < a.pages && at < (uint32_t)kPoolBits) atomicOr(bits + (at >> 5), 1u << (at & 31));
        }
        b += rows_on;
        run += runs_on;
        if (run >= runs) { run -= runs; ++b; }
    }
    __syncthreads();
}

__device__ __forceinline__ void clear_bits(uint32_t *bits, int words) {
    for (int i = threadIdx.x; i < words; i += kTableThreads) bits[i] = 0;
    __syncthreads();
}

// The bits of a share of the kept entries, to a.marks + blockIdx.x * words.
__global__ __launch_bounds__(kTableThreads) void page_table_mark_kernel(const TableArgs a) {
    __shared__ uint32_t bits[kPoolBits / 32];
    const int words = (a.pages + 31) / 32;
    clear_bits(bits, words);
    mark_kept(a, bits, 0, __builtin_amdgcn_readfirstlane(blockIdx.x * (kTableThreads / 64) + (threadIdx.x >> 6)), kMarkers * (kTableThreads / 64));
    uint32_t *out = a.marks + (int64_t)blockIdx.x * words;
    for (int i = threadIdx.x; i < words; i += kTableThreads) out[i] = bits[i];
}

__global__ __launch_bounds__(kTableThreads) void page_table_update_kernel(const TableArgs a) {
    __shared__ uint32_t ends[kTableRows], bits[kPoolBits / 32], base[kPoolBits / kPoolGroup + 1], fresh[kTableThreads], part[kTableThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    block_sums<kTableThreads>(ends, part, a.B, [&](int b) __attribute__((always_inline)) {
        const RowPages r = row_pages(a, b);
        return r.fits && r.wants > r.has ? (uint32_t)(r.wants - r.has) : 0u;
    });
    const uint32_t demand = ends[a.B - 1];
    // The free pages of `span` pages from lo on: of each group the number of those before it (base), and in all.
    auto count = [&](int lo, int span) __attribute__((always_inline)) {
        const int groups = (span + kPoolGroup - 1) / kPoolGroup;
        for (int g = w; g < groups; g += kTableThreads / 64) {
            const int first = g * kPoolGroup + 32 * lane, there = min(max(span - first, 0), 32);
            const uint32_t free = there ? ~bits[first >> 5] & (~0u >> (32 - there)) : 0u;
            const uint32_t incl = wave_scan_up(__popc(free));
            if (lane == 63) base[g] = incl;
        }
        __syncthreads();
        if (w == 0) {
            uint32_t all = 0;
            for (int g0 = 0; g0 < groups; g0 += 64) {
                const uint32_t x = g0 + lane < groups ? base[g0 + lane] : 0u, incl = wave_scan_up(x);
                if (g0 + lane < groups) base[g0 + lane] = all + incl - x;
                all += (uint32_t)__builtin_amdgcn_readlane((int)incl, 63);
            }
            if (lane == 0) base[groups] = all;
        }
        __syncthreads();
        return base[groups];
    };
    auto span_of = [&](int lo) { return min(a.pages - lo, kPoolBits); };
    auto mark = [&](int lo) __attribute__((always_inline)) {
        const int words = (span_of(lo) + 31) / 32;
        if (a.marks) {                             // (the pool is one part then)
            for (int i = tid; i < words; i += kTableThreads) {
                uint32_t x[kMarkers];
#pragma unroll
                for (int k = 0; k < kMarkers; ++k) x[k] = a.marks[k * words + i];
#pragma unroll
                for (int k = 1; k < kMarkers; ++k) x[0] |= x[k];
                bits[i] = x[0];
            }
            __syncthreads();
        } else {
            clear_bits(bits, words);
            mark_kept(a, bits, lo, w, kTableThreads / 64);
        }
    };
    uint32_t free = 0;
    for (int lo = 0; lo < a.pages; lo += kPoolBits) {        // (pages <= 2^30: lo stays below 2^31)
        mark(lo);
        free += count(lo, span_of(lo));
        __syncthreads();
    }
    // Rows in their order: whoever's demand, with those in front of it, passes what is free gets nothing, nor does any behind it that wants pages.
    uint32_t given = demand;
    if (demand > free) {
        const int served = first_above(ends, a.B, free);
        given = served ? ends[served - 1] : 0u;
    }
    uint32_t before = 0;
    for (int lo = 0; lo < a.pages && before < given; lo += kPoolBits) {
        uint32_t here = free;
        if (a.pages > kPoolBits) {                 // (otherwise the bits are there)
            mark(lo);
            here = count(lo, span_of(lo));
        }
        const int span = span_of(lo), groups = (span + kPoolGroup - 1) / kPoolGroup;
        const uint32_t end = min(before + here, given);
        // A page for each thread at a time, into LDS by its rank; who gets a rank is found in the sums.
        for (uint32_t c0 = before + blockIdx.x * kTableThreads; c0 < end; c0 += gridDim.x * kTableThreads) {
            const uint32_t c1 = min(c0 + kTableThreads, end);
            for (int g = w; g < groups; g += kTableThreads / 64) {
                if (before + base[g + 1] <= c0 || before + base[g] >= c1) continue;
                const int first = g * kPoolGroup + 32 * lane, there = min(max(span - first, 0), 32);
                uint32_t set = there ? ~bits[first >> 5] & (~0u >> (32 - there)) : 0u;
                const uint32_t number = __popc(set);
                uint32_t rank = before + base[g] + wave_scan_up(number) - number;
                for (; set; set &= set - 1, ++rank)
                    if (rank >= c0 && rank < c1) fresh[rank - c0] = (uint32_t)(lo + first + __ffs(set) - 1);
            }
            __syncthreads();
            if (c0 + tid < c1) {
                const int b = first_above(ends, a.B, c0 + tid);
                a.table[b * a.stride + row_pages(a, b).has + (c0 + tid - (b ? ends[b - 1] : 0u))] = (int32_t)fresh[tid];
            }
            __syncthreads();
        }
        before += here;
    }
    if (tid == 0 && blockIdx.x == 0) *a.left = (int32_t)(free - given);
    for (int b0 = (blockIdx.x * (kTableThreads / 64) + w) * 64; b0 < a.B; b0 += gridDim.x * kTableThreads) {
        const int b = b0 + lane;
        RowPages r{0, 0, true};
        if (b < a.B) {
            r = row_pages(a, b);
            a.seqlens[b] = max(r.fits && (r.wants <= r.has || ends[b] <= free) ? a.want[b] : a.have[b], 0);
        }
        // what rows give back, the wavefront's one after the other
        unsigned long long back = __builtin_amdgcn_ballot_w64(r.has > r.wants);
        while (back) {
            const int l = __builtin_ctzll(back), has = __builtin_amdgcn_readlane(r.has, l), wants = __builtin_amdgcn_readlane(r.wants, l);
            back &= back - 1;
            for (int i = wants + lane; i < has; i += 64) a.table[(int64_t)(b0 + l) * a.stride + i] = -1;
        }
    }
}

// Tokens of a call that has counts[b] of each row, back to back: one to a thread (two, four: what a token waits for adds up, 96 rows of 132000 tokens 3.9 us, so 4.4, 5.7; 1024 rows of one
// 4.0, 4.8, 7.1; only a million tokens of 1000 rows 11.8, 10.4, 10.4).  ROWS: sums that LDS has room for, with few of them more workgroups run at a time: 270000 tokens 4.6 and not 6.7 us.
constexpr int kMapThreads = 256, kMapFewRows = 2048;
template <int ROWS>
__global__ __launch_bounds__(kMapThreads) void token_map_kernel(const TableArgs a) {
    __shared__ uint32_t ends[ROWS], part[kMapThreads / 64];
    block_sums<kMapThreads>(ends, part, a.B, [&](int b) __attribute__((always_inline)) { return (uint32_t)max(a.want[b], 0); });
    const uint32_t all = ends[a.B - 1], used = min(all, (uint32_t)a.total);
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.used = (int32_t)used;
    const int t = blockIdx.x * kMapThreads + threadIdx.x;
    if (t >= a.total) return;
    int row = -1, position = 0, first = (int)used;
    int64_t slot = -1;
    if ((uint32_t)t < used) {
        row = first_above(ends, a.B, (uint32_t)t);
        first = row ? (int)ends[row - 1] : 0;
        const int64_t at = (int64_t)a.have[row] + (t - first);
        position = (int)min(at, (int64_t)0x7fffffff);
        const int64_t entry = at >> a.page_shift;
        if (at >= 0 && entry < a.width) {
            const int page = a.table[row * a.stride + entry];
            if (page >= 0) slot = ((int64_t)page << a.page_shift) + (at & ((1 << a.page_shift) - 1));
        }
    }
    a.row[t] = row;
    a.position[t] = position;
    a.first[t] = first;
    a.slot[t] = slot;
}

}  // namespace gptoss
