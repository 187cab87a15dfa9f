// Whose page is whose (gptoss_attn_page_table_update) and where the tokens of a call go (gptoss_attn_token_map): whole numbers only.
//
// What bounds both: latencies.  A decoding step's update reads some ten thousand entries and writes a dozen; what it takes is a launch and a chain of
// dependent loads and barriers, so it is one workgroup with its counts and the pool's bits in LDS, and no list of free pages is kept
// from call to call: a page is free iff no row's kept entry names it.
#pragma once
#include "paged_common.h"

namespace gptoss {

constexpr int kTableRows = 16384;                  // rows of a call: a number of 32 bits each in LDS
constexpr int kTableThreads = 1024;
constexpr int kPoolBits = 1 << 19;                 // pages that are looked at together: 64 KB of LDS
constexpr int kPoolGroup = 64 * 32;                // pages of a wavefront's word each
constexpr uint32_t kMany = (1u << 30) + 1;         // sums stay here: more than there are pages or tokens

struct TableArgs {
    int32_t *table;
    const int32_t *have, *want;                    // update; start and counts of the map
    int32_t *seqlens, *left;
    int32_t *row, *position, *first, *used;        // map
    int64_t *slot;
    int64_t stride;
    int B, width, pages, page_shift, total;
    int row_threads_shift;                         // update: 2^this threads read a row's entries
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

// ends[i] = value(0) + ... + value(i) for i < n, by all THREADS; `part`: a number for each wavefront.  Ends with a barrier.
template <int THREADS, typename F>
__device__ __forceinline__ void block_sums(uint32_t *ends, uint32_t *part, int n, F value) {
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    uint32_t before = 0;
    for (int i0 = 0; i0 < n; i0 += THREADS) {
        const uint32_t x = wave_scan_up(i0 + tid < n ? min(value(i0 + tid), kMany) : 0u);
        if (lane == 63) part[w] = x;
        __syncthreads();
        uint32_t mine = before;
        for (int k = 0; k < THREADS / 64; ++k) {
            const uint32_t p = part[k];
            mine = k < w ? add_up(mine, p) : mine;
            before = add_up(before, p);
        }
        if (i0 + tid < n) ends[i0 + tid] = add_up(mine, x);
        __syncthreads();
    }
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

// Bits of the pages lo .. lo + kPoolBits - 1 that rows keep.  Ends with a barrier.
__device__ __forceinline__ void mark_kept(const TableArgs &a, uint32_t *bits, int lo, int words) {
    constexpr int kAtOnce = 16;                    // loads under way
    for (int i = threadIdx.x; i < words; i += kTableThreads) bits[i] = 0;
    __syncthreads();
    const int n = 1 << a.row_threads_shift, lane = threadIdx.x & (n - 1);
    for (int b = threadIdx.x >> a.row_threads_shift; b < a.B; b += kTableThreads >> a.row_threads_shift) {
        const RowPages r = row_pages(a, b);
        const int kept = min(r.has, r.wants);
        const int32_t *row = a.table + b * a.stride;
        for (int i0 = lane; i0 < kept; i0 += kAtOnce * n) {
            int page[kAtOnce];
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) page[k] = i0 + k * n < kept ? row[i0 + k * n] : -1;
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) {
                const int at = page[k] - lo;
                if (page[k] >= 0 && page[k] < a.pages && at >= 0 && at < kPoolBits) atomicOr(bits + (at >> 5), 1u << (at & 31));
            }
        }
    }
    __syncthreads();
}

__global__ __launch_bounds__(kTableThreads) void page_table_update_kernel(const TableArgs a) {
    __shared__ uint32_t ends[kTableRows], bits[kPoolBits / 32], base[kPoolBits / kPoolGroup], part[kTableThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
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
        uint32_t all = 0;
        if (w == 0) {
            for (int g0 = 0; g0 < groups; g0 += 64) {
                const uint32_t x = g0 + lane < groups ? base[g0 + lane] : 0u, incl = wave_scan_up(x);
                if (g0 + lane < groups) base[g0 + lane] = all + incl - x;
                all += (uint32_t)__builtin_amdgcn_readlane((int)incl, 63);
            }
            if (lane == 0) part[0] = all;
        }
        __syncthreads();
        all = part[0];
        __syncthreads();
        return all;
    };
    auto span_of = [&](int lo) { return min(a.pages - lo, kPoolBits); };
    uint32_t free = 0;
    for (int lo = 0; lo < a.pages; lo += kPoolBits) {        // (pages <= 2^30: lo stays below 2^31)
        mark_kept(a, bits, lo, (span_of(lo) + 31) / 32);
        free += count(lo, span_of(lo));
    }
    // Rows in their order: whoever's demand, with those in front of it, passes what is free gets nothing, nor does any behind it that wants pages.
    const bool enough = demand <= free;
    const int served_rows = enough ? a.B : first_above(ends, a.B, free);
    const uint32_t given = enough ? demand : served_rows ? ends[served_rows - 1] : 0u;
    uint32_t before = 0;
    for (int lo = 0; lo < a.pages && before < given; lo += kPoolBits) {
        uint32_t here = free;
        if (a.pages > kPoolBits) {                 // (otherwise the bits are there)
            mark_kept(a, bits, lo, (span_of(lo) + 31) / 32);
            here = count(lo, span_of(lo));
        }
        const int span = span_of(lo), groups = (span + kPoolGroup - 1) / kPoolGroup;
        for (int g = w; g < groups; g += kTableThreads / 64) {
            const uint32_t from = before + base[g];
            if (from >= given) break;
            const int first = g * kPoolGroup + 32 * lane, there = min(max(span - first, 0), 32);
            uint32_t set = there ? ~bits[first >> 5] & (~0u >> (32 - there)) : 0u;
            const uint32_t number = __popc(set);
            uint32_t rank = from + wave_scan_up(number) - number;
            if (!set || rank >= given) continue;
            int b = first_above(ends, a.B, rank);
            while (set && rank < given) {
                while (ends[b] <= rank) ++b;
                const RowPages r = row_pages(a, b);
                const uint32_t row_first = b ? ends[b - 1] : 0u;
                // (the row's pages that this word holds)
                int32_t *to = a.table + b * a.stride + r.has;
                do {
                    const int bit = __ffs(set) - 1;
                    set &= set - 1;
                    to[rank - row_first] = lo + first + bit;
                    ++rank;
                } while (set && rank < ends[b]);
            }
        }
        before += here;
        __syncthreads();
    }
    for (int b = tid; b < a.B; b += kTableThreads) {
        const RowPages r = row_pages(a, b);
        a.seqlens[b] = max(r.fits && (r.wants <= r.has || ends[b] <= free) ? a.want[b] : a.have[b], 0);
    }
    if (tid == 0) *a.left = (int32_t)(free - given);
    // what rows give back
    const int n = 1 << a.row_threads_shift, l = tid & (n - 1);
    for (int b = tid >> a.row_threads_shift; b < a.B; b += kTableThreads >> a.row_threads_shift) {
        const RowPages r = row_pages(a, b);
        for (int i = r.wants + l; i < r.has; i += n) a.table[b * a.stride + i] = -1;
    }
}

// Tokens t = kMapTokens blockIdx.x + ... of a call that has counts[b] of each row, back to back.
constexpr int kMapThreads = 256, kMapTokens = 1024;
__global__ __launch_bounds__(kMapThreads) void token_map_kernel(const TableArgs a) {
    __shared__ uint32_t ends[kTableRows], part[kMapThreads / 64];
    block_sums<kMapThreads>(ends, part, a.B, [&](int b) __attribute__((always_inline)) { return (uint32_t)max(a.want[b], 0); });
    const uint32_t all = ends[a.B - 1], used = min(all, (uint32_t)a.total);
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.used = (int32_t)used;
#pragma unroll
    for (int k = 0; k < kMapTokens / kMapThreads; ++k) {
        const int t = blockIdx.x * kMapTokens + k * kMapThreads + threadIdx.x;
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
}

}  // namespace gptoss
