// Attention of new queries over a key / value cache in pages (gptoss_attn_paged_fwd).
#pragma once
#include "paged_common.h"

namespace gptoss {

// One (batch row, query head, query) per workgroup: eight lanes a key, 32 keys at a time, each group of eight with a running maximum
// and sum of its own, joined at the end.  A key that the query does not see is not read.
template <typename T, typename ST>
__global__ __launch_bounds__(256) void attn_paged_kernel(const PagedArgs a) {
    __shared__ float red[32][kD + 2];
    int64_t bid = blockIdx.x;
    const int i = (int)(bid % a.Sq); bid /= a.Sq;
    const int head = (int)(bid % a.H), b = (int)(bid / a.H), g = head / a.r;
    const int grp = threadIdx.x >> 3, c8 = (threadIdx.x & 7) * 8;
    const int n = paged_length(a, b);
    const int64_t pos64 = (a.start ? (int64_t)a.start[b] : (int64_t)n - a.Sq) + i;
    const int pos = pos64 >= 0 && pos64 < n ? (int)pos64 : -1;
    float q[8], o[8], m = kLowest, l = 0.0f;
    load8(static_cast<const T *>(a.q) + b * a.qs.b + head * a.qs.h + i * a.qs.s + c8, q);
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = 0.0f;
    for (int j = (a.window ? max(0, pos - a.window + 1) : 0) + grp; j <= pos; j += 32) {
        const int page = paged_page(a, b, j);
        if (page < 0) continue;
        float k[8], v[8];
        load8(reinterpret_cast<const ST *>(a.k_pages) + slot_offset(a.kps, page, g, j, a.page_shift) + c8, k);
        load8(reinterpret_cast<const ST *>(a.v_pages) + slot_offset(a.vps, page, g, j, a.page_shift) + c8, v);
        float fk = a.scale_log2, fv = 1.0f;
        if constexpr (sizeof(ST) == 1) {
            fk = exp_of_byte(a.k_exp[slot_offset(a.kes, page, g, j, a.page_shift)]);
            fv = exp_of_byte(a.v_exp[slot_offset(a.ves, page, g, j, a.page_shift)]);
        }
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf(q[e], k[e], s);
        s += __shfl_xor(s, 1); s += __shfl_xor(s, 2); s += __shfl_xor(s, 4);
        s *= fk;
        if constexpr (sizeof(ST) == 1) s *= a.scale_log2;
        const float mn = fmaxf(m, s), f = fast_exp2(m - mn), p = fast_exp2(s - mn);
        l = l * f + p;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = o[e] * f + p * (v[e] * fv);
        m = mn;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) red[grp][c8 + e] = o[e];
    if (c8 == 0) { red[grp][kD] = m; red[grp][kD + 1] = l; }
    __syncthreads();
    if (threadIdx.x >= kD) return;
    const float sink2 = paged_sink(a, head) * kLog2e;
    float top = fmaxf(sink2, kLowest), l_all = 0.0f, x = 0.0f;
    for (int k = 0; k < 32; ++k) top = fmaxf(top, red[k][kD]);
    for (int k = 0; k < 32; ++k) {
        const float f = fast_exp2(red[k][kD] - top);
        l_all += f * red[k][kD + 1];
        x += f * red[k][threadIdx.x];
    }
    const float z = l_all + fast_exp2(sink2 - top);      // (0 where the row sees no key and has no sink)
    static_cast<T *>(a.o)[b * a.os.b + head * a.os.h + i * a.os.s + threadIdx.x] = (T)(z == 0.0f ? 0.0f : x / z);
    if (threadIdx.x == 0) a.lse[((int64_t)b * a.H + head) * a.Sq + i] = l_all == 0.0f ? paged_sink(a, head) : (top + fast_log2(z)) * kLn2;
}

}  // namespace gptoss
