// C ABI of the rotary positions (declared in include/gptoss_attn.h): argument checks and launch.
#include <hip/hip_runtime.h>

#include "../../include/gptoss_attn.h"
#include "rotary.h"

using namespace gptoss;

namespace {

bool on(const void *p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

Strides cvt(const gptoss_attn_strides &s) { return Strides{s.b, s.h, s.s}; }

// Whether rows at `p` with strides `s` (elements of `eb` bytes) all start on boundaries of `n` bytes.
bool rows_on(const void *p, const gptoss_attn_strides &s, int eb, int n) {
    return on(p, n) && s.b * eb % n == 0 && s.h * eb % n == 0 && s.s * eb % n == 0;
}

template <typename T, int V>
const void *kernel_of(bool paired, bool tables) {
    if (paired) return tables ? reinterpret_cast<const void *>(rotary_kernel<T, V, true, true>) : reinterpret_cast<const void *>(rotary_kernel<T, V, true, false>);
    return tables ? reinterpret_cast<const void *>(rotary_kernel<T, V, false, true>) : reinterpret_cast<const void *>(rotary_kernel<T, V, false, false>);
}

}  // namespace

extern "C" {

int gptoss_attn_rotary_validate(const gptoss_attn_rotary_params *p) {
    if (!p) return GPTOSS_ATTN_ERR_NULL_PARAMS;
    if (p->struct_size != sizeof(gptoss_attn_rotary_params)) return GPTOSS_ATTN_ERR_ABI;
    if (p->dtype != GPTOSS_ATTN_BF16 && p->dtype != GPTOSS_ATTN_FP32) return GPTOSS_ATTN_ERR_DTYPE;
    if (p->H <= 0 || p->G <= 0 || p->H > (1 << 20) || p->G > (1 << 20)) return GPTOSS_ATTN_ERR_HEADS;
    if (p->B <= 0 || p->S <= 0) return GPTOSS_ATTN_ERR_SHAPE;
    if (p->D <= 0 || p->D > 256 || p->R <= 0 || p->R > p->D || p->R % 2) return GPTOSS_ATTN_ERR_HEAD_DIM;
    const int eb = p->dtype == GPTOSS_ATTN_FP32 ? 4 : 2;
    for (const void *t : {p->q, p->k, static_cast<const void *>(p->q_out), static_cast<const void *>(p->k_out)}) {
        if (!t) return GPTOSS_ATTN_ERR_NULL_TENSOR;
        if (!on(t, eb)) return GPTOSS_ATTN_ERR_ALIGNMENT;
    }
    const bool tables = p->cos_table || p->sin_table;
    if (tables ? !p->cos_table || !p->sin_table || p->positions || p->frequencies : !p->positions || !p->frequencies) return GPTOSS_ATTN_ERR_NULL_TENSOR;
    if (tables) {
        if (p->table_dtype != GPTOSS_ATTN_BF16 && p->table_dtype != GPTOSS_ATTN_FP32) return GPTOSS_ATTN_ERR_DTYPE;
        const int tb = p->table_dtype == GPTOSS_ATTN_FP32 ? 4 : 2;
        if (!on(p->cos_table, tb) || !on(p->sin_table, tb)) return GPTOSS_ATTN_ERR_ALIGNMENT;
    } else {
        if (p->position_bytes != 4 && p->position_bytes != 8) return GPTOSS_ATTN_ERR_DTYPE;
        if (!on(p->positions, p->position_bytes) || !on(p->frequencies, 8)) return GPTOSS_ATTN_ERR_ALIGNMENT;
    }
    // (token, chunk) pairs are counted in 31 bits, one number to a chunk at worst
    if ((int64_t)p->B * p->S > 0x7fffffffll / p->D) return GPTOSS_ATTN_ERR_SHAPE;
    return GPTOSS_ATTN_OK;
}

int gptoss_attn_rotary(const gptoss_attn_rotary_params *p, void *stream) {
    const int rc = gptoss_attn_rotary_validate(p);
    if (rc) return rc;
    RotaryArgs a{};
    a.q = p->q; a.k = p->k; a.q_out = p->q_out; a.k_out = p->k_out;
    a.positions = p->positions; a.frequencies = p->frequencies;
    a.cos = p->cos_table; a.sin = p->sin_table;
    a.qs = cvt(p->q_stride); a.ks = cvt(p->k_stride); a.qo = cvt(p->q_out_stride); a.ko = cvt(p->k_out_stride);
    a.pos_b = p->position_stride_b; a.pos_s = p->position_stride_s;
    a.cos_b = p->cos_stride_b; a.cos_s = p->cos_stride_s;
    a.sin_b = p->sin_stride_b; a.sin_s = p->sin_stride_s;
    a.H = p->H; a.heads = p->H + p->G; a.D = p->D; a.R = p->R; a.S = p->S;
    a.wide = p->position_bytes == 8;
    a.f32_tables = p->table_dtype == GPTOSS_ATTN_FP32;
    a.inverse = p->inverse != 0;
    a.scale = (float)p->scale;
    const bool f32 = p->dtype == GPTOSS_ATTN_FP32, paired = p->interleaved != 0, tables = p->cos_table != nullptr;
    // The widest access that divides the turned and the other part and that all rows start on.
    const int eb = f32 ? 4 : 2;
    auto wide = [&](int v) {
        return p->R / 2 % v == 0 && (p->D - p->R) % v == 0 && rows_on(p->q, p->q_stride, eb, v * eb) && rows_on(p->k, p->k_stride, eb, v * eb) &&
               rows_on(p->q_out, p->q_out_stride, eb, v * eb) && rows_on(p->k_out, p->k_out_stride, eb, v * eb);
    };
    const int v = wide(16 / eb) ? 16 / eb : wide(2) ? 2 : 1;
    a.pairs = p->R / 2 / v;
    const int tb = a.f32_tables ? 4 : 2, piece = v * tb < 16 ? v * tb : 16;
    a.whole_tables = on(p->cos_table, piece) && on(p->sin_table, piece) && a.cos_b * tb % piece == 0 && a.cos_s * tb % piece == 0 && a.sin_b * tb % piece == 0 &&
                     a.sin_s * tb % piece == 0;
    a.chunks = a.pairs + (p->D - p->R) / v;
    const int64_t lines = (int64_t)p->B * p->S;
    // Heads of a token that a thread walks: up to four, whose numbers are under way together, as soon as that leaves 65536 threads.  us, 64 and 8 heads in bfloat16, one / four /
    // eight: 1000 tokens 7.3 / 5.8 / 5.8, 4096 19 / 13.5 / 15.3, 16384 - / 55.4 / 58.4 (5.5 TB/s; a large copy 5.0).
    int64_t walk = lines * a.chunks * a.heads / 65536;
    walk = walk < 1 ? 1 : walk > 4 ? 4 : walk;
    a.slots = (int)((a.heads + walk - 1) / walk);
    while (lines * a.chunks * a.slots > 0x7fffffff) a.slots = (a.slots + 1) / 2;        // (one slot fits: the check above)
    a.items = lines * a.chunks * a.slots;
    a.by_chunks = div_by(a.chunks);
    // Threads next to each other take heads of a token, or tokens of a head where these lie closer, as the attention's gradients do: 16384 tokens of those 73.4 / 58.9 us, 4096
    // 13.7 / 13.4 (four rows of 8192 120.7 / 128.8).  Of rows of one token the next token is the next row's, and the stride from token to token says nothing; us, heads of a token / tokens of a
    // head as a projection leaves them, 64 and 8 heads: 256 rows 4.0 / 4.0, 512 4.8 / 5.2, 2048 9.9 / 9.2, 8192 29.3 / 30.2, 8 and 2 heads: 8192 7.3 / 7.1.
    a.along_tokens = p->q_stride.h > (p->S > 1 ? p->q_stride.s : p->q_stride.b);
    a.inner = a.along_tokens ? (int)lines : a.slots;
    a.by_inner = div_by(a.inner);
    a.by_s = div_by(p->S);
    const void *kernel = f32 ? (v == 4 ? kernel_of<float, 4>(paired, tables) : v == 2 ? kernel_of<float, 2>(paired, tables) : kernel_of<float, 1>(paired, tables))
                             : (v == 8 ? kernel_of<bf16, 8>(paired, tables) : v == 2 ? kernel_of<bf16, 2>(paired, tables) : kernel_of<bf16, 1>(paired, tables));
    void *args[] = {&a};
    const hipError_t e = hipLaunchKernel(kernel, dim3((unsigned)((a.items + kRotaryThreads - 1) / kRotaryThreads)), dim3(kRotaryThreads), args, 0, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? GPTOSS_ATTN_OK : static_cast<int>(e);
}

}  // extern "C"
