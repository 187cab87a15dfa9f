// C ABI of the key / value cache in pages (declared in include/gptoss_attn.h): argument checks and launches.
#include <hip/hip_runtime.h>

#include "../../include/gptoss_attn.h"
#include "attn_paged.h"
#include "paged_cache.h"

using namespace gptoss;

namespace {

enum Call { kFwd = 0, kWrite = 1, kRead = 2 };

bool aligned(const void *p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Rows of 64 elements of `eb` bytes, each on a 16-byte boundary.
int check_rows(const void *p, const gptoss_attn_strides &s, int eb) {
    if (!p) return GPTOSS_ATTN_ERR_NULL_TENSOR;
    const int64_t per16 = 16 / eb;
    if (!aligned(p, 16) || s.b % per16 || s.h % per16 || s.s % per16) return GPTOSS_ATTN_ERR_ALIGNMENT;
    return s.s < kD || s.s > (1 << 24) ? GPTOSS_ATTN_ERR_STRIDE : GPTOSS_ATTN_OK;
}

Strides cvt(const gptoss_attn_strides &s) { return Strides{s.b, s.h, s.s}; }

PagedArgs make_args(const gptoss_attn_paged_params *p) {
    PagedArgs a{};
    a.q = p->q;
    a.sinks = p->sinks;
    a.o = p->o;
    a.lse = p->lse;
    a.k_pages = static_cast<char *>(p->k_pages);
    a.v_pages = static_cast<char *>(p->v_pages);
    a.k_exp = p->k_exp;
    a.v_exp = p->v_exp;
    a.table = p->page_table;
    a.seqlens = p->seqlens;
    a.start = p->start;
    a.k = static_cast<char *>(p->k);
    a.v = static_cast<char *>(p->v);
    a.qs = cvt(p->q_stride); a.os = cvt(p->o_stride); a.ks = cvt(p->k_stride); a.vs = cvt(p->v_stride);
    a.kps = cvt(p->k_page_stride); a.vps = cvt(p->v_page_stride); a.kes = cvt(p->k_exp_stride); a.ves = cvt(p->v_exp_stride);
    a.table_stride = p->table_stride;
    a.B = p->B; a.H = p->H; a.G = p->G; a.Sq = p->Sq;
    a.r = p->H > 0 ? p->H / p->G : 0;
    a.pages = p->pages;
    a.page_shift = __builtin_ctz((unsigned)p->page_size);
    a.width = p->table_width;
    a.window = p->window;
    a.scale_log2 = p->scale * kLog2e;
    a.sinks_bf16 = p->sinks_dtype == GPTOSS_ATTN_BF16;
    return a;
}

// One launch; a launch that fails reports its own status.
template <typename Kernel>
int launch(Kernel kernel, int64_t workgroups, int threads, void *stream, const PagedArgs &a) {
    if (workgroups <= 0 || workgroups > 0x7fffffff) return GPTOSS_ATTN_ERR_SHAPE;
    void *args[] = {const_cast<PagedArgs *>(&a)};
    const hipError_t e = hipLaunchKernel(reinterpret_cast<const void *>(kernel), dim3((unsigned)workgroups), dim3((unsigned)threads), args, 0,
                                         static_cast<hipStream_t>(stream));
    return e == hipSuccess ? GPTOSS_ATTN_OK : static_cast<int>(e);
}

}  // namespace

extern "C" {

int gptoss_attn_paged_validate(const gptoss_attn_paged_params *p, int call) {
    if (!p) return GPTOSS_ATTN_ERR_NULL_PARAMS;
    if (p->struct_size != sizeof(gptoss_attn_paged_params)) return GPTOSS_ATTN_ERR_ABI;
    if (p->dtype != GPTOSS_ATTN_BF16 && p->dtype != GPTOSS_ATTN_FP32) return GPTOSS_ATTN_ERR_DTYPE;
    if (p->storage != p->dtype && p->storage != GPTOSS_ATTN_E4M3) return GPTOSS_ATTN_ERR_DTYPE;
    if (p->D != kD) return GPTOSS_ATTN_ERR_HEAD_DIM;
    if (p->G <= 0 || (call == kFwd && (p->H <= 0 || p->H % p->G))) return GPTOSS_ATTN_ERR_HEADS;
    if (p->B <= 0 || p->Sq <= 0 || p->Sq > (1 << 30)) return GPTOSS_ATTN_ERR_SHAPE;
    if (p->pages <= 0 || p->table_width <= 0 || p->table_stride < 0 || p->page_size < 16 || p->page_size > 1024 || (p->page_size & (p->page_size - 1)) ||
        (int64_t)p->table_width * p->page_size > (1 << 30))
        return GPTOSS_ATTN_ERR_PAGES;
    const int eb = p->dtype == GPTOSS_ATTN_FP32 ? 4 : 2;
    const bool codes = p->storage == GPTOSS_ATTN_E4M3;
    int rc;
    if ((rc = check_rows(p->k_pages, p->k_page_stride, codes ? 1 : eb))) return rc;
    if ((rc = check_rows(p->v_pages, p->v_page_stride, codes ? 1 : eb))) return rc;
    if (!p->page_table || (codes && (!p->k_exp || !p->v_exp))) return GPTOSS_ATTN_ERR_NULL_TENSOR;
    if (!aligned(p->page_table, 4) || !aligned(p->seqlens, 4) || !aligned(p->start, 4)) return GPTOSS_ATTN_ERR_ALIGNMENT;
    if (call == kWrite ? !p->start : !p->seqlens) return GPTOSS_ATTN_ERR_NULL_TENSOR;
    if (call != kFwd) {
        if ((rc = check_rows(p->k, p->k_stride, eb))) return rc;
        return check_rows(p->v, p->v_stride, eb);
    }
    if (p->sinks_dtype != GPTOSS_ATTN_FP32 && p->sinks_dtype != GPTOSS_ATTN_BF16) return GPTOSS_ATTN_ERR_DTYPE;
    if (p->window < 0 || p->window > (1 << 30) || p->max_len < 0 || !(p->scale > 0.0f) || !(p->scale < 3.0e38f)) return GPTOSS_ATTN_ERR_SHAPE;
    if ((rc = check_rows(p->q, p->q_stride, eb))) return rc;
    if ((rc = check_rows(p->o, p->o_stride, eb))) return rc;
    if (!p->lse) return GPTOSS_ATTN_ERR_NULL_TENSOR;
    if (!aligned(p->scratch, 16)) return GPTOSS_ATTN_ERR_ALIGNMENT;
    if (p->scratch_bytes < gptoss_attn_paged_workspace_bytes(p) || (!p->scratch && gptoss_attn_paged_workspace_bytes(p))) return GPTOSS_ATTN_ERR_WORKSPACE;
    return GPTOSS_ATTN_OK;
}

size_t gptoss_attn_paged_workspace_bytes(const gptoss_attn_paged_params *) { return 0; }

int gptoss_attn_paged_fwd(const gptoss_attn_paged_params *p, void *stream) {
    const int rc = gptoss_attn_paged_validate(p, kFwd);
    if (rc) return rc;
    const PagedArgs a = make_args(p);
    const int64_t grid = (int64_t)a.B * a.H * a.Sq;
    if (p->dtype == GPTOSS_ATTN_BF16)
        return p->storage == GPTOSS_ATTN_E4M3 ? launch(attn_paged_kernel<bf16, e4m3>, grid, 256, stream, a) : launch(attn_paged_kernel<bf16, bf16>, grid, 256, stream, a);
    return p->storage == GPTOSS_ATTN_E4M3 ? launch(attn_paged_kernel<float, e4m3>, grid, 256, stream, a) : launch(attn_paged_kernel<float, float>, grid, 256, stream, a);
}

int gptoss_attn_paged_write(const gptoss_attn_paged_params *p, void *stream) {
    const int rc = gptoss_attn_paged_validate(p, kWrite);
    if (rc) return rc;
    PagedArgs a = make_args(p);
    const int64_t blocks = ((int64_t)a.Sq * a.G + 31) / 32;
    if (blocks * a.B > 0x7fffffff || (int64_t)a.Sq * a.G > 0x7fffffff - 32) return GPTOSS_ATTN_ERR_SHAPE;
    a.blocks = (int)blocks;
    if (p->dtype == GPTOSS_ATTN_BF16)
        return p->storage == GPTOSS_ATTN_E4M3 ? launch(paged_write_kernel<bf16, true>, blocks * a.B, 256, stream, a) : launch(paged_write_kernel<bf16, false>, blocks * a.B, 256, stream, a);
    return p->storage == GPTOSS_ATTN_E4M3 ? launch(paged_write_kernel<float, true>, blocks * a.B, 256, stream, a) : launch(paged_write_kernel<float, false>, blocks * a.B, 256, stream, a);
}

int gptoss_attn_paged_read(const gptoss_attn_paged_params *p, void *stream) {
    const int rc = gptoss_attn_paged_validate(p, kRead);
    if (rc) return rc;
    PagedArgs a = make_args(p);
    const int64_t blocks = ((int64_t)a.Sq + 31) / 32;
    if (blocks * a.G * a.B > 0x7fffffff) return GPTOSS_ATTN_ERR_SHAPE;
    a.blocks = (int)blocks;
    const int64_t grid = blocks * a.G * a.B;
    if (p->dtype == GPTOSS_ATTN_BF16)
        return p->storage == GPTOSS_ATTN_E4M3 ? launch(paged_read_kernel<bf16, e4m3>, grid, 256, stream, a) : launch(paged_read_kernel<bf16, bf16>, grid, 256, stream, a);
    return p->storage == GPTOSS_ATTN_E4M3 ? launch(paged_read_kernel<float, e4m3>, grid, 256, stream, a) : launch(paged_read_kernel<float, float>, grid, 256, stream, a);
}

}  // extern "C"
