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

PagedPool pool(void *base, const gptoss_attn_strides &s, int eb) { return PagedPool{static_cast<char *>(base), s.h * eb, (uint32_t)(s.b * eb), (uint32_t)(s.s * eb)}; }

// Strides that the kernels keep in 32 bits.
bool pool_fits(const gptoss_attn_strides &s, int eb) { return s.b >= 0 && s.b * eb <= 0xffffffffll && s.s >= 0 && s.s <= (1 << 24); }

PagedArgs make_args(const gptoss_attn_paged_params *p) {
    PagedArgs a{};
    a.q = p->q;
    a.sinks = p->sinks;
    a.o = p->o;
    a.lse = p->lse;
    const int eb = p->storage == GPTOSS_ATTN_E4M3 ? 1 : p->storage == GPTOSS_ATTN_FP32 ? 4 : 2;
    a.kp = pool(p->k_pages, p->k_page_stride, eb);
    a.vp = pool(p->v_pages, p->v_page_stride, eb);
    a.ke = pool(p->k_exp, p->k_exp_stride, 1);
    a.ve = pool(p->v_exp, p->v_exp_stride, 1);
    a.table = p->page_table;
    a.seqlens = p->seqlens;
    a.start = p->start;
    a.k = static_cast<char *>(p->k);
    a.v = static_cast<char *>(p->v);
    a.qs = cvt(p->q_stride); a.os = cvt(p->o_stride); a.ks = cvt(p->k_stride); a.vs = cvt(p->v_stride);
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

// How the attention's work is divided: column blocks of 16 pairs, blocks of pairs of a row, (row, block) units, shares of all units'
// tiles for each KV head that there are at most beside one for each unit (0: units stay whole, each walked by `alone` wavefronts), how many are to be expected, and
// the scratch that takes; `across`: a slot's KV heads on one XCD.  How long shares are is the kernel's to find, from the lengths (PagedShare).
struct PagedDivision { int nb, blocks, shares, usual, alone; bool across; int64_t units; size_t plan_bytes, bytes; };

// Workgroups of four wavefronts that a compute unit runs at a time.
template <typename T, typename ST, int NB> constexpr int per_simd() { return paged_occupancy<T, ST, NB, kPagedWaves>(); }

PagedDivision paged_division(const gptoss_attn_paged_params *p) {
    PagedDivision d{};
    const bool codes = p->storage == GPTOSS_ATTN_E4M3, f32 = p->storage == GPTOSS_ATTN_FP32;      // f32: the fp32 MFMA
    const int64_t r = p->H / p->G, pairs = (int64_t)p->Sq * r;
    const int most = p->dtype == GPTOSS_ATTN_FP32 ? paged_pairs<float>() : paged_pairs<bf16>();
    d.nb = pairs <= 16 ? 1 : pairs <= 32 || most == 32 ? 2 : pairs <= 48 ? 3 : 4;
    const int64_t blocks = (pairs + 16 * d.nb - 1) / (16 * d.nb);
    d.blocks = (int)(blocks < 0x7fffffff ? blocks : 0x7fffffff);
    d.units = blocks * p->B;
    // the most keys that a unit can see
    int64_t keys = (int64_t)p->table_width * p->page_size;
    if (p->max_len > 0 && p->max_len < keys) keys = p->max_len;
    const int64_t queries = (16 * d.nb - 1) / r + 2;                   // that a unit's pairs touch
    if (p->window > 0 && p->window + queries < keys) keys = p->window + queries;
    // Short rows: a workgroup walks a unit alone, as many wavefronts as its keys and the compute unit's share of the workgroups have room for, and
    // there is nothing to add in a second launch.  What counts is what the host knows of the lengths: in a table far wider than the rows, without max_len, these are cut too, 32 x 1000
    // tokens 18.7 and not 15.3, with four queries 23.1 / 15.7, 32 x 2000 in codes 21.8 / 16.0.  Rows of few bytes, and workgroups that fill the chip by themselves, go alone for longer.  us, cut / alone, 64
    // heads on 8 KV heads ("to n": rows of 50 to n tokens):
    //   bfloat16: 1 x 1025 tokens 9.1 / 8.0, but 1 x 1500 9.0 / 11.9; 32 x 1000 18.4 / 14.6, 16 to 1100 10.0 / 10.4, 32 to 2000 14.3 / 16.1; more than a workgroup to a
    //   compute unit: 64 x 2000 48.1 / 43.4, 64 to 2500 22.0 / 22.3, 40 to 3500 19.8 / 23.3
    //   codes: 1 x 1500 9.4 / 9.5, 8 x 1500 12.2 / 10.2, but 4 to 2000 10.1 / 11.5; half a workgroup to a compute unit and more: 16 to 2000 11.8 / 11.2, 32 x 2000 20.5 / 16.2, but
    //   16 to 3500 12.6 / 15.7; more than one: 64 to 3500 21.1 / 18.4, 40 to 3500 17.0 / 17.2, 40 to 4500 17.9 / 20.4
    //   four queries a row (four wavefronts): 3 to 800 10.2 / 10.1, 3 to 1000 10.3 / 11.4, 32 x 500 16.3 / 9.4; 16 to 1000 11.4 / 10.9, 16 to 1300 12.9 / 13.2; 64 to 2000 24.9 / 20.2, 40 to
    //   3000 22.4 / 23.5
    //   32 bits: 1 x 300 10.2 / 9.6, 8 x 300 11.0 / 9.9, but 1 x 500 10.4 / 11.6; 128 x 500 on two KV heads 21.7 / 16.4
    const int64_t wgs = d.units * p->G;
    const bool full = wgs > (f32 ? 128 : 256), half = wgs >= 128;
    d.alone = d.nb > 1 || keys <= 128 || wgs > (f32 ? 256 : 512) ? kPagedWaves : f32 || full || keys <= 256 ? 8 : 16;
    const int most_alone = f32 ? (full ? 576 : 288) : d.nb > 1 ? (full ? 2304 : half ? 1152 : 832) : codes ? (full ? 3456 : half ? 2304 : 1536) : full ? 2304 : 1152;
    if (d.units > kPagedMaxUnits || keys <= most_alone) return d;
    d.alone = kPagedWaves;
    // As many workgroups as a 256-CU part holds at a time: they start and end together.  A unit's last share is half of one on average; at
    // least half of the workgroups are shares all the same, so that a long row among many is cut.  No more than the units can have.  us with half as many,
    // as many, twice as many: 16 x 8192 tokens 46.3 / 47.5 / 50.1, 64 x 3540 73.9 / 77.4 / 80.3, but 64 rows of 150 to 16384 103 / 81.6 / 83.5, 32 of 6000 to
    // 16384 137 / 112 / 114, and four queries on each of those in e4m3 44.3 / 33.4 / 41.2.
#define GPTOSS_HELD(T, NB) (codes ? per_simd<T, e4m3, NB>() : per_simd<T, T, NB>())
    const int at_a_time = p->dtype == GPTOSS_ATTN_FP32 ? (d.nb == 1 ? GPTOSS_HELD(float, 1) : GPTOSS_HELD(float, 2))
                           : d.nb == 1 ? GPTOSS_HELD(bf16, 1) : d.nb == 2 ? GPTOSS_HELD(bf16, 2) : d.nb == 3 ? GPTOSS_HELD(bf16, 3) : GPTOSS_HELD(bf16, 4);
#undef GPTOSS_HELD
    const int64_t held = 256 * at_a_time / p->G, left = held - d.units / 2, can = d.units * ((keys + 127) / 128);
    int64_t shares = left > held / 2 ? left : held / 2;
    if (shares > can) shares = can;
    d.shares = shares > 1 ? (int)shares : 1;
    // (of rows as long as can be, in shares of 128 to 384 keys)
    const int64_t per_cu = (wgs * ((keys + 127) / 128) + 255) / 256, least = 128 * (per_cu < 3 ? per_cu : 3), usual = d.units * ((keys + least - 1) / least);
    d.usual = usual < shares ? (int)usual : d.shares;
    // The exponents of a page's KV heads share cache lines, which the heads' workgroups then read from one L2.  us, heads next to each other / on one
    // XCD, e4m3: 32 rows of 6000 to 16384 tokens 65.4 / 63.5, 24 of 150 to 30000 37.1 / 35.1, 200 of up to 4000 67.5 / 64.1; but 8 of up to 6000 14.5 / 15.4,
    // and in bfloat16 200 rows 102 / 106.
    d.across = codes && p->B * keys >= 1 << 17;
    d.plan_bytes = ((size_t)d.units * 2 * sizeof(int) + 15) & ~(size_t)15;
    d.bytes = d.plan_bytes + (size_t)(d.shares + d.units) * p->G * paged_partial_floats(d.nb) * sizeof(float);
    return d;
}

template <typename T, typename ST, int NB>
int attend(const PagedDivision &d, void *stream, PagedArgs &a) {
    if constexpr (NB == 1) {
        if constexpr (sizeof(ST) < 4)
            if (d.alone == 16) return launch(attn_paged_kernel<T, ST, NB, 16>, d.units * a.G, 1024, stream, a);
        if (d.alone == 8) return launch(attn_paged_kernel<T, ST, NB, 8>, d.units * a.G, 512, stream, a);
    }
    const int64_t slots = d.shares + d.units;
    a.across = d.across;
    const int s = launch(attn_paged_kernel<T, ST, NB, kPagedWaves>, (a.across ? (slots + 7) / 8 * 8 : slots) * a.G, 64 * kPagedWaves, stream, a);
    if (s || !d.shares) return s;
    // A wavefront adds eight shares at a time; four of them for each row where a unit has more than that and rows are few, or more than twice that (us: 1 x 65536
    // tokens 32.7 / 28.7, 1 x 1300 8.6 / 8.3, 8 of 700 to 6000 15.3 / 15.0; with eight shares a unit 16 x 8192 47.3 / 47.9, five queries on those eight rows 19.3 / 21.9).
    const int64_t heads = (int64_t)a.B * a.G, pairs = (int64_t)a.Sq * a.r;
    const bool many = d.usual > (heads * pairs <= 512 ? 8 : 16) * d.units;
    const int64_t wgs = many ? pairs : (pairs + 3) / 4;
    a.by_wgs = div_by(wgs);
    return many ? launch(attn_paged_combine_kernel<T, NB, 4>, heads * wgs, 256, stream, a) : launch(attn_paged_combine_kernel<T, NB, 1>, heads * wgs, 256, stream, a);
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
    if (!pool_fits(p->k_page_stride, codes ? 1 : eb) || !pool_fits(p->v_page_stride, codes ? 1 : eb)) return GPTOSS_ATTN_ERR_STRIDE;
    if (codes && (!pool_fits(p->k_exp_stride, 1) || !pool_fits(p->v_exp_stride, 1))) return GPTOSS_ATTN_ERR_STRIDE;
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
    if (!aligned(p->lse, 4) || !aligned(p->scratch, 16)) return GPTOSS_ATTN_ERR_ALIGNMENT;
    if (p->scratch_bytes < gptoss_attn_paged_workspace_bytes(p) || (!p->scratch && gptoss_attn_paged_workspace_bytes(p))) return GPTOSS_ATTN_ERR_WORKSPACE;
    return GPTOSS_ATTN_OK;
}

size_t gptoss_attn_paged_workspace_bytes(const gptoss_attn_paged_params *p) {
    if (!p || p->B <= 0 || p->G <= 0 || p->H <= 0 || p->H % p->G || p->Sq <= 0 || p->table_width <= 0 || p->page_size <= 0) return 0;
    return paged_division(p).bytes;
}

int gptoss_attn_paged_fwd(const gptoss_attn_paged_params *p, void *stream) {
    const int rc = gptoss_attn_paged_validate(p, kFwd);
    if (rc) return rc;
    PagedArgs a = make_args(p);
    const PagedDivision d = paged_division(p);
    if (d.units > 0x7fffffff || (int64_t)a.Sq * a.r > (1 << 30)) return GPTOSS_ATTN_ERR_SHAPE;
    a.blocks = d.blocks;
    a.units = (int)d.units;
    a.shares = d.shares;
    a.by_r = div_by(a.r);
    a.by_g = div_by(a.G);
    a.by_blocks = div_by(a.blocks);
    if (d.shares) {
        a.plan = static_cast<int *>(p->scratch);
        a.partial = reinterpret_cast<float *>(static_cast<char *>(p->scratch) + d.plan_bytes);
    }
    const bool codes = p->storage == GPTOSS_ATTN_E4M3;
    if (p->dtype == GPTOSS_ATTN_BF16) {
#define GPTOSS_PAGED(NB) (codes ? attend<bf16, e4m3, NB>(d, stream, a) : attend<bf16, bf16, NB>(d, stream, a))
        return d.nb == 1 ? GPTOSS_PAGED(1) : d.nb == 2 ? GPTOSS_PAGED(2) : d.nb == 3 ? GPTOSS_PAGED(3) : GPTOSS_PAGED(4);
#undef GPTOSS_PAGED
    }
#define GPTOSS_PAGED(NB) (codes ? attend<float, e4m3, NB>(d, stream, a) : attend<float, float, NB>(d, stream, a))
    return d.nb == 1 ? GPTOSS_PAGED(1) : GPTOSS_PAGED(2);
#undef GPTOSS_PAGED
}

int gptoss_attn_paged_write(const gptoss_attn_paged_params *p, void *stream) {
    const int rc = gptoss_attn_paged_validate(p, kWrite);
    if (rc) return rc;
    PagedArgs a = make_args(p);
    const int64_t rows = (int64_t)a.Sq * a.G;
    if (rows > (1 << 30)) return GPTOSS_ATTN_ERR_SHAPE;
    const int64_t blocks = (rows + 31) / 32, grid = blocks * a.B;
    a.blocks = (int)blocks;
    a.by_blocks = div_by(blocks);
    a.by_g = div_by(a.G);
    const bool codes = p->storage == GPTOSS_ATTN_E4M3;
    if (p->dtype == GPTOSS_ATTN_BF16)
        return codes ? launch(paged_write_kernel<bf16, true>, grid, 256, stream, a) : launch(paged_write_kernel<bf16, false>, grid, 256, stream, a);
    return codes ? launch(paged_write_kernel<float, true>, grid, 256, stream, a) : launch(paged_write_kernel<float, false>, grid, 256, stream, a);
}

int gptoss_attn_paged_read(const gptoss_attn_paged_params *p, void *stream) {
    const int rc = gptoss_attn_paged_validate(p, kRead);
    if (rc) return rc;
    PagedArgs a = make_args(p);
    const int64_t blocks = ((int64_t)a.Sq + 31) / 32, grid = blocks * a.G * a.B;
    if ((int64_t)a.G * a.B > 0x7fffffff) return GPTOSS_ATTN_ERR_SHAPE;
    a.blocks = (int)blocks;
    a.by_blocks = div_by(blocks);
    a.by_g = div_by(a.G);
    const bool codes = p->storage == GPTOSS_ATTN_E4M3;
    if (p->dtype == GPTOSS_ATTN_BF16)
        return codes ? launch(paged_read_kernel<bf16, e4m3>, grid, 256, stream, a) : launch(paged_read_kernel<bf16, bf16>, grid, 256, stream, a);
    return codes ? launch(paged_read_kernel<float, e4m3>, grid, 256, stream, a) : launch(paged_read_kernel<float, float>, grid, 256, stream, a);
}

}  // extern "C"
