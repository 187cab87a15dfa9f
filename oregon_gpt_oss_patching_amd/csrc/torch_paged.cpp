// PyTorch operators of the key / value cache in pages (gptoss_attn_paged_* in include/gptoss_attn.h): argument checks, allocation and launch.
//
//   gptoss_attn::paged_write, paged_write_slots, paged_read, paged_fwd      the four library calls; none has a gradient (an operator cannot return None: an
//                                                        empty lse stands for "not requested")
//
// Native for the same reason as attention() (torch_ops.cpp): a decoding step makes two of these calls for each layer, and each takes
// a few microseconds on the GPU.
#include "torch_direct.h"

namespace {

constexpr auto kPairs = at::ScalarType::Float4_e2m1fn_x2;        // two e2m1 numbers to an element

int abi_dtype(at::ScalarType t) {
    return t == at::kFloat ? GPTOSS_ATTN_FP32 : t == at::kBFloat16 ? GPTOSS_ATTN_BF16 : t == at::kFloat8_e4m3fn ? GPTOSS_ATTN_E4M3 : t == kPairs ? GPTOSS_ATTN_E2M1 : -1;
}

void set3(gptoss_attn_strides &s, const Tensor &t) {
    s.b = t.stride(0);
    s.h = t.stride(1);
    s.s = t.stride(2);
}

void require_near(const Tensor &pages, const char *name, const Tensor &t) {
    TORCH_CHECK(t.device() == pages.device(), name, " is on ", t.device(), " but the cache is on ", pages.device(), ": every tensor must be on the cache's GPU");
}

// The parameter block and the tensors it points into.
struct PagedCall {
    gptoss_attn_paged_params p{};
    Tensor table, seqlens, start, sinks, q, k, v, scratch;
};

Tensor lengths_of(const Tensor &t, const Tensor &pages, int64_t batch, const char *name) {
    TORCH_CHECK(t.numel() == batch && is_integers(t), name, " must hold one integer per batch row");
    return int32_on(t, pages).contiguous();
}

// The cache; `dtype`: the model's type.
void fill_cache(PagedCall &c, const Tensor &k_pages, const Tensor &v_pages, const OptTensor &k_exp, const OptTensor &v_exp, at::ScalarType dtype, int64_t batch) {
    TORCH_CHECK(k_pages.is_cuda(), "gptoss attention runs on the GPU only (HIP kernels); the cache is on ", k_pages.device());
    require_near(k_pages, "v of the cache", v_pages);
    const auto storage = k_pages.scalar_type();
    TORCH_CHECK(dtype == at::kBFloat16 || dtype == at::kFloat, "unsupported dtype ", dtype, ": bfloat16 or float32");
    const bool pairs = storage == kPairs, codes = pairs || storage == at::kFloat8_e4m3fn;
    TORCH_CHECK(v_pages.scalar_type() == storage && (storage == dtype || codes), "a cache of ", storage, "/", v_pages.scalar_type(),
                " does not go with tensors of ", dtype, ": it holds their type, float8_e4m3fn or float4_e2m1fn_x2");
    const int64_t row = pairs ? 32 : 64;
    TORCH_CHECK(k_pages.dim() == 4 && k_pages.sizes() == v_pages.sizes() && k_pages.size(3) == row, "the cache's k and v must both be (pages, G, page_size, ", row, "), got ",
                k_pages.sizes(), " and ", v_pages.sizes());
    TORCH_CHECK(k_pages.stride(3) == 1 && v_pages.stride(3) == 1, "the cache's rows of ", row, " must be contiguous, got strides ", k_pages.strides(), " and ", v_pages.strides());
    gptoss_attn_paged_params &p = c.p;
    p.struct_size = sizeof(p);
    p.dtype = abi_dtype(dtype);
    p.storage = abi_dtype(storage);
    if (codes) {
        TORCH_CHECK(k_exp && v_exp, "a ", pairs ? "float4_e2m1fn_x2" : "float8_e4m3fn", " cache needs its exponents");
        for (const auto &[name, t, e] : {std::tuple<const char *, const Tensor &, uint8_t **>("k_exp", *k_exp, &p.k_exp), {"v_exp", *v_exp, &p.v_exp}}) {
            require_near(k_pages, name, t);
            TORCH_CHECK(t.scalar_type() == at::kByte && t.dim() == (pairs ? 4 : 3) && t.sizes().slice(0, 3) == k_pages.sizes().slice(0, 3) &&
                            (!pairs || (t.size(3) == 2 && t.stride(3) == 1)),
                        name, " must be uint8 (pages, G, page_size", pairs ? ", 2), a row's bytes side by side, got " : "), got ", t.scalar_type(), " ", t.sizes());
            *e = const_cast<uint8_t *>(t.const_data_ptr<uint8_t>());
        }
        set3(p.k_exp_stride, *k_exp);
        set3(p.v_exp_stride, *v_exp);
    }
    p.pages = size32(k_pages.size(0));
    p.G = size32(k_pages.size(1));
    p.page_size = size32(k_pages.size(2));
    p.D = 64;
    p.B = size32(batch);
    p.k_pages = const_cast<void *>(k_pages.const_data_ptr());
    p.v_pages = const_cast<void *>(v_pages.const_data_ptr());
    set3(p.k_page_stride, k_pages);
    set3(p.v_page_stride, v_pages);
}

// The cache, the table and what all calls with one have.
void fill(PagedCall &c, const Tensor &k_pages, const Tensor &v_pages, const OptTensor &k_exp, const OptTensor &v_exp, const Tensor &page_table,
          at::ScalarType dtype, int64_t batch) {
    fill_cache(c, k_pages, v_pages, k_exp, v_exp, dtype, batch);
    gptoss_attn_paged_params &p = c.p;
    TORCH_CHECK(page_table.dim() == 2 && page_table.size(0) == batch && is_integers(page_table), "page_table must be (B, pages of a row) integers, got ",
                page_table.sizes(), " for ", batch, " rows");
    c.table = int32_on(page_table, k_pages);
    if (c.table.stride(1) != 1 && c.table.size(1) > 1) c.table = c.table.contiguous();
    p.table_width = size32(c.table.size(1));
    p.table_stride = c.table.stride(0);
    p.page_table = c.table.const_data_ptr<int32_t>();
}

// (float16 is bfloat16 to these calls, which the attention computes with in any case.  Into codes that rounds twice: a number within 2^-9 of itself of the middle between two codes counts as
// that middle, so it may come back 2^-9 of itself further off than from the nearer one; the code's own half step is 2^-4 or 2^-2.)

// Rows (B, G, S, 64) or (B, H, S, 64) as the kernels take them, and their strides; a dimension of one element has a stride that says nothing.  What is laid out
// otherwise is copied (a copy that is one: `contiguous` gives such a tensor back as it is, on whatever address).
Tensor rows_of(const Tensor &t, gptoss_attn_strides &s) {
    const int64_t per16 = 16 / t.element_size();
    s.b = t.size(0) == 1 ? 0 : t.stride(0);
    s.h = t.size(1) == 1 ? 0 : t.stride(1);
    s.s = t.size(2) == 1 ? 64 : t.stride(2);
    if (t.stride(3) == 1 && s.b % per16 == 0 && s.h % per16 == 0 && s.s % per16 == 0 && s.s >= 64 && s.s <= kMaxSeqStride &&
        reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0)
        return t;
    const Tensor r = t.clone(at::MemoryFormat::Contiguous);
    set3(s, r);
    return r;
}

// Tokens (T, G, 64) as a batch row of theirs.
Tensor tokens_of(const Tensor &t, gptoss_attn_strides &s) {
    const int64_t per16 = 16 / t.element_size();
    s.b = 0;
    s.h = t.size(1) == 1 ? 0 : t.stride(1);
    s.s = t.size(0) == 1 ? 64 : t.stride(0);
    if (t.stride(2) == 1 && s.h % per16 == 0 && s.s % per16 == 0 && s.s >= 64 && s.s <= kMaxSeqStride && reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0) return t;
    const Tensor r = t.clone(at::MemoryFormat::Contiguous);
    s.h = r.stride(1);
    s.s = r.stride(0);
    return r;
}

void *stream_of(const Tensor &t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

void paged_write(const Tensor &k_pages, const Tensor &v_pages, const OptTensor &k_exp, const OptTensor &v_exp, const Tensor &k_, const Tensor &v_,
                 const Tensor &page_table, const Tensor &start, const OptTensor &seqlens) {
    const c10::OptionalDeviceGuard guard(k_pages.device());
    TORCH_CHECK(k_.scalar_type() == v_.scalar_type(), "k and v must be of one type, got ", k_.scalar_type(), " and ", v_.scalar_type());
    TORCH_CHECK(k_.dim() == 4 && k_.sizes() == v_.sizes(), "k and v must both be (B, G, S, 64), got ", k_.sizes(), " and ", v_.sizes());
    const bool half = k_.scalar_type() == at::kHalf;
    PagedCall c;
    fill(c, k_pages, v_pages, k_exp, v_exp, page_table, half ? at::kBFloat16 : k_.scalar_type(), k_.size(0));
    TORCH_CHECK(k_.size(1) == c.p.G && k_.size(3) == 64, "k and v must be (B, ", c.p.G, ", S, 64) for this cache, got ", k_.sizes());
    require_near(k_pages, "k", k_);
    require_near(k_pages, "v", v_);
    c.k = rows_of(half ? k_.to(at::kBFloat16) : k_, c.p.k_stride);
    c.v = rows_of(half ? v_.to(at::kBFloat16) : v_, c.p.v_stride);
    c.p.k = const_cast<void *>(c.k.const_data_ptr());
    c.p.v = const_cast<void *>(c.v.const_data_ptr());
    c.p.Sq = size32(k_.size(2));
    c.start = lengths_of(start, k_pages, c.p.B, "start");
    c.p.start = c.start.const_data_ptr<int32_t>();
    if (seqlens) {
        c.seqlens = lengths_of(*seqlens, k_pages, c.p.B, "seqlens");
        c.p.seqlens = c.seqlens.const_data_ptr<int32_t>();
    }
    about_to_write({&k_pages, &v_pages, k_exp ? &*k_exp : nullptr, v_exp ? &*v_exp : nullptr});
    check("gptoss_attn_paged_write", gptoss_attn_paged_write(&c.p, stream_of(k_pages)));
}

// k, v (T, G, 64) to slots of their own.
void paged_write_slots(const Tensor &k_pages, const Tensor &v_pages, const OptTensor &k_exp, const OptTensor &v_exp, const Tensor &k_, const Tensor &v_, const Tensor &slots_) {
    const c10::OptionalDeviceGuard guard(k_pages.device());
    TORCH_CHECK(k_.scalar_type() == v_.scalar_type(), "k and v must be of one type, got ", k_.scalar_type(), " and ", v_.scalar_type());
    TORCH_CHECK(k_.dim() == 3 && k_.sizes() == v_.sizes(), "k and v must both be (T, G, 64), got ", k_.sizes(), " and ", v_.sizes());
    const bool half = k_.scalar_type() == at::kHalf;
    PagedCall c;
    fill_cache(c, k_pages, v_pages, k_exp, v_exp, half ? at::kBFloat16 : k_.scalar_type(), 1);
    TORCH_CHECK(k_.size(1) == c.p.G && k_.size(2) == 64, "k and v must be (T, ", c.p.G, ", 64) for this cache, got ", k_.sizes());
    TORCH_CHECK(slots_.dim() == 1 && slots_.size(0) == k_.size(0) && is_integers(slots_), "slots must hold one integer per token, got ", slots_.scalar_type(), " ", slots_.sizes(),
                " for ", k_.size(0));
    require_near(k_pages, "k", k_);
    require_near(k_pages, "v", v_);
    if (k_.size(0) == 0) return;
    c.k = tokens_of(half ? k_.to(at::kBFloat16) : k_, c.p.k_stride);
    c.v = tokens_of(half ? v_.to(at::kBFloat16) : v_, c.p.v_stride);
    c.p.k = const_cast<void *>(c.k.const_data_ptr());
    c.p.v = const_cast<void *>(c.v.const_data_ptr());
    c.p.Sq = size32(k_.size(0));
    c.start = slots_.scalar_type() == at::kLong && slots_.device() == k_pages.device() ? slots_ : slots_.to(k_pages.device(), at::kLong);
    if (c.start.stride(0) != 1) c.start = c.start.contiguous();
    about_to_write({&k_pages, &v_pages, k_exp ? &*k_exp : nullptr, v_exp ? &*v_exp : nullptr});
    check("gptoss_attn_paged_write_slots", gptoss_attn_paged_write_slots(&c.p, c.start.const_data_ptr<int64_t>(), stream_of(k_pages)));
}

std::tuple<Tensor, Tensor> paged_read(const Tensor &k_pages, const Tensor &v_pages, const OptTensor &k_exp, const OptTensor &v_exp, const Tensor &page_table,
                                      const Tensor &seqlens, int64_t max_len, const OptTensor &start, at::ScalarType dtype) {
    const c10::OptionalDeviceGuard guard(k_pages.device());
    const bool half = dtype == at::kHalf;
    const int64_t batch = seqlens.numel();
    PagedCall c;
    fill(c, k_pages, v_pages, k_exp, v_exp, page_table, half ? at::kBFloat16 : dtype, batch);
    TORCH_CHECK(max_len > 0, "max_len must be positive, got ", max_len);
    c.p.Sq = size32(max_len);
    c.seqlens = lengths_of(seqlens, k_pages, batch, "seqlens");
    c.p.seqlens = c.seqlens.const_data_ptr<int32_t>();
    if (start) {
        c.start = lengths_of(*start, k_pages, batch, "start");
        c.p.start = c.start.const_data_ptr<int32_t>();
    }
    Tensor k = new_tensor({batch, c.p.G, max_len, 64}, half ? at::kBFloat16 : dtype, k_pages), v = new_tensor(k.sizes(), k.scalar_type(), k_pages);
    set3(c.p.k_stride, k);
    set3(c.p.v_stride, v);
    c.p.k = k.data_ptr();
    c.p.v = v.data_ptr();
    check("gptoss_attn_paged_read", gptoss_attn_paged_read(&c.p, stream_of(k_pages)));
    return half ? std::make_tuple(k.to(dtype), v.to(dtype)) : std::make_tuple(k, v);
}

// (lse undefined where it is not asked for)
std::tuple<Tensor, Tensor> attend(const Tensor &q_, const Tensor &k_pages, const Tensor &v_pages, const OptTensor &k_exp, const OptTensor &v_exp,
                                  const Tensor &page_table, const Tensor &seqlens, const OptTensor &start, const OptTensor &sinks, double sm_scale,
                                  int64_t window, int64_t max_len, bool need_lse) {
    const c10::OptionalDeviceGuard guard(k_pages.device());
    TORCH_CHECK(q_.dim() == 4 && q_.size(3) == 64, "q must be (B, H, S, 64), got ", q_.sizes());
    const bool half = q_.scalar_type() == at::kHalf;
    const int64_t b = q_.size(0), h = q_.size(1), s = q_.size(2);
    PagedCall c;
    fill(c, k_pages, v_pages, k_exp, v_exp, page_table, half ? at::kBFloat16 : q_.scalar_type(), b);
    require_near(k_pages, "q", q_);
    gptoss_attn_paged_params &p = c.p;
    c.q = rows_of(half ? q_.to(at::kBFloat16) : q_, p.q_stride);
    p.q = c.q.const_data_ptr();
    p.H = size32(h);
    p.Sq = size32(s);
    TORCH_CHECK(window >= 0 && window <= INT_MAX && max_len >= 0, "the window and max_len must not be negative");
    p.window = static_cast<int32_t>(window);
    p.max_len = static_cast<int32_t>(std::min<int64_t>(max_len, INT_MAX));
    p.scale = static_cast<float>(sm_scale);
    c.seqlens = lengths_of(seqlens, k_pages, b, "seqlens");
    p.seqlens = c.seqlens.const_data_ptr<int32_t>();
    if (start) {
        c.start = lengths_of(*start, k_pages, b, "start");
        p.start = c.start.const_data_ptr<int32_t>();
    }
    p.sinks_dtype = GPTOSS_ATTN_FP32;
    if (sinks) {
        require_near(k_pages, "sinks", *sinks);
        TORCH_CHECK(sinks->numel() == h, "sinks must hold one logit per query head");
        const bool bf16 = sinks->scalar_type() == at::kBFloat16;
        c.sinks = (bf16 || sinks->scalar_type() == at::kFloat ? *sinks : sinks->to(at::kFloat)).contiguous();
        p.sinks_dtype = bf16 ? GPTOSS_ATTN_BF16 : GPTOSS_ATTN_FP32;
        p.sinks = c.sinks.const_data_ptr();
    }
    Tensor o = new_tensor({b, s, h, 64}, c.q.scalar_type(), k_pages);
    Tensor lse = need_lse ? new_tensor({b, h, s}, at::kFloat, k_pages) : Tensor();
    set(p.o_stride, o, true);
    p.o = o.data_ptr();
    p.lse = need_lse ? lse.data_ptr<float>() : nullptr;
    p.scratch_bytes = gptoss_attn_paged_workspace_bytes(&p);
    if (p.scratch_bytes) {
        c.scratch = new_tensor({static_cast<int64_t>(p.scratch_bytes / sizeof(float))}, at::kFloat, k_pages);
        p.scratch = c.scratch.data_ptr();
    }
    check("gptoss_attn_paged_fwd", gptoss_attn_paged_fwd(&p, stream_of(k_pages)));
    return {half ? o.to(at::kHalf) : o, lse};
}

std::tuple<Tensor, Tensor> paged_fwd(const Tensor &q, const Tensor &k_pages, const Tensor &v_pages, const OptTensor &k_exp, const OptTensor &v_exp,
                                     const Tensor &page_table, const Tensor &seqlens, const OptTensor &start, const OptTensor &sinks, double sm_scale,
                                     int64_t window, int64_t max_len, bool need_lse) {
    auto [o, lse] = attend(q, k_pages, v_pages, k_exp, v_exp, page_table, seqlens, start, sinks, sm_scale, window, max_len, need_lse);
    return {o, need_lse ? lse : new_tensor({0}, at::kFloat, o)};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(gptoss_attn, m) {
    m.def("paged_write(Tensor(a!) k_pages, Tensor(b!) v_pages, Tensor(c!)? k_exp, Tensor(d!)? v_exp, Tensor k, Tensor v, Tensor page_table, Tensor start, "
          "Tensor? seqlens) -> ()");
    m.def("paged_write_slots(Tensor(a!) k_pages, Tensor(b!) v_pages, Tensor(c!)? k_exp, Tensor(d!)? v_exp, Tensor k, Tensor v, Tensor slots) -> ()");
    m.def("paged_read(Tensor k_pages, Tensor v_pages, Tensor? k_exp, Tensor? v_exp, Tensor page_table, Tensor seqlens, SymInt max_len, Tensor? start, "
          "ScalarType dtype) -> (Tensor, Tensor)");
    m.def("paged_fwd(Tensor q, Tensor k_pages, Tensor v_pages, Tensor? k_exp, Tensor? v_exp, Tensor page_table, Tensor seqlens, Tensor? start, Tensor? sinks, "
          "float sm_scale, SymInt window, SymInt max_len, bool need_lse=True) -> (Tensor, Tensor)");
}
TORCH_LIBRARY_IMPL(gptoss_attn, CUDA, m) {
    m.impl("paged_write", &paged_write);
    m.impl("paged_write_slots", &paged_write_slots);
    m.impl("paged_read", &paged_read);
    m.impl("paged_fwd", &paged_fwd);
}
#define GPTOSS_PAGED_IMPL(KEY, FN)                                                               \
    TORCH_LIBRARY_IMPL(gptoss_attn, KEY, m) {                                                    \
        for (const char *name : {"paged_write", "paged_write_slots", "paged_read", "paged_fwd"}) \
            m.impl(name, torch::CppFunction::makeFromBoxedFunction<&FN>());                      \
    }
GPTOSS_PAGED_IMPL(Autograd, refuse_gradients)
GPTOSS_PAGED_IMPL(CPU, refuse_cpu)
GPTOSS_PAGED_IMPL(FuncTorchBatched, refuse_vmap)

// ---- the same calls from Python, without the dispatcher ------------------------------------------------------------------
// A decoding step's calls take the GPU 2 to 8 us each, and the host as much, of which 2.4 are a launch.  Where nothing stands between caller and kernel (plain GPU
// tensors, no gradient wanted, no mode, no tracing, no profiler) the dispatcher and the arguments' way onto its stack are not needed: these functions make
// the call, and give NotImplemented where something does, or where arguments are of other types; then it goes through the operator.  us of the host for a call
// from Python, through the operator / so: write 4.25 / 3.45, attention 5.8 / 4.2 (with an empty result less), read 6.2 / 4.75.
namespace {

PyObject *write_now(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 9 || !direct_now()) return not_implemented();
    Arguments a{args};
    const Tensor &k_pages = a.tensor(0), &v_pages = a.tensor(1), &k = a.tensor(4), &v = a.tensor(5), &table = a.tensor(6), &start = a.tensor(7);
    const OptTensor k_exp = a.optional(2), v_exp = a.optional(3), seqlens = a.optional(8);
    if (!a.ok) return not_implemented();
    {
        const pybind11::gil_scoped_release free;
        paged_write(k_pages, v_pages, k_exp, v_exp, k, v, table, start, seqlens);
    }
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

PyObject *write_slots_now(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 7 || !direct_now()) return not_implemented();
    Arguments a{args};
    const Tensor &k_pages = a.tensor(0), &v_pages = a.tensor(1), &k = a.tensor(4), &v = a.tensor(5), &slots = a.tensor(6);
    const OptTensor k_exp = a.optional(2), v_exp = a.optional(3);
    if (!a.ok) return not_implemented();
    {
        const pybind11::gil_scoped_release free;
        paged_write_slots(k_pages, v_pages, k_exp, v_exp, k, v, slots);
    }
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

PyObject *read_now(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 9 || !direct_now()) return not_implemented();
    Arguments a{args};
    const Tensor &k_pages = a.tensor(0), &v_pages = a.tensor(1), &table = a.tensor(4), &seqlens = a.tensor(5);
    const OptTensor k_exp = a.optional(2), v_exp = a.optional(3), start = a.optional(7);
    const int64_t max_len = a.integer(6);
    const at::ScalarType dtype = a.dtype(8);
    if (!a.ok) return not_implemented();
    Pair out;
    {
        const pybind11::gil_scoped_release free;
        out = paged_read(k_pages, v_pages, k_exp, v_exp, table, seqlens, max_len, start, dtype);
    }
    return pair(out);
    END_HANDLE_TH_ERRORS
}

PyObject *fwd_now(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 13 || !direct_now()) return not_implemented();
    Arguments a{args};
    const Tensor &q = a.tensor(0), &k_pages = a.tensor(1), &v_pages = a.tensor(2), &table = a.tensor(5), &seqlens = a.tensor(6);
    const OptTensor k_exp = a.optional(3), v_exp = a.optional(4), start = a.optional(7), sinks = a.optional(8);
    const double scale = a.number(9);
    const int64_t window = a.integer_or_none(10), max_len = a.integer_or_none(11);
    const bool need_lse = a.truth(12);
    if (!a.ok) return not_implemented();
    Pair out;
    {
        const pybind11::gil_scoped_release free;
        out = attend(q, k_pages, v_pages, k_exp, v_exp, table, seqlens, start, sinks, scale, window, max_len, need_lse);
    }
    return need_lse ? pair(out) : THPVariable_Wrap(std::get<0>(out));
    END_HANDLE_TH_ERRORS
}

PyMethodDef kDirect[] = {
    {"paged_write_now", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(&write_now)), METH_FASTCALL, nullptr},
    {"paged_read_now", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(&read_now)), METH_FASTCALL, nullptr},
    {"paged_fwd_now", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(&fwd_now)), METH_FASTCALL, nullptr},
    {"paged_write_slots_now", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(&write_slots_now)), METH_FASTCALL, nullptr},
};

}  // namespace

// (paged_write, paged_read, paged_fwd, paged_write_slots) for Python
extern "C" PyObject *gptoss_paged_direct() { return functions_of(kDirect); }
