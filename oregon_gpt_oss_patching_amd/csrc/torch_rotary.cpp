// PyTorch operators of the rotary positions (gptoss_attn_rotary in include/gptoss_attn.h): argument checks, allocation, launch and the autograd node.
//
//   gptoss_attn::rotary_turn     the library call (opaque to tracing)
//   gptoss_attn::rotary          the differentiable call made of it; its gradient is the call again with the angles' sign turned, so it has one of its own
//
// Angles come from positions and frequencies, or from tables of their cosines and sines.  Results lie as (B, S, heads, D): the layout of the projection in
// front of the call and of its gradient, which then need no copy; the attention takes either layout in the same time (16384 tokens and less, both directions).
#include <c10/core/impl/VirtualGuardImpl.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/variable.h>

#include "torch_direct.h"

namespace {

// Rows with contiguous numbers, and their strides; a dimension of one element has a stride that says nothing.
Tensor heads_of(const Tensor &t, gptoss_attn_strides &s) {
    const Tensor r = t.size(3) == 1 || t.stride(3) == 1 ? t : t.contiguous();
    s.b = r.size(0) == 1 ? 0 : r.stride(0);
    s.h = r.size(1) == 1 ? 0 : r.stride(1);
    s.s = r.size(2) == 1 ? 0 : r.stride(2);
    return r;
}

Tensor new_heads(const Tensor &like, gptoss_attn_strides &s) {
    const int64_t b = like.size(0), h = like.size(1), n = like.size(2), d = like.size(3);
    s.b = n * h * d;
    s.h = d;
    s.s = h * d;
    return Tensor(at::detail::empty_strided_cuda({b, h, n, d}, {s.b, s.h, s.s, 1}, like.scalar_type(), like.device()));
}

Pair turn(const Tensor &q_, const Tensor &k_, const OptTensor &positions, const OptTensor &frequencies, const OptTensor &cos, const OptTensor &sin, double scale,
          bool interleaved, bool inverse) {
    TORCH_CHECK(q_.is_cuda(), "gptoss attention runs on the GPU only (HIP kernels); q is on ", q_.device());
    const c10::OptionalDeviceGuard guard(q_.device());
    const auto dtype = q_.scalar_type();
    TORCH_CHECK((dtype == at::kBFloat16 || dtype == at::kFloat || dtype == at::kHalf) && k_.scalar_type() == dtype, "unsupported dtypes ", dtype, "/", k_.scalar_type(),
                ": q and k must both be bfloat16 or both be float32");
    TORCH_CHECK(q_.dim() == 4 && k_.dim() == 4 && q_.size(0) == k_.size(0) && q_.size(2) == k_.size(2) && q_.size(3) == k_.size(3),
                "q must be (B, H, S, D) and k (B, G, S, D), got ", q_.sizes(), " and ", k_.sizes());
    require_on(q_, "k", k_);
    const bool half = dtype == at::kHalf;        // (through float32, which holds it: rounded once all the same)
    const Tensor qh = half ? q_.to(at::kFloat) : q_, kh = half ? k_.to(at::kFloat) : k_;
    const int64_t b = q_.size(0), s = q_.size(2), d = q_.size(3);
    gptoss_attn_rotary_params p{};
    p.struct_size = sizeof(p);
    p.dtype = qh.scalar_type() == at::kFloat ? GPTOSS_ATTN_FP32 : GPTOSS_ATTN_BF16;
    p.B = size32(b);
    p.H = size32(q_.size(1));
    p.G = size32(k_.size(1));
    p.S = size32(s);
    p.D = size32(d);
    p.interleaved = interleaved;
    p.inverse = inverse;
    p.scale = scale;
    Tensor at0, at1;                             // what the block points into
    auto rows = [&](const Tensor &t, const char *name, int64_t &stride_b, int64_t &stride_s) {
        TORCH_CHECK((t.size(0) == b || t.size(0) == 1) && t.size(1) == s, name, " must be of ", b, " rows (or one for all) of ", s, " tokens, got ", t.sizes());
        stride_b = t.size(0) == 1 ? 0 : t.stride(0);
        stride_s = t.size(1) == 1 ? 0 : t.stride(1);
    };
    if (positions) {
        TORCH_CHECK(frequencies && !cos && !sin, "angles come from positions and frequencies, or from cos and sin");
        TORCH_CHECK(is_integers(*positions) && (positions->dim() == 2 || positions->dim() == 1), "positions must be (B, S) or (S) integers, got ", positions->scalar_type(), " ",
                    positions->sizes());
        TORCH_CHECK(frequencies->is_floating_point() && frequencies->dim() == 1, "frequencies must be a floating-point vector, got ", frequencies->scalar_type(), " ",
                    frequencies->sizes());
        at0 = *positions;
        if (at0.device() != q_.device() || (at0.scalar_type() != at::kInt && at0.scalar_type() != at::kLong))
            at0 = at0.to(q_.device(), at0.scalar_type() == at::kInt ? at::kInt : at::kLong);
        if (at0.dim() == 1) at0 = at0.unsqueeze(0);
        rows(at0, "positions", p.position_stride_b, p.position_stride_s);
        at1 = *frequencies;
        if (at1.device() != q_.device() || at1.scalar_type() != at::kDouble) at1 = at1.to(q_.device(), at::kDouble);
        at1 = at1.contiguous();
        p.positions = at0.const_data_ptr();
        p.position_bytes = static_cast<int32_t>(at0.element_size());
        p.frequencies = at1.const_data_ptr<double>();
        p.R = size32(2 * at1.size(0));
    } else {
        TORCH_CHECK(cos && sin && !frequencies, "angles come from positions and frequencies, or from cos and sin");
        TORCH_CHECK(cos->is_floating_point() && sin->is_floating_point() && cos->dim() == 3 && cos->sizes() == sin->sizes(),
                    "cos and sin must both be (B, S, pairs of a head), got ", cos->sizes(), " and ", sin->sizes());
        require_on(q_, "cos", *cos);
        require_on(q_, "sin", *sin);
        const auto type = cos->scalar_type() == at::kBFloat16 && sin->scalar_type() == at::kBFloat16 ? at::kBFloat16 : at::kFloat;
        at0 = cos->scalar_type() == type ? *cos : cos->to(type);
        at1 = sin->scalar_type() == type ? *sin : sin->to(type);
        if (at0.stride(2) != 1) at0 = at0.contiguous();
        if (at1.stride(2) != 1) at1 = at1.contiguous();
        rows(at0, "cos", p.cos_stride_b, p.cos_stride_s);
        rows(at1, "sin", p.sin_stride_b, p.sin_stride_s);
        p.table_dtype = type == at::kBFloat16 ? GPTOSS_ATTN_BF16 : GPTOSS_ATTN_FP32;
        p.cos_table = at0.const_data_ptr();
        p.sin_table = at1.const_data_ptr();
        p.R = size32(2 * at0.size(2));
    }
    TORCH_CHECK(p.R >= 2 && p.R <= d && d <= 256, "pairs of ", p.R, " numbers do not fit heads of ", d, " (at most 256)");
    const Tensor q = heads_of(qh, p.q_stride), k = heads_of(kh, p.k_stride);
    const Tensor qo = new_heads(q, p.q_out_stride), ko = new_heads(k, p.k_out_stride);
    if (b && s) {                                // (no token: nothing to turn)
        p.q = q.const_data_ptr();
        p.k = k.const_data_ptr();
        p.q_out = qo.data_ptr();
        p.k_out = ko.data_ptr();
        check("gptoss_attn_rotary", gptoss_attn_rotary(&p, c10::hip::getCurrentHIPStream(q.device().index()).stream()));
    }
    return half ? Pair(qo.to(dtype), ko.to(dtype)) : Pair(qo, ko);
}

Pair call_turn(const Tensor &q, const Tensor &k, const OptTensor &positions, const OptTensor &frequencies, const OptTensor &cos, const OptTensor &sin, double scale,
               bool interleaved, bool inverse) {
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("gptoss_attn::rotary_turn", "").typed<decltype(call_turn)>();
    return op.call(q, k, positions, frequencies, cos, sin, scale, interleaved, inverse);
}

Pair rotary(const Tensor &, const Tensor &, const OptTensor &, const OptTensor &, const OptTensor &, const OptTensor &, double, bool, bool);

OptTensor optional_of(const Tensor &t) { return t.defined() ? OptTensor(t) : OptTensor(); }
Tensor tensor_of(const OptTensor &t) { return t ? *t : Tensor(); }

struct RotaryFunction : public torch::autograd::Function<RotaryFunction> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext *ctx, const Tensor &q, const Tensor &k, const OptTensor &positions,
                                                  const OptTensor &frequencies, const OptTensor &cos, const OptTensor &sin, double scale, bool interleaved, bool inverse) {
        const at::AutoDispatchBelowADInplaceOrView below;
        auto [qo, ko] = call_turn(q, k, positions, frequencies, cos, sin, scale, interleaved, inverse);
        ctx->save_for_backward({tensor_of(positions), tensor_of(frequencies), tensor_of(cos), tensor_of(sin)});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["interleaved"] = interleaved;
        ctx->saved_data["inverse"] = inverse;
        // (a result asks for a gradient where its own tensor does: keys that go into a cache while the queries are trained must not)
        torch::autograd::variable_list plain;
        if (!wants_gradient(q)) plain.push_back(qo);
        if (!wants_gradient(k)) plain.push_back(ko);
        ctx->mark_non_differentiable(plain);
        return {qo, ko};
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        // a first-order backward needs no autograd bookkeeping
        std::optional<at::AutoDispatchBelowADInplaceOrView> below;
        if (!at::GradMode::is_enabled()) below.emplace();
        auto [dq, dk] = (below ? call_turn : rotary)(grads[0], grads[1], optional_of(saved[0]), optional_of(saved[1]), optional_of(saved[2]), optional_of(saved[3]),
                                                     ctx->saved_data["scale"].toDouble(), ctx->saved_data["interleaved"].toBool(), !ctx->saved_data["inverse"].toBool());
        return {dq, dk, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

// While a graph is recorded, a gradient goes into the autograd node that its tensor has.  A leaf keeps its node, and the stream that it was made on, for as long as any result of
// the leaf lives; torch lets that stream wait for the gradient.  A node of another stream than the recording one (of an eager result of the same leaf, or of an eager call that made
// the tensor) so draws that stream into the recording; this has ended the process.  Refused where it can be seen: before the forward call.
void require_recorded(const char *name, const Tensor &t) {
    if (!at::GradMode::is_enabled() || !wants_gradient(t)) return;
    const auto node = t.grad_fn() ? t.grad_fn() : torch::autograd::impl::try_get_grad_accumulator(t);
    const auto stream = node ? node->stream() : std::nullopt;
    const c10::impl::VirtualGuardImpl streams(t.device().type());
    const auto recorded = [] { return c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None; };
    if (!stream || *stream == streams.getStream(t.device()) || !recorded()) return;
    // (a stream that has joined the recording is as good; the default stream cannot, and must not be asked)
    bool joined = false;
    if (*stream != streams.getDefaultStream(t.device())) {
        const c10::StreamGuard on(*stream);
        joined = recorded();
    }
    TORCH_CHECK(joined, "rotary: the gradient of ", name,
                " would leave the graph that is being recorded, for a stream on which ", name, " has an eager result that is still alive (or was made): drop it before recording, ",
                "or run it on the recording stream");
}

Pair rotary(const Tensor &q, const Tensor &k, const OptTensor &positions, const OptTensor &frequencies, const OptTensor &cos, const OptTensor &sin, double scale,
            bool interleaved, bool inverse) {
    for (const auto &[name, t] : {std::pair<const char *, const OptTensor &>("frequencies", frequencies), {"cos", cos}, {"sin", sin}})
        if (t) TORCH_CHECK(!(at::GradMode::is_enabled() && wants_gradient(*t)) && !has_tangent(*t), "rotary has no gradient for ", name, ": detach it");
    bool plain = true;
    for (const Tensor *t : {&q, &k}) plain = plain && !(at::GradMode::is_enabled() && wants_gradient(*t)) && !has_tangent(*t);
    if (plain) {
        const at::AutoDispatchBelowADInplaceOrView below;
        return call_turn(q, k, positions, frequencies, cos, sin, scale, interleaved, inverse);
    }
    require_recorded("q", q);
    require_recorded("k", k);
    const auto out = RotaryFunction::apply(q, k, positions, frequencies, cos, sin, scale, interleaved, inverse);
    return {out[0], out[1]};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(gptoss_attn, m) {
    m.def("rotary_turn(Tensor q, Tensor k, Tensor? positions, Tensor? frequencies, Tensor? cos, Tensor? sin, float scale, bool interleaved, bool inverse) -> (Tensor, Tensor)");
    m.def("rotary(Tensor q, Tensor k, Tensor? positions, Tensor? frequencies, Tensor? cos, Tensor? sin, float scale, bool interleaved, bool inverse=False) -> (Tensor, Tensor)",
          &rotary);
}
TORCH_LIBRARY_IMPL(gptoss_attn, CUDA, m) { m.impl("rotary_turn", &turn); }
TORCH_LIBRARY_IMPL(gptoss_attn, CPU, m) { m.impl("rotary_turn", torch::CppFunction::makeFromBoxedFunction<&refuse_cpu>()); }
TORCH_LIBRARY_IMPL(gptoss_attn, Autograd, m) { m.impl("rotary_turn", torch::autograd::autogradNotImplementedFallback()); }
TORCH_LIBRARY_IMPL(gptoss_attn, FuncTorchBatched, m) {
    m.impl("rotary", torch::CppFunction::makeFromBoxedFunction<&refuse_vmap>());
    m.impl("rotary_turn", torch::CppFunction::makeFromBoxedFunction<&refuse_vmap>());
}

// Without the dispatcher, as the calls of the cache (torch_paged.cpp): of a decoding step's few microseconds the way through it takes a good part.
namespace {

PyObject *rotary_now(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 8 || !direct_now()) return not_implemented();
    Arguments a{args};
    const Tensor &q = a.tensor(0), &k = a.tensor(1);
    const OptTensor positions = a.optional(2), frequencies = a.optional(3), cos = a.optional(4), sin = a.optional(5);
    const double scale = a.number(6);
    const bool interleaved = a.truth(7);
    if (!a.ok) return not_implemented();
    Pair out;
    {
        const pybind11::gil_scoped_release free;
        out = turn(q, k, positions, frequencies, cos, sin, scale, interleaved, false);
    }
    return pair(out);
    END_HANDLE_TH_ERRORS
}

PyMethodDef kRotaryNow = {"rotary_now", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(&rotary_now)), METH_FASTCALL, nullptr};

}  // namespace

extern "C" PyObject *gptoss_rotary_direct() { return PyCFunction_New(&kRotaryNow, nullptr); }
