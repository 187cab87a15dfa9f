// What the PyTorch operators of the serving calls share: what they refuse, and the way past the dispatcher from Python.
#pragma once
#include <climits>

#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/record_function.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include "torch_common.h"

namespace {

using Pair = std::tuple<Tensor, Tensor>;

inline int32_t size32(int64_t n) {
    TORCH_CHECK(n <= INT_MAX, "a dimension of ", n, " is too long");
    return static_cast<int32_t>(n);
}

// As int32 on the cache's GPU; what is so already does not go through the dispatcher (half a microsecond each).  Wider numbers that int32 does not hold become its
// ends, which are no page, in front of every position and behind each (cut off, 2^32 + 3 would be page 3).
inline bool is_integers(const Tensor &t) { return at::isIntegralType(t.scalar_type(), /*includeBool=*/true) && t.scalar_type() != at::kUInt64; }
inline Tensor int32_on(const Tensor &t, const Tensor &pages) {
    if (t.scalar_type() == at::kInt && t.device() == pages.device()) return t;
    const bool wide = t.scalar_type() == at::kLong || t.scalar_type() == at::kUInt32;
    return (wide ? t.to(at::kLong).clamp(INT_MIN, INT_MAX) : t).to(pages.device(), at::kInt);
}

// Before a launch that writes into tensors of the caller: this refuses those that were made in inference mode and are written outside of it.
inline void about_to_write(std::initializer_list<const Tensor *> tensors) {
    for (const Tensor *t : tensors)
        if (t) t->unsafeGetTensorImpl()->bump_version();
}

// What a tensor asks for (most have no record of either): a gradient, which torch.no_grad() takes back, or the tangent of forward mode, which it does not.
inline bool wants_gradient(const Tensor &t) { return t.unsafeGetTensorImpl()->autograd_meta() && t.requires_grad(); }
inline bool has_tangent(const Tensor &t) { return t.unsafeGetTensorImpl()->autograd_meta() && t._fw_grad(0).defined(); }

// Tensors with either are refused, as these calls would drop it without a word.
inline void refuse_gradients(const c10::OperatorHandle &op, c10::DispatchKeySet keys, torch::jit::Stack *stack) {
    const size_t n = op.schema().arguments().size();
    for (size_t i = stack->size() - n; i < stack->size(); ++i) {
        if (!(*stack)[i].isTensor()) continue;
        const Tensor &t = (*stack)[i].toTensor();
        TORCH_CHECK(!at::GradMode::is_enabled() || !wants_gradient(t), op.schema().name(), " has no gradient: call it under torch.no_grad() (argument ",
                    op.schema().arguments()[i + n - stack->size()].name(), " requires one)");
        TORCH_CHECK(!has_tangent(t), op.schema().name(), " has no gradient, forward mode's neither: argument ", op.schema().arguments()[i + n - stack->size()].name(),
                    " has a tangent");
    }
    const at::AutoDispatchBelowADInplaceOrView below;
    op.redispatchBoxed(keys & c10::after_ADInplaceOrView_keyset, stack);
}

inline void refuse_cpu(const c10::OperatorHandle &, torch::jit::Stack *) {
    TORCH_CHECK(false, "gptoss attention runs on the GPU only (HIP kernels); got CPU tensors");
}

inline void refuse_vmap(const c10::OperatorHandle &, torch::jit::Stack *) {
    TORCH_CHECK(false, "gptoss attention cannot be vmapped: its tensors have a batch dimension of their own");
}

// Whether what is dispatched now reaches the GPU's kernel as it is.
inline bool direct_now() {
    return (c10::impl::tls_local_dispatch_key_set().included_ - c10::default_included_set).empty() && !at::impl::torch_function_mode_enabled() && !torch::jit::tracer::isTracing() &&
           !at::getStepCallbacksUnlessEmpty(at::RecordScope::FUNCTION).has_value();
}

// Arguments from Python; `ok` falls where one is not what a direct call takes.
struct Arguments {
    PyObject *const *args;
    const bool grad = at::GradMode::is_enabled();
    bool ok = true;

    const Tensor &tensor(int i) {
        static const Tensor none;
        static const c10::DispatchKeySet plain = c10::DispatchKeySet(c10::DispatchKey::CUDA) | c10::autograd_dispatch_keyset_with_ADInplaceOrView | c10::autocast_dispatch_keyset |
                                                 c10::getAutogradRelatedKeySetFromBackend(c10::BackendComponent::CUDABit);
        if (!THPVariable_CheckExact(args[i])) return ok = false, none;
        const Tensor &t = THPVariable_Unpack(args[i]);
        if ((t.key_set().raw_repr() & ~plain.raw_repr()) != 0 || (grad && wants_gradient(t)) || has_tangent(t)) ok = false;
        return t;
    }
    OptTensor optional(int i) { return args[i] == Py_None ? OptTensor() : OptTensor(tensor(i)); }
    int64_t integer(int i) {
        if (!PyLong_CheckExact(args[i])) return ok = false, 0;
        int overflow = 0;
        const long long x = PyLong_AsLongLongAndOverflow(args[i], &overflow);
        if (overflow) ok = false;
        return x;
    }
    int64_t integer_or_none(int i) { return args[i] == Py_None ? 0 : integer(i); }        // None: 0, where that says the same
    double number(int i) { return PyFloat_CheckExact(args[i]) ? PyFloat_AS_DOUBLE(args[i]) : (ok = false, 0.0); }
    bool truth(int i) { return PyBool_Check(args[i]) ? args[i] == Py_True : (ok = false); }
    at::ScalarType dtype(int i) { return THPDtype_Check(args[i]) ? reinterpret_cast<THPDtype *>(args[i])->scalar_type : (ok = false, at::kBFloat16); }
};

inline PyObject *not_implemented() { Py_RETURN_NOTIMPLEMENTED; }

inline PyObject *pair(const Pair &x) {
    const pybind11::object a = pybind11::reinterpret_steal<pybind11::object>(THPVariable_Wrap(std::get<0>(x))),
                           b = pybind11::reinterpret_steal<pybind11::object>(THPVariable_Wrap(std::get<1>(x)));
    return a && b ? PyTuple_Pack(2, a.ptr(), b.ptr()) : nullptr;
}

// A tuple of Python functions.
template <size_t N>
inline PyObject *functions_of(PyMethodDef (&defs)[N]) {
    PyObject *out = PyTuple_New(N);
    for (size_t i = 0; out && i < N; ++i) {
        PyObject *f = PyCFunction_New(&defs[i], nullptr);
        if (!f) { Py_DECREF(out); return nullptr; }
        PyTuple_SET_ITEM(out, i, f);
    }
    return out;
}

}  // namespace
