// What the PyTorch operators over the C ABI share: checks, memory, strides, errors.
#pragma once
#include <ATen/ATen.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <pybind11/pybind11.h>
#include <torch/library.h>

#include "../../include/gptoss_attn.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using c10::SymInt;

constexpr int64_t kMaxSeqStride = int64_t(1) << 24;   // elements; the library refuses larger sequence strides (ERR_STRIDE)

// The kernels need unit stride along head_dim, 16-byte aligned rows and a sequence stride of at least head_dim and at most
// 2^24 elements; anything else is copied.
inline Tensor row_contiguous(const Tensor &t, int64_t seq_dim) {
    const auto st = t.strides();
    const int64_t eb = t.element_size();
    const bool ok = st[3] == 1 && (st[0] * eb) % 16 == 0 && (st[1] * eb) % 16 == 0 && (st[2] * eb) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0 && st[seq_dim] >= t.size(3) && st[seq_dim] <= kMaxSeqStride;
    return ok ? t : t.contiguous();
}

inline void require_on(const Tensor &q, const char *name, const Tensor &t) {
    TORCH_CHECK(t.device() == q.device(), name, " is on ", t.device(), " but q is on ", q.device(), ": every tensor must be on q's GPU");
}

// Memory for a result or for scratch, without the dispatcher: every value of it is written before it is read.  A call's allocations are a tenth of its host time.
inline Tensor new_tensor(at::IntArrayRef sizes, at::ScalarType dtype, const Tensor &like) {
    return Tensor(at::detail::empty_cuda(sizes, dtype, like.device(), std::nullopt));
}

inline void set(gptoss_attn_strides &s, const Tensor &t, bool bshd) {
    s.b = t.stride(0);
    s.h = t.stride(bshd ? 2 : 1);
    s.s = t.stride(bshd ? 1 : 2);
}

// A failed library call is the package's GptossAttnError wherever it happens: in a call, a backward or a traced program.
inline void check(const char *name, int rc) {
    if (rc == 0) return;
    const pybind11::gil_scoped_acquire gil;
    const pybind11::object type = pybind11::module_::import("oregon_gpt_oss_patching_amd._lib").attr("GptossAttnError");
    PyErr_SetObject(type.ptr(), type(name, rc, gptoss_attn_status_string(rc)).ptr());
    throw pybind11::error_already_set();
}

}  // namespace
