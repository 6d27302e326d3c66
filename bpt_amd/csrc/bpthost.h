// What the host sides of bptblockop.cpp and bptlinearop.cpp share: checks of arguments, streams, status codes.
#pragma once
#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <optional>
#include <tuple>

#include "../../include/bptattn.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

using Optional = std::optional<Tensor>;

inline void *stream_of(const Tensor &t) { return (void *)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

inline void check_status(int st, const char *what) { TORCH_CHECK(st == BPT_OK, what, ": ", bpt_strerror(st), " (status ", st, ")"); }

inline void check_input(const Tensor &t, const char *name) {
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(t.layout() == at::kStrided && t.is_contiguous(), name, " must be contiguous");
}
inline void check_like(const Tensor &t, const Tensor &x, const char *name) {
    check_input(t, name);
    TORCH_CHECK(t.scalar_type() == x.scalar_type(), "all floating point arguments must share one dtype");
    TORCH_CHECK_VALUE(t.device() == x.device(), "all tensors of a call must be on one device");
}
inline void check_shape(const Tensor &t, at::IntArrayRef shape, const char *name) {
    TORCH_CHECK_VALUE(t.sizes() == shape, name, " must have shape ", shape, ", got ", t.sizes());
}

inline int dtype_code(const Tensor &t) {
    const auto s = t.scalar_type();
    return s == at::kFloat ? BPT_F32 : s == at::kBFloat16 ? BPT_BF16 : s == at::kDouble ? BPT_F64 : -1;
}

inline bool differentiated(std::initializer_list<const Tensor *> tensors) {
    for (const Tensor *t : tensors)
        if (t->defined() && ((at::GradMode::is_enabled() && t->requires_grad()) || t->_fw_grad(/*level=*/0).defined())) return true;
    return false;
}

inline void *ptr(const Tensor &t) { return t.defined() && t.numel() ? t.data_ptr() : nullptr; }

}  // namespace
