// Checks, outputs and rows of tensors for the host sides of the operators that are called one by one.
#pragma once
#include "host.h"
#include <torch/csrc/autograd/custom_function.h>
#include <ATen/cuda/EmptyTensor.h>

namespace vig_host {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptT = std::optional<Tensor>;

[[noreturn]] inline void not_implemented(const char* msg) {
    PyErr_SetString(PyExc_NotImplementedError, msg);
    throw py::error_already_set();
}
inline std::string shape_of(const Tensor& t) {
    std::ostringstream s;
    s << t.sizes();
    return s.str();
}
// the message is only put together where it is needed: these calls are a few microseconds long
#define want(ok, msg) do { if (!(ok)) throw py::value_error(msg); } while (0)
#define want_type(ok, msg) do { if (!(ok)) throw py::type_error(msg); } while (0)

inline void on_gpu(const Tensor& t) { if (!t.is_cuda()) throw std::runtime_error("vig_b200 kernels need CUDA tensors; there is no CPU path"); }
inline void same_device(const Tensor& t, const Tensor& like, const char* name) {
    on_gpu(t);
    want(t.device() == like.device(), std::string(name) + " lives on another device");
}
inline int code(const Tensor& t) {
    const int c = dtype_code(t);
    want_type(c >= 0, std::string("unsupported dtype ") + toString(t.scalar_type()) + "; expected float32, bfloat16 or float16");
    return c;
}
inline bool unit_last(const Tensor& t) { return t.dim() == 0 || t.size(-1) <= 1 || t.stride(-1) == 1; }
inline Tensor get(const OptT& t) { return t ? *t : Tensor(); }
inline bool wants_grad(std::initializer_list<const Tensor*> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : ts) if (t->defined() && t->requires_grad()) return true;
    return false;
}
// a dual tensor of forward mode, which need not require a gradient: its tangent would be dropped
inline void no_tangents(std::initializer_list<const Tensor*> ts) {
    for (const Tensor* t : ts)
        if (t->defined() && t->_fw_grad(0).defined()) not_implemented("forward-mode gradients are not implemented");
}
// runs on a thread of the autograd engine, without Python's lock: a torch error, no Python one
inline void once(const variable_list& ds, const variable_list& saved) {
    for (const Tensor& t : ds) TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(), "forward-mode gradients are not implemented");
    if (!at::GradMode::is_enabled()) return;
    for (const auto* list : {&ds, &saved})
        for (const Tensor& t : *list) TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t.requires_grad(), "gradients of these gradients are not implemented");
}
inline Tensor rows(const Tensor& t) { return t.defined() && !unit_last(t) ? t.contiguous() : t; }

// an output on the device of `like`: the allocator's call without the dispatcher's way to it, which is a tenth of a short call
inline Tensor fresh(at::IntArrayRef sizes, const Tensor& like, at::ScalarType type) { return Tensor(at::detail::empty_cuda(sizes, type, like.device(), std::nullopt)); }
inline Tensor fresh(at::IntArrayRef sizes, const Tensor& like) { return fresh(sizes, like, like.scalar_type()); }

// [..., N] seen as rows; a copy where they have no common stride
inline Tensor as_rows(const Tensor& t) {
    if (t.dim() == 2 && unit_last(t)) return t;
    const int64_t N = t.size(-1);
    if (t.is_contiguous()) return t.view({N ? t.numel() / N : 0, N});
    return rows(t.reshape({N ? t.numel() / N : 0, N}));
}
inline int64_t ld(const Tensor& t) { return t.defined() ? t.size(0) > 1 ? t.stride(0) : t.size(1) : 0; }

}  // namespace vig_host
