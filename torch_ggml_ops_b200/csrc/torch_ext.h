// What the parts of the module over libtorch's C++ API share.
#pragma once

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include "../../include/tgo_mmq.h"

namespace tgo_ext {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::tensor_list;
using torch::autograd::Variable;
using torch::autograd::variable_list;

template <typename Fn>
const c10::TypedOperatorHandle<Fn> op(const char* name) {
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Fn>();
}
// Whether one of an operator's differentiable inputs wants a gradient.  No operator here has a forward-mode derivative: a tangent is
// refused, on whichever input it is, because the way below autograd would drop it and answer with a derivative of zero.
inline bool one_wants_grad(const Tensor& t) {
    TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), "torch_ggml_ops operators do not support forward-mode differentiation");
    return t.requires_grad();
}
inline bool one_wants_grad(const std::optional<Tensor>& t) { return t.has_value() && one_wants_grad(*t); }
template <typename... T>
bool wants_grad(const T&... t) {
    return (... | one_wants_grad(t)) && at::GradMode::is_enabled();
}
inline void check_rc(int rc, const char* what) { TORCH_CHECK(rc == TGO_OK, what, " failed: ", tgo_last_error()); }
inline void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// an uninitialised CUDA tensor, without the way through the dispatcher (some 0.4 us of a call of 8)
inline Tensor new_cuda(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
    return Tensor(at::detail::empty_cuda(sizes, type, like.device(), std::nullopt));
}

}  // namespace tgo_ext
