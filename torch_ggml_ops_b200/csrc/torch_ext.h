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
inline bool wants_grad(const Tensor& t) { return at::GradMode::is_enabled() && t.requires_grad(); }
inline void check_rc(int rc, const char* what) { TORCH_CHECK(rc == TGO_OK, what, " failed: ", tgo_last_error()); }
inline void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// an uninitialised CUDA tensor, without the way through the dispatcher (some 0.4 us of a call of 8)
inline Tensor new_cuda(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
    return Tensor(at::detail::empty_cuda(sizes, type, like.device(), std::nullopt));
}

}  // namespace tgo_ext
