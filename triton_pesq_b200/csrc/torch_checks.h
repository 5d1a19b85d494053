// What the torch ops of the training operators share: checks of their operands, errors, autograd.
#pragma once

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include "../../include/pesq_cuda.h"

namespace pesq_torch {

using OptTensor = std::optional<at::Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

inline void check_status(int status, const char* what) {
  if (status == PESQ_OK) return;
  const char* msg = pesq_last_error();
  if (status == PESQ_ERR_INVALID_ARGUMENT) TORCH_CHECK_VALUE(false, what, ": ", msg);
  TORCH_CHECK(false, what, " failed (status ", status, "): ", msg);
}

inline int dtype_code(const at::Tensor& t, const char* op, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat:
      return PESQ_F32;
    case at::kBFloat16:
      return PESQ_BF16;
    case at::kHalf:
      return PESQ_F16;
    default:
      TORCH_CHECK(false, "The CUDA ", op, " supports float32, bfloat16 and float16, `", name, "` is ", t.scalar_type(),
                  ".");
  }
}

inline void check_cuda(const at::Tensor& t, const at::Tensor& first, const char* op, const char* name) {
  TORCH_CHECK(t.is_cuda(), "The CUDA ", op, " needs `", name, "` to live on a GPU.");
  TORCH_CHECK(t.device() == first.device(), "The CUDA ", op, " needs all tensors on one device, `", name, "` is on ",
              t.device(), ", not ", first.device(), ".");
}

inline void check_shape(const at::Tensor& t, at::IntArrayRef want, const char* op, const char* name) {
  TORCH_CHECK_VALUE(t.sizes() == want, "The CUDA ", op, " needs `", name, "` of shape ", want, ", got ", t.sizes(), ".");
}

inline void check_float(const at::Tensor& t, const char* op, const char* name) {
  TORCH_CHECK(t.scalar_type() == at::kFloat, "The CUDA ", op, " needs `", name, "` in float32, it is ", t.scalar_type(),
              ".");
}

inline bool given(const OptTensor& t) { return t.has_value() && t->defined(); }

inline void check_gradient(const at::Tensor& t, const at::Tensor& of, at::IntArrayRef want, const char* op, const char* name) {
  check_cuda(t, of, op, name);
  check_shape(t, want, op, name);
}

inline const float* floats(const OptTensor& t) { return t.has_value() && t->defined() ? t->data_ptr<float>() : nullptr; }

inline OptTensor optional_of(const Variable& v) { return v.defined() ? OptTensor(v) : std::nullopt; }

inline void no_second_derivative(const char* op) {
  TORCH_CHECK(!at::GradMode::is_enabled(), "The CUDA ", op, " has no second derivative (create_graph=True).");
}

inline bool has_tangent(const at::Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }
inline bool has_tangent(const OptTensor& t) { return t.has_value() && has_tangent(*t); }
template <class... Ts>
inline void no_forward_mode(const char* op, const Ts&... inputs) {
  TORCH_CHECK(!(has_tangent(inputs) || ...), "The CUDA ", op, " has no forward-mode derivative.");
}

inline bool wants_grad(const at::Tensor& t) { return t.requires_grad(); }
inline bool wants_grad(const OptTensor& t) { return t.has_value() && t->defined() && t->requires_grad(); }

}  // namespace pesq_torch
