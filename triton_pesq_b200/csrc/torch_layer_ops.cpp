// torch custom ops of the layer norm over the C ABI of
// libpesq_cuda.so, with their autograd nodes: as in torch_train_ops.cpp, the op that
// a caller uses, and the forward and backward it is made of.
#include <algorithm>

#include "torch_checks.h"

namespace {

using namespace pesq_torch;

pesq_heads heads_of(const at::Tensor& t) { return {t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)}; }

// channels adjacent
at::Tensor rows(const at::Tensor& t) { return t.size(3) <= 1 || t.stride(3) == 1 ? t : t.contiguous(); }

// ------------------------------------------------------------------ layer norm

constexpr const char* kNorm = "layer norm";

at::ScalarType type_of(int64_t code) { return code == PESQ_F32 ? at::kFloat : code == PESQ_BF16 ? at::kBFloat16 : at::kHalf; }

struct NormCall {
  at::Tensor x, weight, bias;
  pesq_layer_norm_desc d{};
  at::ScalarType out;

  // x [batch, step, head, channel], weight and bias [head, channel]
  NormCall(const at::Tensor& x_, const at::Tensor& weight_, const OptTensor& bias_, double eps, int64_t dtype) {
    check_cuda(x_, x_, kNorm, "x");
    TORCH_CHECK(x_.dim() == 4, "The CUDA layer norm needs `x` [batch, step, head, channel], got ", x_.sizes(), ".");
    d.dtype = dtype_code(x_, kNorm, "x");
    TORCH_CHECK_VALUE(dtype >= PESQ_F32 && dtype <= PESQ_F16, "The CUDA layer norm has no type ", dtype, ".");
    d.out_dtype = static_cast<int32_t>(dtype);
    out = type_of(dtype);
    TORCH_CHECK(x_.scalar_type() == at::kFloat || x_.scalar_type() == out,
                "The CUDA layer norm needs `x` in float32 or in the result's type, it is ", x_.scalar_type(), ".");
    TORCH_CHECK_VALUE(eps >= 0.0, "The CUDA layer norm needs an `eps` that is not negative, got ", eps, ".");
    d.eps = static_cast<float>(eps);
    x = rows(x_);
    d.batch = x.size(0);
    d.steps = x.size(1);
    d.heads = x.size(2);
    d.width = x.size(3);
    d.x = heads_of(x);
    weight = vector(weight_, "weight");
    d.weight = weight.data_ptr<float>();
    if (given(bias_)) {
      bias = vector(*bias_, "bias");
      d.bias = bias.data_ptr<float>();
    }
  }

  at::Tensor vector(const at::Tensor& t, const char* name) {
    check_cuda(t, x, kNorm, name);
    check_float(t, kNorm, name);
    check_shape(t, {x.size(2), x.size(3)}, kNorm, name);
    return t.contiguous();
  }

  bool empty() const { return x.numel() == 0; }
};

at::Tensor layer_norm_forward(const at::Tensor& x, const at::Tensor& weight, const OptTensor& bias, double eps,
                              int64_t dtype) {
  NormCall c(x, weight, bias, eps, dtype);
  c10::cuda::CUDAGuard guard(x.device());
  at::Tensor y = at::empty(x.sizes(), x.options().dtype(c.out));
  if (!c.empty())
    check_status(pesq_layer_norm_forward(&c.d, at::cuda::getCurrentCUDAStream(), y.data_ptr()), "pesq_layer_norm_forward");
  return y;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> layer_norm_backward(const at::Tensor& x, const at::Tensor& weight,
                                                                   const OptTensor& bias, double eps, int64_t dtype,
                                                                   const at::Tensor& dy_) {
  NormCall c(x, weight, bias, eps, dtype);
  check_gradient(dy_, x, x.sizes(), kNorm, "dy");
  c10::cuda::CUDAGuard guard(x.device());
  at::Tensor dx = at::empty(x.sizes(), x.options()), dweight = at::empty(c.weight.sizes(), c.weight.options()),
             dbias = c.bias.defined() ? at::empty(c.bias.sizes(), c.bias.options()) : at::empty({0}, c.weight.options());
  if (c.empty()) {
    dweight.zero_();
    dbias.zero_();
    return {dx, dweight, dbias};
  }
  const at::Tensor dy = rows(dy_.to(c.out));
  size_t bytes = 0;
  check_status(pesq_layer_norm_workspace(&c.d, &bytes), "pesq_layer_norm_workspace");
  at::Tensor ws = at::empty({static_cast<int64_t>(bytes)}, x.options().dtype(at::kByte));
  check_status(pesq_layer_norm_backward(&c.d, at::cuda::getCurrentCUDAStream(), heads_of(dy), dx.data_ptr(),
                                        dweight.data_ptr<float>(), c.bias.defined() ? dbias.data_ptr<float>() : nullptr,
                                        ws.data_ptr(), bytes),
               "pesq_layer_norm_backward");
  return {dx, dweight, dbias};
}

const auto& norm_forward_op() {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("pesq_cuda::layer_norm_forward", "")
                       .typed<decltype(layer_norm_forward)>();
  return op;
}
const auto& norm_backward_op() {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("pesq_cuda::layer_norm_backward", "")
                       .typed<decltype(layer_norm_backward)>();
  return op;
}

struct LayerNorm : public torch::autograd::Function<LayerNorm> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& weight, const OptTensor& bias,
                            double eps, int64_t dtype) {
    at::AutoDispatchBelowADInplaceOrView below;
    at::Tensor y = norm_forward_op().call(x, weight, bias, eps, dtype);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, weight, bias.value_or(at::Tensor())});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["dtype"] = dtype;
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grad) {
    no_second_derivative(kNorm);
    const auto s = ctx->get_saved_variables();
    variable_list out(5);
    if (!grad[0].defined()) return out;
    auto [dx, dweight, dbias] = norm_backward_op().call(s[0], s[1], optional_of(s[2]), ctx->saved_data["eps"].toDouble(),
                                                        ctx->saved_data["dtype"].toInt(), grad[0]);
    out[0] = dx;
    out[1] = dweight;
    if (s[2].defined()) out[2] = dbias;
    return out;
  }
};

// x [..., channel] with weight [channel], or [..., head, channel] with [head, channel]; dtype < 0: x's
at::Tensor layer_norm(const at::Tensor& x_, const at::Tensor& weight_, const OptTensor& bias_, double eps, int64_t dtype) {
  check_cuda(x_, x_, kNorm, "x");
  const int64_t dims = x_.dim(), vector = weight_.dim();
  TORCH_CHECK_VALUE(vector == 1 || vector == 2, "The CUDA layer norm needs `weight` [channel] or [head, channel], got ",
                    weight_.sizes(), ".");
  TORCH_CHECK_VALUE(dims >= vector && x_.sizes().slice(dims - vector) == weight_.sizes(),
                    "The CUDA layer norm needs `x` whose last sizes are `weight`'s ", weight_.sizes(), ", got ", x_.sizes(), ".");
  if (given(bias_)) check_shape(*bias_, weight_.sizes(), kNorm, "bias");
  no_forward_mode(kNorm, x_, weight_, bias_);
  if (dtype < 0) dtype = dtype_code(x_, kNorm, "x");
  at::Tensor x = x_, weight = weight_;
  OptTensor bias = bias_;
  if (vector == 1) {
    weight = weight.unsqueeze(0);
    if (given(bias)) bias = bias->unsqueeze(0);
    x = x.unsqueeze(dims - 1);
  }
  while (x.dim() < 4) x = x.unsqueeze(0);
  if (x.dim() > 4) x = x.flatten(0, x.dim() - 4);
  const bool grad = at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight) || wants_grad(bias));
  const at::Tensor y = grad ? LayerNorm::apply(x, weight, bias, eps, dtype) : norm_forward_op().call(x, weight, bias, eps, dtype);
  return y.sizes() == x_.sizes() ? y : y.view(x_.sizes());
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(pesq_cuda, m) {
  m.def("layer_norm(Tensor x, Tensor weight, Tensor? bias, float eps, int dtype) -> Tensor");
  m.def("layer_norm_forward(Tensor x, Tensor weight, Tensor? bias, float eps, int dtype) -> Tensor");
  m.def("layer_norm_backward(Tensor x, Tensor weight, Tensor? bias, float eps, int dtype, Tensor dy) -> "
        "(Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(pesq_cuda, CompositeImplicitAutograd, m) {
  m.impl("layer_norm", &layer_norm);
}

TORCH_LIBRARY_IMPL(pesq_cuda, CUDA, m) {
  m.impl("layer_norm_forward", &layer_norm_forward);
  m.impl("layer_norm_backward", &layer_norm_backward);
}
