// torch custom ops of the layer norm, the linear attention and Muon over the C ABI of
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

  // x [..., channel], weight and bias [channel]; or [..., head, channel] and [head, channel]
  NormCall(const at::Tensor& x_, const at::Tensor& weight_, const OptTensor& bias_, double eps, int64_t dtype) {
    check_cuda(x_, x_, kNorm, "x");
    const int64_t dims = x_.dim(), own = weight_.dim();
    TORCH_CHECK_VALUE(own == 1 || own == 2, "The CUDA layer norm needs `weight` [channel] or [head, channel], got ",
                      weight_.sizes(), ".");
    TORCH_CHECK_VALUE(dims >= own && x_.sizes().slice(dims - own) == weight_.sizes(),
                      "The CUDA layer norm needs `x` whose last sizes are `weight`'s ", weight_.sizes(), ", got ", x_.sizes(), ".");
    d.dtype = dtype_code(x_, kNorm, "x");
    TORCH_CHECK_VALUE(dtype >= PESQ_F32 && dtype <= PESQ_F16, "The CUDA layer norm has no type ", dtype, ".");
    d.out_dtype = static_cast<int32_t>(dtype);
    out = type_of(dtype);
    TORCH_CHECK(x_.scalar_type() == at::kFloat || x_.scalar_type() == out,
                "The CUDA layer norm needs `x` in float32 or in the result's type, it is ", x_.scalar_type(), ".");
    TORCH_CHECK_VALUE(eps >= 0.0, "The CUDA layer norm needs an `eps` that is not negative, got ", eps, ".");
    d.eps = static_cast<float>(eps);
    heads = own == 2;
    x = rows(x_);
    d.width = x.size(-1);
    d.heads = heads ? x.size(-2) : 1;
    lead = dims - own;
    d.batch = lead == 2 ? x.size(0) : 1;
    d.steps = 1;
    for (int64_t k = lead == 2 ? 1 : 0; k < lead; ++k) d.steps *= x.size(k);
    d.x = strides_of(x);
    weight = vector(weight_, "weight");
    d.weight = weight.data_ptr<float>();
    if (given(bias_)) {
      bias = vector(*bias_, "bias");
      d.bias = bias.data_ptr<float>();
    }
  }

  // of up to two leading dimensions any strides, of more a dense tensor; channels adjacent
  at::Tensor rows(const at::Tensor& t) const {
    const int64_t leading = t.dim() - (heads ? 2 : 1);
    return leading <= 2 && (t.size(-1) <= 1 || t.stride(-1) == 1) ? t : t.contiguous();
  }
  pesq_heads strides_of(const at::Tensor& t) const {
    const int64_t row = d.heads * d.width;
    return {t.data_ptr(), lead == 2 ? t.stride(0) : 0, lead == 2 ? t.stride(1) : lead == 1 ? t.stride(0) : row,
            heads ? t.stride(-2) : d.width};
  }
  at::Tensor vector(const at::Tensor& t, const char* name) const {
    check_cuda(t, x, kNorm, name);
    check_float(t, kNorm, name);
    check_shape(t, x.sizes().slice(lead), kNorm, name);
    return t.contiguous();
  }

  bool empty() const { return x.numel() == 0; }
  bool heads = false;
  int64_t lead = 0;  // dimensions before the weight's
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
  const at::Tensor dy = c.rows(dy_.scalar_type() == c.out ? dy_ : dy_.to(c.out));
  size_t bytes = 0;
  check_status(pesq_layer_norm_workspace(&c.d, &bytes), "pesq_layer_norm_workspace");
  at::Tensor ws = at::empty({static_cast<int64_t>(bytes)}, x.options().dtype(at::kByte));
  check_status(pesq_layer_norm_backward(&c.d, at::cuda::getCurrentCUDAStream(), c.strides_of(dy), dx.data_ptr(),
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

// dtype < 0: x's
at::Tensor layer_norm(const at::Tensor& x, const at::Tensor& weight, const OptTensor& bias, double eps, int64_t dtype) {
  check_cuda(x, x, kNorm, "x");
  no_forward_mode(kNorm, x, weight, bias);
  if (dtype < 0) dtype = dtype_code(x, kNorm, "x");
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight) || wants_grad(bias)))
    return LayerNorm::apply(x, weight, bias, eps, dtype);
  return norm_forward_op().call(x, weight, bias, eps, dtype);
}

// ------------------------------------------------------------ linear attention

constexpr const char* kAttention = "linear attention";

struct AttentionCall {
  at::Tensor q, k, v, decay, state, reset, lengths;
  pesq_linear_attention_desc d{};

  AttentionCall(const at::Tensor& q_, const at::Tensor& k_, const at::Tensor& v_, const at::Tensor& decay_,
                const OptTensor& state_, const OptTensor& reset_, const OptTensor& lengths_, bool reverse, double scale) {
    check_cuda(q_, q_, kAttention, "q");
    d.dtype = dtype_code(q_, kAttention, "q");
    TORCH_CHECK(q_.dim() == 4, "The CUDA linear attention needs `q` [batch, step, head, key], got ", q_.sizes(), ".");
    check_cuda(k_, q_, kAttention, "k");
    check_cuda(v_, q_, kAttention, "v");
    check_cuda(decay_, q_, kAttention, "log_decay");
    check_shape(k_, q_.sizes(), kAttention, "k");
    TORCH_CHECK_VALUE(v_.dim() == 4 && v_.sizes().slice(0, 3) == q_.sizes().slice(0, 3),
                      "The CUDA linear attention needs `v` [batch, step, head, value] beside `q` of shape ", q_.sizes(), ", got ",
                      v_.sizes(), ".");
    TORCH_CHECK(k_.scalar_type() == q_.scalar_type() && v_.scalar_type() == q_.scalar_type(),
                "The CUDA linear attention needs `q`, `k` and `v` in one type, got ", q_.scalar_type(), ", ",
                k_.scalar_type(), " and ", v_.scalar_type(), ".");
    check_float(decay_, kAttention, "log_decay");
    TORCH_CHECK_VALUE(scale - scale == 0.0, "The CUDA linear attention needs a finite `scale`, got ", scale, ".");
    q = rows(q_);
    k = rows(k_);
    v = rows(v_);
    decay = decay_;
    d.batch = q.size(0);
    d.steps = q.size(1);
    d.heads = q.size(2);
    d.key = q.size(3);
    d.value = v.size(3);
    d.decay_shared = decay.dim() == 1;
    if (d.decay_shared) {
      check_shape(decay, {d.heads}, kAttention, "log_decay");
      d.decay_head_stride = decay.stride(0);
    } else {
      const int64_t want[3] = {d.batch, d.steps, d.heads};
      check_shape(decay, want, kAttention, "log_decay");
      d.decay_batch_stride = decay.stride(0);
      d.decay_step_stride = decay.stride(1);
      d.decay_head_stride = decay.stride(2);
    }
    d.log_decay = decay.data_ptr<float>();
    if (given(state_)) {
      check_cuda(*state_, q_, kAttention, "state");
      check_float(*state_, kAttention, "state");
      const int64_t want[4] = {d.batch, d.heads, d.key, d.value};
      check_shape(*state_, want, kAttention, "state");
      state = state_->contiguous();
      d.state = state.data_ptr<float>();
    }
    if (given(reset_)) {
      check_cuda(*reset_, q_, kAttention, "reset");
      check_shape(*reset_, {d.batch, d.steps}, kAttention, "reset");
      TORCH_CHECK(reset_->scalar_type() == at::kBool, "The CUDA linear attention needs `reset` in bool, it is ",
                  reset_->scalar_type(), ".");
      reset = *reset_;
      d.reset = static_cast<const uint8_t*>(reset.data_ptr());
      d.reset_batch_stride = reset.stride(0);
      d.reset_step_stride = reset.stride(1);
    }
    if (given(lengths_)) {
      check_cuda(*lengths_, q_, kAttention, "lengths");
      check_shape(*lengths_, {d.batch}, kAttention, "lengths");
      TORCH_CHECK(lengths_->scalar_type() == at::kLong || lengths_->scalar_type() == at::kInt,
                  "The CUDA linear attention needs `lengths` in int64 or int32, it is ", lengths_->scalar_type(), ".");
      lengths = lengths_->to(at::kLong).contiguous();
      d.lengths = lengths.data_ptr<int64_t>();
    }
    d.reverse = reverse;
    d.scale = static_cast<float>(scale);
    d.q = heads_of(q);
    d.k = heads_of(k);
    d.v = heads_of(v);
  }

  bool empty() const { return q.numel() == 0 || v.numel() == 0; }
  at::Tensor matrix() const { return at::empty({d.batch, d.heads, d.key, d.value}, q.options().dtype(at::kFloat)); }
};

// (y, last, the states kept for the backward where `keep`)
std::tuple<at::Tensor, at::Tensor, at::Tensor> linear_attention_forward(const at::Tensor& q, const at::Tensor& k,
                                                                        const at::Tensor& v, const at::Tensor& decay,
                                                                        const OptTensor& state, const OptTensor& reset,
                                                                        const OptTensor& lengths, bool reverse, double scale,
                                                                        bool keep) {
  AttentionCall c(q, k, v, decay, state, reset, lengths, reverse, scale);
  c10::cuda::CUDAGuard guard(q.device());
  const auto bytes = q.options().dtype(at::kByte);
  at::Tensor y = at::empty(v.sizes(), v.options()), last = c.matrix();
  if (c.empty()) {
    y.zero_();  // (no keys: nothing is ever in the state)
    if (c.d.state) {
      last.copy_(c.state);
    } else {
      last.zero_();
    }
    return {y, last, at::empty({0}, bytes)};
  }
  size_t work = 0, kept = 0, back = 0;
  check_status(pesq_linear_attention_sizes(&c.d, &work, &kept, &back), "pesq_linear_attention_sizes");
  at::Tensor states = at::empty({keep ? static_cast<int64_t>(kept) : 0}, bytes), ws;
  if (work) ws = at::empty({static_cast<int64_t>(work)}, bytes);
  check_status(pesq_linear_attention_forward(&c.d, at::cuda::getCurrentCUDAStream(), y.data_ptr(), last.data_ptr<float>(),
                                             keep ? states.data_ptr() : nullptr, keep ? kept : 0,
                                             work ? ws.data_ptr() : nullptr, work),
               "pesq_linear_attention_forward");
  return {y, last, states};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> linear_attention_backward(
    const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& decay, const OptTensor& state,
    const OptTensor& reset, const OptTensor& lengths, bool reverse, double scale, const at::Tensor& kept_,
    const OptTensor& dy_, const OptTensor& dlast_) {
  AttentionCall c(q, k, v, decay, state, reset, lengths, reverse, scale);
  c10::cuda::CUDAGuard guard(q.device());
  at::Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(q.sizes(), q.options()),
             dv = at::empty(v.sizes(), v.options()), ddecay = at::empty(decay.sizes(), decay.options()), dstate = c.matrix();
  at::Tensor dlast, dy;
  if (given(dy_)) check_gradient(*dy_, q, v.sizes(), kAttention, "dy");
  if (given(dlast_)) {
    check_gradient(*dlast_, q, dstate.sizes(), kAttention, "dlast");
    dlast = dlast_->to(at::kFloat).contiguous();
  }
  if (c.empty()) {
    for (at::Tensor* t : {&dq, &dk, &dv, &ddecay}) t->zero_();
    if (dlast.defined()) {
      dstate.copy_(dlast);
    } else {
      dstate.zero_();
    }
    return {dq, dk, dv, ddecay, dstate};
  }
  dy = given(dy_) ? rows(dy_->to(q.scalar_type())) : at::zeros({1}, q.options()).expand(v.sizes());
  if (dy.stride(3) != 1 && dy.size(3) > 1) dy = dy.contiguous();
  size_t work = 0, kept = 0, back = 0;
  check_status(pesq_linear_attention_sizes(&c.d, &work, &kept, &back), "pesq_linear_attention_sizes");
  check_cuda(kept_, q, kAttention, "kept");
  TORCH_CHECK(kept_.scalar_type() == at::kByte && kept_.is_contiguous() && kept_.numel() == static_cast<int64_t>(kept),
              "The CUDA linear attention needs the states that its forward kept.");
  at::Tensor ws;
  if (back) ws = at::empty({static_cast<int64_t>(back)}, q.options().dtype(at::kByte));
  check_status(pesq_linear_attention_backward(&c.d, at::cuda::getCurrentCUDAStream(), kept_.data_ptr(), kept, heads_of(dy),
                                              dlast.defined() ? dlast.data_ptr<float>() : nullptr, dq.data_ptr(),
                                              dk.data_ptr(), dv.data_ptr(), ddecay.data_ptr<float>(),
                                              dstate.data_ptr<float>(), back ? ws.data_ptr() : nullptr, back),
               "pesq_linear_attention_backward");
  return {dq, dk, dv, ddecay, dstate};
}

const auto& attention_forward_op() {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("pesq_cuda::linear_attention_forward", "")
                       .typed<decltype(linear_attention_forward)>();
  return op;
}
const auto& attention_backward_op() {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("pesq_cuda::linear_attention_backward", "")
                       .typed<decltype(linear_attention_backward)>();
  return op;
}

struct LinearAttention : public torch::autograd::Function<LinearAttention> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                               const at::Tensor& decay, const OptTensor& state, const OptTensor& reset,
                               const OptTensor& lengths, bool reverse, double scale) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [y, last, kept] = attention_forward_op().call(q, k, v, decay, state, reset, lengths, reverse, scale, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({q, k, v, decay, state.value_or(at::Tensor()), reset.value_or(at::Tensor()),
                            lengths.value_or(at::Tensor()), kept});
    ctx->saved_data["reverse"] = reverse;
    ctx->saved_data["scale"] = scale;
    return {y, last};
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    no_second_derivative(kAttention);
    const auto s = ctx->get_saved_variables();
    variable_list out(9);
    if (!g[0].defined() && !g[1].defined()) return out;
    auto [dq, dk, dv, ddecay, dstate] = attention_backward_op().call(
        s[0], s[1], s[2], s[3], optional_of(s[4]), optional_of(s[5]), optional_of(s[6]),
        ctx->saved_data["reverse"].toBool(), ctx->saved_data["scale"].toDouble(), s[7], optional_of(g[0]), optional_of(g[1]));
    out[0] = dq;
    out[1] = dk;
    out[2] = dv;
    out[3] = ddecay;
    if (s[4].defined()) out[4] = dstate;
    return out;
  }
};

std::tuple<at::Tensor, at::Tensor> linear_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                    const at::Tensor& decay, const OptTensor& state, const OptTensor& reset,
                                                    const OptTensor& lengths, bool reverse, double scale) {
  check_cuda(q, q, kAttention, "q");
  no_forward_mode(kAttention, q, k, v, decay, state);
  if (at::GradMode::is_enabled() &&
      (wants_grad(q) || wants_grad(k) || wants_grad(v) || wants_grad(decay) || wants_grad(state))) {
    auto out = LinearAttention::apply(q, k, v, decay, state, reset, lengths, reverse, scale);
    return {out[0], out[1]};
  }
  auto [y, last, kept] = attention_forward_op().call(q, k, v, decay, state, reset, lengths, reverse, scale, false);
  return {y, last};
}

// ------------------------------------------------------------------------ Muon

constexpr const char* kMuon = "Muon step";
constexpr const char* kOrthogonalize = "orthogonalisation";

void check_dense(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_contiguous(), "The CUDA Muon step needs dense `", name, "`.");
}

void muon_step(at::TensorList params, at::TensorList grads, at::TensorList momenta, at::TensorList copies, double lr,
               double momentum, bool nesterov, double weight_decay, double a, double b, double c, double eps, int64_t steps,
               int64_t adjust, const OptTensor& grad_scale) {
  TORCH_CHECK_VALUE(params.size() == grads.size() && params.size() == momenta.size(),
                    "The CUDA Muon step needs a gradient and a momentum for every parameter, got ", params.size(), ", ",
                    grads.size(), " and ", momenta.size(), ".");
  TORCH_CHECK_VALUE(copies.empty() || copies.size() == params.size(),
                    "The CUDA Muon step needs a copy for every parameter or none, got ", copies.size(), ".");
  if (params.empty()) return;
  const at::Tensor& first = params[0];
  check_cuda(first, first, kMuon, "params");
  c10::cuda::CUDAGuard guard(first.device());
  pesq_muon_desc d{};
  d.nesterov = nesterov;
  d.adjust = static_cast<int32_t>(adjust);
  TORCH_CHECK_VALUE(steps >= 1 && steps <= 100, "The CUDA Muon step takes between 1 and 100 steps, got ", steps, ".");
  d.steps = static_cast<int32_t>(steps);
  d.momentum = momentum;
  d.lr = static_cast<float>(lr);
  d.weight_decay = static_cast<float>(weight_decay);
  d.eps = static_cast<float>(eps);
  d.a = static_cast<float>(a), d.b = static_cast<float>(b), d.c = static_cast<float>(c);
  if (given(grad_scale)) {
    check_cuda(*grad_scale, first, kMuon, "grad_scale");
    check_float(*grad_scale, kMuon, "grad_scale");
    TORCH_CHECK_VALUE(grad_scale->numel() == 1, "The CUDA Muon step needs one `grad_scale`.");
    d.grad_scale = grad_scale->data_ptr<float>();
  }
  std::vector<pesq_muon_tensor> table;
  std::vector<at::Tensor> dense;  // gradients that had to be copied
  table.reserve(params.size());
  bool typed = false;
  at::ScalarType type = at::kFloat;
  for (size_t i = 0; i < params.size(); ++i) {
    const at::Tensor &p = params[i], &m = momenta[i];
    at::Tensor g = grads[i];
    check_cuda(p, first, kMuon, "params");
    check_float(p, kMuon, "params");
    TORCH_CHECK_VALUE(p.dim() == 2, "The CUDA Muon step needs matrices, got `params` of shape ", p.sizes(), ".");
    check_dense(p, "params");
    if (!g.defined() || g.numel() == 0) continue;
    check_cuda(g, first, kMuon, "grads");
    check_shape(g, p.sizes(), kMuon, "grads");
    check_cuda(m, first, kMuon, "momenta");
    check_float(m, kMuon, "momenta");
    check_shape(m, p.sizes(), kMuon, "momenta");
    check_dense(m, "momenta");
    if (!typed) type = g.scalar_type(), d.grad_dtype = dtype_code(g, kMuon, "grads"), typed = true;
    TORCH_CHECK(g.scalar_type() == type, "The CUDA Muon step needs gradients of one type, got ", type, " and ",
                g.scalar_type(), ".");
    if (!g.is_contiguous()) {
      dense.push_back(g.contiguous());
      g = dense.back();
    }
    pesq_muon_tensor e{p.data_ptr<float>(), g.data_ptr(), m.data_ptr<float>(), nullptr, p.size(0), p.size(1)};
    if (!copies.empty()) {
      const at::Tensor& q = copies[i];
      check_cuda(q, first, kMuon, "copies");
      check_shape(q, p.sizes(), kMuon, "copies");
      check_dense(q, "copies");
      TORCH_CHECK(q.scalar_type() == type && type != at::kFloat,
                  "The CUDA Muon step needs copies in the gradients' 16-bit type, they are ", q.scalar_type(), ".");
      e.copy = q.data_ptr();
    }
    table.push_back(e);
  }
  const int64_t count = static_cast<int64_t>(table.size());
  size_t bytes = 0;
  check_status(pesq_muon_workspace(&d, table.data(), count, &bytes), "pesq_muon_workspace");
  if (!count) return;
  at::Tensor ws = at::empty({static_cast<int64_t>(bytes)}, first.options().dtype(at::kByte));
  check_status(pesq_muon_step(&d, table.data(), count, at::cuda::getCurrentCUDAStream(), ws.data_ptr(), bytes),
               "pesq_muon_step");
  for (size_t i = 0; i < params.size(); ++i) {
    if (!grads[i].defined() || grads[i].numel() == 0) continue;
    params[i].unsafeGetTensorImpl()->bump_version();
    momenta[i].unsafeGetTensorImpl()->bump_version();
    if (!copies.empty()) copies[i].unsafeGetTensorImpl()->bump_version();
  }
}

at::Tensor orthogonalize(const at::Tensor& x_, double a, double b, double c, double eps, int64_t steps) {
  check_cuda(x_, x_, kOrthogonalize, "x");
  pesq_orthogonalize_desc d{};
  d.dtype = dtype_code(x_, kOrthogonalize, "x");
  TORCH_CHECK_VALUE(x_.dim() >= 2, "The CUDA orthogonalisation needs `x` [..., row, column], got ", x_.sizes(), ".");
  TORCH_CHECK_VALUE(steps >= 1 && steps <= 100, "The CUDA orthogonalisation takes between 1 and 100 steps, got ", steps, ".");
  c10::cuda::CUDAGuard guard(x_.device());
  const at::Tensor x = x_.contiguous();
  at::Tensor out = at::empty(x.sizes(), x.options());
  if (x.numel() == 0) return out;
  d.rows = x.size(-2);
  d.cols = x.size(-1);
  d.count = x.numel() / (d.rows * d.cols);
  d.steps = static_cast<int32_t>(steps);
  d.eps = static_cast<float>(eps);
  d.a = static_cast<float>(a), d.b = static_cast<float>(b), d.c = static_cast<float>(c);
  size_t bytes = 0;
  check_status(pesq_orthogonalize_workspace(&d, &bytes), "pesq_orthogonalize_workspace");
  at::Tensor ws = at::empty({static_cast<int64_t>(bytes)}, x.options().dtype(at::kByte));
  check_status(pesq_orthogonalize(&d, at::cuda::getCurrentCUDAStream(), x.data_ptr(), out.data_ptr(), ws.data_ptr(), bytes),
               "pesq_orthogonalize");
  return out;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(pesq_cuda, m) {
  m.def(
      "muon_step(Tensor(a!)[] params, Tensor[] grads, Tensor(b!)[] momenta, Tensor(c!)[] copies, float lr, float momentum, "
      "bool nesterov, float weight_decay, float a, float b, float c, float eps, int steps, int adjust, Tensor? grad_scale) "
      "-> ()");
  m.def("orthogonalize(Tensor x, float a, float b, float c, float eps, int steps) -> Tensor");
}

TORCH_LIBRARY_FRAGMENT(pesq_cuda, m) {
  const char* in = "(Tensor q, Tensor k, Tensor v, Tensor log_decay, Tensor? state, Tensor? reset, Tensor? lengths, "
                   "bool reverse, float scale";
  m.def((std::string("linear_attention") + in + ") -> (Tensor, Tensor)").c_str());
  m.def((std::string("linear_attention_forward") + in + ", bool keep) -> (Tensor, Tensor, Tensor)").c_str());
  m.def((std::string("linear_attention_backward") + in +
         ", Tensor kept, Tensor? dy, Tensor? dlast) -> (Tensor, Tensor, Tensor, Tensor, Tensor)")
            .c_str());
}

TORCH_LIBRARY_FRAGMENT(pesq_cuda, m) {
  m.def("layer_norm(Tensor x, Tensor weight, Tensor? bias, float eps, int dtype) -> Tensor");
  m.def("layer_norm_forward(Tensor x, Tensor weight, Tensor? bias, float eps, int dtype) -> Tensor");
  m.def("layer_norm_backward(Tensor x, Tensor weight, Tensor? bias, float eps, int dtype, Tensor dy) -> "
        "(Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(pesq_cuda, CompositeImplicitAutograd, m) {
  m.impl("layer_norm", &layer_norm);
  m.impl("linear_attention", &linear_attention);
}

TORCH_LIBRARY_IMPL(pesq_cuda, CUDA, m) {
  m.impl("layer_norm_forward", &layer_norm_forward);
  m.impl("layer_norm_backward", &layer_norm_backward);
  m.impl("linear_attention_forward", &linear_attention_forward);
  m.impl("linear_attention_backward", &linear_attention_backward);
  m.impl("muon_step", &muon_step);
  m.impl("orthogonalize", &orthogonalize);
}
