// torch custom ops of the training operators over the C ABI of
// libpesq_cuda.so, with their autograd nodes.
//
// Every operator is three ops: the one a caller uses (composite: it records an
// autograd node when a gradient is wanted), and the forward and backward it is
// made of, which allocate with torch's caching allocator, take the current
// stream and call the C ABI.  Both check the shapes, types and devices of what
// they are given.
#include <algorithm>
#include <limits>

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include "../../include/pesq_cuda.h"

namespace {

using OptTensor = std::optional<at::Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

void check_status(int status, const char* what) {
  if (status == PESQ_OK) return;
  const char* msg = pesq_last_error();
  if (status == PESQ_ERR_INVALID_ARGUMENT) TORCH_CHECK_VALUE(false, what, ": ", msg);
  TORCH_CHECK(false, what, " failed (status ", status, "): ", msg);
}

int dtype_code(const at::Tensor& t, const char* op, const char* name) {
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

void check_cuda(const at::Tensor& t, const at::Tensor& first, const char* op, const char* name) {
  TORCH_CHECK(t.is_cuda(), "The CUDA ", op, " needs `", name, "` to live on a GPU.");
  TORCH_CHECK(t.device() == first.device(), "The CUDA ", op, " needs all tensors on one device, `", name, "` is on ",
              t.device(), ", not ", first.device(), ".");
}

void check_shape(const at::Tensor& t, at::IntArrayRef want, const char* op, const char* name) {
  TORCH_CHECK_VALUE(t.sizes() == want, "The CUDA ", op, " needs `", name, "` of shape ", want, ", got ", t.sizes(), ".");
}

void check_float(const at::Tensor& t, const char* op, const char* name) {
  TORCH_CHECK(t.scalar_type() == at::kFloat, "The CUDA ", op, " needs `", name, "` in float32, it is ", t.scalar_type(),
              ".");
}

bool given(const OptTensor& t) { return t.has_value() && t->defined(); }

void check_gradient(const at::Tensor& t, const at::Tensor& of, at::IntArrayRef want, const char* op, const char* name) {
  check_cuda(t, of, op, name);
  check_shape(t, want, op, name);
}

// channels adjacent, steps less than 2 GiB apart
at::Tensor rows(const at::Tensor& t) {
  const int64_t far = INT64_C(0x7fffffff) / t.element_size();
  const bool near = t.size(1) <= 1 || (t.stride(1) <= far && t.stride(1) >= -far);
  return near && (t.size(2) <= 1 || t.stride(2) == 1) ? t : t.contiguous();
}

// as aligned as a dense tensor (the pointer and every stride of more than one
// element a multiple of 16 bytes, or of what a row is), or a copy that is
at::Tensor aligned(const at::Tensor& t) {
  const int64_t size = t.element_size();
  int64_t unit = 16 / size;
  while (t.size(2) % unit) unit /= 2;
  const auto good = [&](int64_t n, int64_t stride) { return n <= 1 || (stride > 0 && stride % unit == 0); };
  const bool ok = reinterpret_cast<uintptr_t>(t.data_ptr()) % (unit * size) == 0 && good(t.size(0), t.stride(0)) &&
                  good(t.size(1), t.stride(1));
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

pesq_stream stream_of(const at::Tensor& t) { return {t.data_ptr(), t.stride(0), t.stride(1)}; }

const float* floats(const OptTensor& t) { return t.has_value() && t->defined() ? t->data_ptr<float>() : nullptr; }

OptTensor optional_of(const Variable& v) { return v.defined() ? OptTensor(v) : std::nullopt; }

void no_second_derivative(const char* op) {
  TORCH_CHECK(!at::GradMode::is_enabled(), "The CUDA ", op, " has no second derivative (create_graph=True).");
}

bool has_tangent(const at::Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }
bool has_tangent(const OptTensor& t) { return t.has_value() && has_tangent(*t); }
template <class... Ts>
void no_forward_mode(const char* op, const Ts&... inputs) {
  TORCH_CHECK(!(has_tangent(inputs) || ...), "The CUDA ", op, " has no forward-mode derivative.");
}

bool wants_grad(const at::Tensor& t) { return t.requires_grad(); }
bool wants_grad(const OptTensor& t) { return t.has_value() && t->defined() && t->requires_grad(); }

// ------------------------------------------------------------------ gated scan

constexpr const char* kScan = "gated scan";

struct ScanCall {
  at::Tensor x, ig, rg, decay, state, reset, lengths;
  pesq_gated_scan_desc d{};

  ScanCall(const at::Tensor& x_, const at::Tensor& ig_, const at::Tensor& rg_, const at::Tensor& decay_,
           const OptTensor& state_, const OptTensor& reset_, const OptTensor& lengths_, bool reverse, double rate) {
    check_cuda(x_, x_, kScan, "x");
    d.dtype = dtype_code(x_, kScan, "x");
    TORCH_CHECK(x_.dim() == 3, "The CUDA gated scan needs `x` [batch, step, channel], got ", x_.sizes(), ".");
    check_cuda(ig_, x_, kScan, "input_gate");
    check_cuda(rg_, x_, kScan, "decay_gate");
    check_cuda(decay_, x_, kScan, "decay");
    check_shape(ig_, x_.sizes(), kScan, "input_gate");
    check_shape(rg_, x_.sizes(), kScan, "decay_gate");
    check_shape(decay_, {x_.size(2)}, kScan, "decay");
    check_float(decay_, kScan, "decay");
    TORCH_CHECK(ig_.scalar_type() == x_.scalar_type() && rg_.scalar_type() == x_.scalar_type(),
                "The CUDA gated scan needs `x` and the gates in one type, got ", x_.scalar_type(), ", ",
                ig_.scalar_type(), " and ", rg_.scalar_type(), ".");
    TORCH_CHECK_VALUE(rate > 0.0 && rate <= 1e6, "The CUDA gated scan needs a `rate` above 0 and up to 1e6, got ", rate, ".");
    x = rows(x_);
    ig = rows(ig_);
    rg = rows(rg_);
    decay = decay_.contiguous();
    d.batch = x.size(0);
    d.steps = x.size(1);
    d.width = x.size(2);
    if (state_.has_value() && state_->defined()) {
      check_cuda(*state_, x_, kScan, "state");
      check_float(*state_, kScan, "state");
      check_shape(*state_, {d.batch, d.width}, kScan, "state");
      state = state_->contiguous();
      d.state = state.data_ptr<float>();
    }
    if (reset_.has_value() && reset_->defined()) {
      check_cuda(*reset_, x_, kScan, "reset");
      check_shape(*reset_, {d.batch, d.steps}, kScan, "reset");
      TORCH_CHECK(reset_->scalar_type() == at::kBool, "The CUDA gated scan needs `reset` in bool, it is ",
                  reset_->scalar_type(), ".");
      reset = *reset_;
      d.reset = static_cast<const uint8_t*>(reset.data_ptr());
      d.reset_batch_stride = reset.stride(0);
      d.reset_step_stride = reset.stride(1);
    }
    if (lengths_.has_value() && lengths_->defined()) {
      check_cuda(*lengths_, x_, kScan, "lengths");
      check_shape(*lengths_, {d.batch}, kScan, "lengths");
      TORCH_CHECK(lengths_->scalar_type() == at::kLong || lengths_->scalar_type() == at::kInt,
                  "The CUDA gated scan needs `lengths` in int64 or int32, it is ", lengths_->scalar_type(), ".");
      lengths = lengths_->to(at::kLong).contiguous();
      d.lengths = lengths.data_ptr<int64_t>();
    }
    d.reverse = reverse;
    d.rate = static_cast<float>(rate);
    d.x = stream_of(x);
    d.input_gate = stream_of(ig);
    d.decay_gate = stream_of(rg);
    d.decay = decay.data_ptr<float>();
  }

  bool empty() const { return d.batch == 0 || d.steps == 0 || d.width == 0; }

  // Rows go to the C entries in parts of about one size, which they then treat alike: as few as their
  // limit of 65535 rows allows, and a multiple of 8 rows each, so that a part of what is kept is aligned
  int64_t parts() const { return (d.batch + 65527) / 65528; }
  int64_t part_rows() const { return ((d.batch + parts() - 1) / parts() + 7) / 8 * 8; }
  // bytes of the states that a forward keeps of n rows
  int64_t kept(int64_t n) const { return (n * ((d.steps + 7) / 8) * d.width * 4 + 15) / 16 * 16; }
  pesq_gated_scan_desc part(int64_t first) const {
    pesq_gated_scan_desc e = d;
    e.batch = std::min(part_rows(), d.batch - first);
    const auto move = [&](pesq_stream& s) {
      s.data = static_cast<const char*>(s.data) + first * s.batch_stride * x.element_size();
    };
    move(e.x), move(e.input_gate), move(e.decay_gate);
    if (e.state) e.state += first * d.width;
    if (e.reset) e.reset += first * d.reset_batch_stride;
    if (e.lengths) e.lengths += first;
    return e;
  }
  // where the results of the rows from `first` on go, of a dense tensor
  static char* at(const at::Tensor& t, int64_t first) {
    return t.defined() ? static_cast<char*>(t.data_ptr()) + first * t.stride(0) * t.element_size() : nullptr;
  }
};

// Steps between the states that this thread's last forward kept; 0 where a tracer stood in for it
thread_local int64_t scan_kept_steps = 0;

// (y, last, the states kept for the backward where `keep`)
std::tuple<at::Tensor, at::Tensor, at::Tensor> gated_scan_forward(const at::Tensor& x, const at::Tensor& ig,
                                                                  const at::Tensor& rg, const at::Tensor& decay,
                                                                  const OptTensor& state, const OptTensor& reset,
                                                                  const OptTensor& lengths, bool reverse, double rate,
                                                                  bool keep) {
  ScanCall c(x, ig, rg, decay, state, reset, lengths, reverse, rate);
  c10::cuda::CUDAGuard guard(x.device());
  const auto f32 = x.options().dtype(at::kFloat), bytes = x.options().dtype(at::kByte);
  at::Tensor y = at::empty(x.sizes(), x.options());
  at::Tensor last = at::empty({c.d.batch, c.d.width}, f32);
  if (c.empty()) {
    if (c.d.state) {
      last.copy_(c.state);
    } else {
      last.zero_();
    }
    return {y, last, at::empty({0}, bytes)};
  }
  size_t work = 0, kept = 0, back = 0;
  pesq_gated_scan_desc d = c.part(0);
  check_status(pesq_gated_scan_sizes(&d, &work, &kept, &back), "pesq_gated_scan_sizes");
  at::Tensor states = at::empty({keep ? c.kept(c.d.batch) : 0}, bytes), ws;
  if (work) ws = at::empty({static_cast<int64_t>(work)}, bytes);
  if (keep) {
    int32_t here = 0, most = 0;
    check_status(pesq_gated_scan_kept_steps(&d, &here, &most), "pesq_gated_scan_kept_steps");
    scan_kept_steps = here;
  }
  for (int64_t first = 0; first < c.d.batch; first += c.part_rows()) {
    if (first > 0) d = c.part(first);
    check_status(pesq_gated_scan_forward(&d, at::cuda::getCurrentCUDAStream(), ScanCall::at(y, first),
                                         last.data_ptr<float>() + first * c.d.width,
                                         keep ? static_cast<char*>(states.data_ptr()) + c.kept(first) : nullptr,
                                         keep ? c.kept(d.batch) : 0, work ? ws.data_ptr() : nullptr, work),
                 "pesq_gated_scan_forward");
  }
  return {y, last, states};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> gated_scan_backward(
    const at::Tensor& x, const at::Tensor& ig, const at::Tensor& rg, const at::Tensor& decay, const OptTensor& state,
    const OptTensor& reset, const OptTensor& lengths, bool reverse, double rate, const at::Tensor& kept,
    int64_t kept_steps, const OptTensor& dy_, const OptTensor& dlast_) {
  ScanCall c(x, ig, rg, decay, state, reset, lengths, reverse, rate);
  c10::cuda::CUDAGuard guard(x.device());
  const auto f32 = x.options().dtype(at::kFloat);
  at::Tensor dx = at::empty(x.sizes(), x.options()), dig = at::empty(x.sizes(), x.options()),
             drg = at::empty(x.sizes(), x.options());
  at::Tensor ddecay = at::empty({c.d.width}, f32), dstate = at::empty({c.d.batch, c.d.width}, f32);
  at::Tensor dlast;
  if (given(dy_)) check_gradient(*dy_, x, x.sizes(), kScan, "dy");
  if (given(dlast_)) {
    check_gradient(*dlast_, x, {c.d.batch, c.d.width}, kScan, "dlast");
    dlast = dlast_->to(at::kFloat).contiguous();
  }
  if (c.empty()) {
    ddecay.zero_();
    if (dlast.defined()) {
      dstate.copy_(dlast);
    } else {
      dstate.zero_();
    }
    return {dx, dig, drg, ddecay, dstate};
  }
  at::Tensor dy;
  pesq_stream dys{nullptr, 0, 0};
  if (given(dy_)) {
    dy = aligned(rows(dy_->to(x.scalar_type())));
    dys = stream_of(dy);
  }
  size_t work = 0, states = 0, back = 0;
  pesq_gated_scan_desc d = c.part(0);
  check_status(pesq_gated_scan_sizes(&d, &work, &states, &back), "pesq_gated_scan_sizes");
  check_cuda(kept, x, kScan, "kept");
  TORCH_CHECK(kept.scalar_type() == at::kByte && kept.is_contiguous() && kept.numel() == c.kept(c.d.batch),
              "The CUDA gated scan needs the states that its forward kept.");
  at::Tensor ws = at::empty({static_cast<int64_t>(back)}, f32.dtype(at::kByte)), before = kept;
  // (hooks on what autograd saves, or a compiler, may bring the streams back in another layout than the forward's,
  // one that asks for states closer together)
  int32_t here = 0, most = 0;
  check_status(pesq_gated_scan_kept_steps(&d, &here, &most), "pesq_gated_scan_kept_steps");
  if ((kept_steps > 0 ? kept_steps : most) > here)
    before = std::get<2>(gated_scan_forward(x, ig, rg, decay, state, reset, lengths, reverse, rate, true));
  at::Tensor sums;  // of the parts
  if (c.parts() > 1) sums = at::empty({c.parts(), c.d.width}, f32);
  for (int64_t first = 0, k = 0; first < c.d.batch; first += c.part_rows(), ++k) {
    if (first > 0) d = c.part(first);
    pesq_stream part = dys;
    if (part.data) part.data = ScanCall::at(dy, first);
    check_status(pesq_gated_scan_backward(&d, at::cuda::getCurrentCUDAStream(),
                                          static_cast<const char*>(before.data_ptr()) + c.kept(first), c.kept(d.batch), part,
                                          dlast.defined() ? dlast.data_ptr<float>() + first * c.d.width : nullptr,
                                          ScanCall::at(dx, first), ScanCall::at(dig, first), ScanCall::at(drg, first),
                                          c.parts() > 1 ? sums.data_ptr<float>() + k * c.d.width : ddecay.data_ptr<float>(),
                                          dstate.data_ptr<float>() + first * c.d.width, ws.data_ptr(), back),
                 "pesq_gated_scan_backward");
  }
  if (c.parts() > 1) ddecay = sums.sum(0);
  return {dx, dig, drg, ddecay, dstate};
}

const auto& scan_forward_op() {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("pesq_cuda::gated_scan_forward", "")
                       .typed<decltype(gated_scan_forward)>();
  return op;
}
const auto& scan_backward_op() {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("pesq_cuda::gated_scan_backward", "")
                       .typed<decltype(gated_scan_backward)>();
  return op;
}

struct GatedScan : public torch::autograd::Function<GatedScan> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& ig, const at::Tensor& rg,
                               const at::Tensor& decay, const OptTensor& state, const OptTensor& reset,
                               const OptTensor& lengths, bool reverse, double rate) {
    at::AutoDispatchBelowADInplaceOrView below;
    scan_kept_steps = 0;
    auto [y, last, kept] = scan_forward_op().call(x, ig, rg, decay, state, reset, lengths, reverse, rate, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, ig, rg, decay, state.value_or(at::Tensor()), reset.value_or(at::Tensor()),
                            lengths.value_or(at::Tensor()), kept});
    ctx->saved_data["reverse"] = reverse;
    ctx->saved_data["rate"] = rate;
    ctx->saved_data["kept_steps"] = scan_kept_steps;
    return {y, last};
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    no_second_derivative(kScan);
    const auto s = ctx->get_saved_variables();
    variable_list out(9);
    if (!g[0].defined() && !g[1].defined()) return out;
    auto [dx, dig, drg, ddecay, dstate] = scan_backward_op().call(
        s[0], s[1], s[2], s[3], optional_of(s[4]), optional_of(s[5]), optional_of(s[6]),
        ctx->saved_data["reverse"].toBool(), ctx->saved_data["rate"].toDouble(), s[7],
        ctx->saved_data["kept_steps"].toInt(), optional_of(g[0]), optional_of(g[1]));
    out[0] = dx;
    out[1] = dig;
    out[2] = drg;
    out[3] = ddecay;
    if (s[4].defined()) out[4] = dstate;
    return out;
  }
};

std::tuple<at::Tensor, at::Tensor> gated_scan(const at::Tensor& x, const at::Tensor& ig, const at::Tensor& rg,
                                              const at::Tensor& decay, const OptTensor& state, const OptTensor& reset,
                                              const OptTensor& lengths, bool reverse, double rate) {
  check_cuda(x, x, kScan, "x");
  no_forward_mode(kScan, x, ig, rg, decay, state);
  if (at::GradMode::is_enabled() &&
      (wants_grad(x) || wants_grad(ig) || wants_grad(rg) || wants_grad(decay) || wants_grad(state))) {
    auto out = GatedScan::apply(x, ig, rg, decay, state, reset, lengths, reverse, rate);
    return {out[0], out[1]};
  }
  auto [y, last, kept] = scan_forward_op().call(x, ig, rg, decay, state, reset, lengths, reverse, rate, false);
  return {y, last};
}

// ------------------------------------------------------------------- norm join

constexpr const char* kJoin = "norm join";

struct JoinCall {
  at::Tensor x, z, g, post, pre, scale;
  pesq_norm_join_desc d{};
  at::ScalarType out;

  at::Tensor vector(const at::Tensor& t, const char* name) {
    check_cuda(t, x, kJoin, name);
    check_float(t, kJoin, name);
    check_shape(t, {x.size(2)}, kJoin, name);
    return t.contiguous();
  }

  JoinCall(const at::Tensor& x_, const OptTensor& z_, const OptTensor& g_, const OptTensor& post_,
           const at::Tensor& pre_, const OptTensor& scale_, double eps, bool silu, bool shared, int64_t dtype) {
    check_cuda(x_, x_, kJoin, "stream");
    TORCH_CHECK(x_.dim() == 3, "The CUDA norm join needs `stream` [batch, step, channel], got ", x_.sizes(), ".");
    d.stream_dtype = dtype_code(x_, kJoin, "stream");
    d.dtype = static_cast<int32_t>(dtype);
    out = dtype == PESQ_F32 ? at::kFloat : dtype == PESQ_BF16 ? at::kBFloat16 : at::kHalf;
    TORCH_CHECK_VALUE(eps >= 0.0, "The CUDA norm join needs an `eps` that is not negative, got ", eps, ".");
    TORCH_CHECK(x_.scalar_type() == at::kFloat || x_.scalar_type() == out,
                "The CUDA norm join needs `stream` in float32 or in the block's type, it is ", x_.scalar_type(), ".");
    x = rows(x_);
    d.batch = x.size(0);
    d.steps = x.size(1);
    d.width = x.size(2);
    d.activation = silu ? PESQ_SILU : PESQ_SIGMOID;
    d.gate_shared = shared;
    d.eps = static_cast<float>(eps);
    d.stream = stream_of(x);
    pre = vector(pre_, "pre_weight");
    d.pre = pre.data_ptr<float>();
    if (!given(z_)) {
      TORCH_CHECK_VALUE(!given(g_), "The CUDA norm join needs a `block` for its `gate`.");
      return;
    }
    check_cuda(*z_, x, kJoin, "block");
    check_shape(*z_, x.sizes(), kJoin, "block");
    TORCH_CHECK(z_->scalar_type() == out, "The CUDA norm join needs `block` in ", out, ", it is ", z_->scalar_type(), ".");
    z = rows(*z_);
    d.block = stream_of(z);
    TORCH_CHECK_VALUE(given(post_), "The CUDA norm join needs `post_weight`.");
    post = vector(*post_, "post_weight");
    d.post = post.data_ptr<float>();
    if (given(g_)) {
      check_cuda(*g_, x, kJoin, "gate");
      const int64_t want[3] = {d.batch, shared ? 1 : d.steps, d.width};
      check_shape(*g_, want, kJoin, "gate");
      TORCH_CHECK(g_->scalar_type() == out, "The CUDA norm join needs `gate` in the block's type ", out, ", it is ",
                  g_->scalar_type(), ".");
      g = rows(*g_);
      d.gate = stream_of(g);
    }
    if (given(scale_)) {
      scale = vector(*scale_, "scale");
      d.scale = scale.data_ptr<float>();
    }
  }

  bool empty() const { return x.numel() == 0; }
};

// (stream', normed); stream' is empty without a block
std::tuple<at::Tensor, at::Tensor> norm_join_forward(const at::Tensor& x, const OptTensor& z, const OptTensor& g,
                                                     const OptTensor& post, const at::Tensor& pre,
                                                     const OptTensor& scale, double eps, bool silu, bool shared,
                                                     int64_t dtype) {
  JoinCall c(x, z, g, post, pre, scale, eps, silu, shared, dtype);
  c10::cuda::CUDAGuard guard(x.device());
  at::Tensor out = c.z.defined() ? at::empty(x.sizes(), x.options()) : at::empty({0}, x.options());
  at::Tensor normed = at::empty(x.sizes(), x.options().dtype(c.out));
  if (!c.empty())
    check_status(pesq_norm_join_forward(&c.d, at::cuda::getCurrentCUDAStream(),
                                        c.z.defined() ? out.data_ptr() : nullptr, normed.data_ptr()),
                 "pesq_norm_join_forward");
  return {out, normed};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> norm_join_backward(
    const at::Tensor& x, const OptTensor& z, const OptTensor& g, const OptTensor& post, const at::Tensor& pre,
    const OptTensor& scale, double eps, bool silu, bool shared, int64_t dtype, const OptTensor& dstream_,
    const OptTensor& dnormed_) {
  JoinCall c(x, z, g, post, pre, scale, eps, silu, shared, dtype);
  c10::cuda::CUDAGuard guard(x.device());
  const auto make = [&](const at::Tensor& t) {
    return t.defined() ? at::empty(t.sizes(), t.options()) : at::empty({0}, x.options());
  };
  at::Tensor dx = make(c.x), dz = make(c.z), dg = make(c.g), dpost = make(c.post), dpre = make(c.pre),
             dscale = make(c.scale);
  if (c.empty()) {
    for (at::Tensor* t : {&dpost, &dpre, &dscale, &dg}) t->zero_();
    return {dx, dz, dg, dpost, dpre, dscale};
  }
  at::Tensor ds, dn;
  pesq_stream s{nullptr, 0, 0}, n{nullptr, 0, 0};
  if (given(dstream_)) {
    check_gradient(*dstream_, x, x.sizes(), kJoin, "dstream");
    ds = rows(dstream_->to(x.scalar_type()));
    s = stream_of(ds);
  }
  if (given(dnormed_)) {
    check_gradient(*dnormed_, x, x.sizes(), kJoin, "dnormed");
    dn = rows(dnormed_->to(c.out));
    n = stream_of(dn);
  }
  size_t bytes = 0;
  check_status(pesq_norm_join_workspace(&c.d, &bytes), "pesq_norm_join_workspace");
  at::Tensor ws = at::empty({static_cast<int64_t>(bytes)}, x.options().dtype(at::kByte));
  const auto vec = [](const at::Tensor& have, at::Tensor& t) { return have.defined() ? t.data_ptr<float>() : nullptr; };
  check_status(pesq_norm_join_backward(&c.d, at::cuda::getCurrentCUDAStream(), s, n, dx.data_ptr(),
                                       c.z.defined() ? dz.data_ptr() : nullptr,
                                       c.g.defined() ? dg.data_ptr() : nullptr, vec(c.post, dpost), vec(c.pre, dpre),
                                       vec(c.scale, dscale), ws.data_ptr(), bytes),
               "pesq_norm_join_backward");
  return {dx, dz, dg, dpost, dpre, dscale};
}

const auto& join_forward_op() {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("pesq_cuda::norm_join_forward", "")
                       .typed<decltype(norm_join_forward)>();
  return op;
}
const auto& join_backward_op() {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("pesq_cuda::norm_join_backward", "")
                       .typed<decltype(norm_join_backward)>();
  return op;
}

struct NormJoin : public torch::autograd::Function<NormJoin> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const OptTensor& z, const OptTensor& g,
                               const OptTensor& post, const at::Tensor& pre, const OptTensor& scale, double eps,
                               bool silu, bool shared, int64_t dtype) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [out, normed] = join_forward_op().call(x, z, g, post, pre, scale, eps, silu, shared, dtype);
    const auto or_none = [](const OptTensor& t) { return t.value_or(at::Tensor()); };
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, or_none(z), or_none(g), or_none(post), pre, or_none(scale)});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["silu"] = silu;
    ctx->saved_data["shared"] = shared;
    ctx->saved_data["dtype"] = dtype;
    return {out, normed};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grad) {
    no_second_derivative(kJoin);
    const auto s = ctx->get_saved_variables();
    variable_list out(10);
    if (!grad[0].defined() && !grad[1].defined()) return out;
    const OptTensor dstream = s[1].defined() ? optional_of(grad[0]) : std::nullopt;
    auto [dx, dz, dg, dpost, dpre, dscale] = join_backward_op().call(
        s[0], optional_of(s[1]), optional_of(s[2]), optional_of(s[3]), s[4], optional_of(s[5]),
        ctx->saved_data["eps"].toDouble(), ctx->saved_data["silu"].toBool(), ctx->saved_data["shared"].toBool(),
        ctx->saved_data["dtype"].toInt(), dstream, optional_of(grad[1]));
    out[0] = dx;
    if (s[1].defined()) out[1] = dz, out[3] = dpost;
    if (s[2].defined()) out[2] = dg;
    out[4] = dpre;
    if (s[1].defined() && s[5].defined()) out[5] = dscale;
    return out;
  }
};

std::tuple<at::Tensor, at::Tensor> norm_join(const at::Tensor& x, const OptTensor& z, const OptTensor& g_,
                                             const OptTensor& post, const at::Tensor& pre, const OptTensor& scale,
                                             double eps, bool silu, int64_t dtype) {
  check_cuda(x, x, kJoin, "stream");
  TORCH_CHECK(x.dim() == 3, "The CUDA norm join needs `stream` [batch, step, channel], got ", x.sizes(), ".");
  no_forward_mode(kJoin, x, z, g_, post, pre, scale);
  // one gate row for all steps of a batch item is summed by the kernels, any other broadcast by torch
  OptTensor g = g_;
  bool shared = false;
  if (given(g) && g->sizes() != x.sizes()) {
    shared = g->dim() == 3 && g->size(0) == x.size(0) && g->size(1) == 1 && g->size(2) == x.size(2);
    if (!shared) g = g->expand(x.sizes());
  }
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(z) || wants_grad(g) || wants_grad(post) ||
                                     wants_grad(pre) || wants_grad(scale))) {
    auto out = NormJoin::apply(x, z, g, post, pre, scale, eps, silu, shared, dtype);
    return {out[0], out[1]};
  }
  return join_forward_op().call(x, z, g, post, pre, scale, eps, silu, shared, dtype);
}

// ---------------------------------------------------------------------- AdamW

constexpr const char* kAdam = "AdamW step";

void check_dense(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_contiguous(), "The CUDA AdamW step needs dense `", name, "`.");
}

void adamw_step(at::TensorList params, at::TensorList grads, const at::Tensor& moment1, const at::Tensor& moment2,
                const at::Tensor& step, const OptTensor& scales, at::TensorList copies, double lr, double beta1,
                double beta2, double eps, double decay, const OptTensor& grad_scale, int64_t seed) {
  TORCH_CHECK_VALUE(params.size() == grads.size(), "The CUDA AdamW step needs a gradient for every parameter, got ",
                    params.size(), " and ", grads.size(), ".");
  TORCH_CHECK_VALUE(copies.empty() || copies.size() == params.size(),
                    "The CUDA AdamW step needs a copy for every parameter or none, got ", copies.size(), ".");
  check_cuda(moment1, moment1, kAdam, "moment1");
  check_cuda(moment2, moment1, kAdam, "moment2");
  check_cuda(step, moment1, kAdam, "step");
  check_dense(moment1, "moment1");
  check_dense(moment2, "moment2");
  check_dense(step, "step");
  TORCH_CHECK(step.scalar_type() == at::kLong && step.numel() == 2,
              "The CUDA AdamW step needs `step` as two int64 values.");
  TORCH_CHECK_VALUE(moment1.numel() == moment2.numel() && moment1.numel() % 256 == 0,
                    "The CUDA AdamW step needs moments of one size, a multiple of 256, got ", moment1.numel(), " and ",
                    moment2.numel(), ".");
  pesq_adamw_desc d{};
  d.units = moment1.numel() / 256;
  const bool eight = moment1.scalar_type() == at::kFloat8_e4m3fn;
  TORCH_CHECK(moment1.scalar_type() == moment2.scalar_type() && (eight || moment1.scalar_type() == at::kFloat),
              "The CUDA AdamW step needs both moments in float32 or float8_e4m3fn, they are ", moment1.scalar_type(),
              " and ", moment2.scalar_type(), ".");
  d.state_bits = eight ? 8 : 32;
  if (eight) {
    TORCH_CHECK_VALUE(given(scales), "The CUDA AdamW step needs `scales` for 8-bit moments.");
    check_cuda(*scales, moment1, kAdam, "scales");
    check_float(*scales, kAdam, "scales");
    const int64_t want[2] = {2, d.units};
    check_shape(*scales, want, kAdam, "scales");
    check_dense(*scales, "scales");
    d.scale1 = scales->data_ptr<float>();
    d.scale2 = d.scale1 + d.units;
  }
  if (given(grad_scale)) {
    check_cuda(*grad_scale, moment1, kAdam, "grad_scale");
    check_float(*grad_scale, kAdam, "grad_scale");
    TORCH_CHECK_VALUE(grad_scale->numel() == 1, "The CUDA AdamW step needs one `grad_scale`.");
    d.grad_scale = grad_scale->data_ptr<float>();
  }
  std::vector<pesq_adamw_tensor> table;
  std::vector<at::Tensor> dense;  // gradients that had to be copied
  table.reserve(params.size());
  bool typed = false;
  at::ScalarType type = at::kFloat;
  for (size_t i = 0; i < params.size(); ++i) {
    const at::Tensor& p = params[i];
    const at::Tensor* g = &grads[i];
    check_cuda(p, moment1, kAdam, "params");
    check_float(p, kAdam, "params");
    check_dense(p, "params");
    pesq_adamw_tensor e{p.data_ptr<float>(), nullptr, nullptr, p.numel()};
    if (g->defined() && g->numel() > 0) {
      check_cuda(*g, moment1, kAdam, "grads");
      check_shape(*g, p.sizes(), kAdam, "grads");
      if (!typed) type = g->scalar_type(), d.grad_dtype = dtype_code(*g, kAdam, "grads"), typed = true;
      TORCH_CHECK(g->scalar_type() == type, "The CUDA AdamW step needs gradients of one type, got ", type, " and ",
                  g->scalar_type(), ".");
      if (!g->is_contiguous()) {
        c10::cuda::CUDAGuard guard(moment1.device());
        dense.push_back(g->contiguous());
        g = &dense.back();
      }
      e.grad = g->data_ptr();
      if (!copies.empty()) {
        const at::Tensor& c = copies[i];
        check_cuda(c, moment1, kAdam, "copies");
        check_shape(c, p.sizes(), kAdam, "copies");
        check_dense(c, "copies");
        TORCH_CHECK(c.scalar_type() == type && type != at::kFloat,
                    "The CUDA AdamW step needs copies in the gradients' 16-bit type, they are ", c.scalar_type(), ".");
        e.copy = c.data_ptr();
        c.unsafeGetTensorImpl()->bump_version();
      }
      p.unsafeGetTensorImpl()->bump_version();
    }
    table.push_back(e);
  }
  d.moment1 = moment1.data_ptr();
  d.moment2 = moment2.data_ptr();
  d.step = step.data_ptr<int64_t>();
  d.beta1 = beta1;
  d.beta2 = beta2;
  d.lr = static_cast<float>(lr);
  d.eps = static_cast<float>(eps);
  d.weight_decay = static_cast<float>(decay);
  d.seed = static_cast<uint32_t>(seed);
  c10::cuda::CUDAGuard guard(moment1.device());
  check_status(pesq_adamw_step(&d, table.data(), static_cast<int64_t>(table.size()), at::cuda::getCurrentCUDAStream()),
               "pesq_adamw_step");
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(pesq_cuda, m) {
  const char* scan_in =
      "(Tensor x, Tensor input_gate, Tensor decay_gate, Tensor decay, Tensor? state, Tensor? reset, Tensor? lengths, "
      "bool reverse, float rate";
  m.def((std::string("gated_scan") + scan_in + ") -> (Tensor, Tensor)").c_str());
  m.def((std::string("gated_scan_forward") + scan_in + ", bool keep) -> (Tensor, Tensor, Tensor)").c_str());
  m.def((std::string("gated_scan_backward") + scan_in +
         ", Tensor kept, int kept_steps, Tensor? dy, Tensor? dlast) -> (Tensor, Tensor, Tensor, Tensor, Tensor)")
            .c_str());
  const char* join_in = "(Tensor stream, Tensor? block, Tensor? gate, Tensor? post, Tensor pre, Tensor? scale, float eps, bool silu";
  m.def((std::string("norm_join") + join_in + ", int dtype) -> (Tensor, Tensor)").c_str());
  m.def((std::string("norm_join_forward") + join_in + ", bool shared, int dtype) -> (Tensor, Tensor)").c_str());
  m.def((std::string("norm_join_backward") + join_in +
         ", bool shared, int dtype, Tensor? dstream, Tensor? dnormed) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)")
            .c_str());
}

TORCH_LIBRARY_FRAGMENT(pesq_cuda, m) {
  m.def(
      "adamw_step(Tensor(a!)[] params, Tensor[] grads, Tensor(b!) moment1, Tensor(c!) moment2, Tensor(d!) step, "
      "Tensor(e!)? scales, Tensor(f!)[] copies, float lr, float beta1, float beta2, float eps, float weight_decay, "
      "Tensor? grad_scale, int seed) -> ()");
}

TORCH_LIBRARY_IMPL(pesq_cuda, CompositeImplicitAutograd, m) {
  m.impl("gated_scan", &gated_scan);
  m.impl("norm_join", &norm_join);
}

TORCH_LIBRARY_IMPL(pesq_cuda, CUDA, m) {
  m.impl("gated_scan_forward", &gated_scan_forward);
  m.impl("gated_scan_backward", &gated_scan_backward);
  m.impl("norm_join_forward", &norm_join_forward);
  m.impl("norm_join_backward", &norm_join_backward);
  m.impl("adamw_step", &adamw_step);
}
