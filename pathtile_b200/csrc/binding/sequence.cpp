// sequence.cpp -- the sequence operators' checks, autograd nodes and calls on
// torch tensors: what pathtile_b200/sequence.py documents.  A call of a single
// token takes the GPU two to three microseconds, so everything around it is
// done here and not in Python.  The kernels are behind the C ABI of
// libpathtile_b200.so.
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <optional>
#include <string>
#include <vector>

#include "pathtile_b200.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// ---------------------------------------------------------------- arguments
int type_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return PT_F32;
    case at::kBFloat16: return PT_BF16;
    case at::kHalf: return PT_F16;
    default: return -1;
  }
}

// A node takes what may be absent as an optional: an undefined tensor it would count as an input.
Tensor given(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
OptTensor maybe(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }
const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* out_ptr(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
template <class T>
T* out_as(const Tensor& t) { return static_cast<T*>(out_ptr(t)); }
template <class T>
const T* as(const Tensor& t) { return static_cast<const T*>(ptr(t)); }

void activation(const Tensor& t, const char* name, int64_t ndim) {
  TORCH_CHECK_VALUE(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK_VALUE(type_code(t) >= 0, name, ": only float32, bfloat16 and float16 are supported, got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.dim() == ndim, name, " must have ", ndim, " dimensions, got shape ", t.sizes());
}

void like(const Tensor& t, const char* name, at::IntArrayRef shape, at::ScalarType type, const Tensor& x) {
  if (!t.defined()) return;
  TORCH_CHECK_VALUE(t.sizes() == shape, name, " must have shape ", shape, ", got ", t.sizes());
  TORCH_CHECK_VALUE(t.scalar_type() == type, name, " must be ", type, ", got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.device() == x.device(), name, " must be on ", x.device(), ", got ", t.device());
}

// t with contiguous channels: itself where they are.
Tensor rows(const Tensor& t) {
  return !t.defined() || t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous();
}
Tensor dense(const Tensor& t) { return t.defined() ? t.contiguous() : t; }

bool wants_grad(std::initializer_list<Tensor> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor& t : tensors)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}
void refuse_grad(const char* what, std::initializer_list<Tensor> tensors) {
  TORCH_CHECK_VALUE(!wants_grad(tensors), what, " has no backward pass: call it under torch.no_grad()");
}

// A cache [rows, a, b] that a step updates in place; returns the elements between its rows.
int64_t cache_row(const Tensor& t, int64_t a, int64_t b, at::ScalarType type, const Tensor& x) {
  TORCH_CHECK_VALUE(t.dim() == 3 && t.size(1) == a && t.size(2) == b, "state must have shape (rows, ", a, ", ", b,
                    "), got ", t.sizes());
  TORCH_CHECK_VALUE(t.scalar_type() == type && t.device() == x.device(), "state must be ", type, " on ", x.device(),
                    ", got ", t.scalar_type(), " on ", t.device());
  const int64_t n = t.size(0), row = t.stride(0);
  if (a * b > 0 && n > 0)
    TORCH_CHECK_VALUE((b == 1 || t.stride(2) == 1) && (a == 1 || t.stride(1) == b) && (n == 1 || row >= a * b),
                      "state is updated in place: each of its rows must be contiguous and none may overlap");
  return row;
}

// The kernel wrote to it behind torch's back: what autograd saved of it is no longer that.
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

Tensor slots_of(const Tensor& slots, int64_t batch, int64_t n, const Tensor& x) {
  if (!slots.defined()) {
    TORCH_CHECK_VALUE(n == batch, "state has ", n, " rows for a batch of ", batch, ": pass slots to choose among them");
    return slots;
  }
  like(slots, "slots", {batch}, at::kInt, x);
  return slots.contiguous();
}

// The kernels count a little past a row's end in 32 bits.
int as_int(int64_t v, const char* what) {
  TORCH_CHECK_VALUE(v <= INT_MAX - 4096, what, " is too large: ", v);
  return static_cast<int>(v);
}

// ---------------------------------------------------------------- launches
void check(int status, const char* what) {
  if (status == PT_OK) return;
  std::string detail = status == PT_ERR_CUDA ? " (cuda error " + std::to_string(pt_last_cuda_error()) + ")" : "";
  TORCH_CHECK(false, what, " failed with status ", status, ": ", pt_status_string(status), detail);
}

// A call on the tensor's device and that device's current stream.  Scratch comes
// from that stream's allocator: calls on other streams, and captured graphs,
// have their own.
struct Call {
  c10::cuda::CUDAGuard guard;
  void* stream;
  explicit Call(const Tensor& x) : guard(x.device()), stream(c10::cuda::getCurrentCUDAStream(x.device().index()).stream()) {}
  static Tensor scratch(size_t bytes, const Tensor& x) {
    return bytes ? at::empty({static_cast<int64_t>(bytes)}, x.options().dtype(at::kByte)) : Tensor();
  }
};

Tensor grad_like(const Tensor& t, bool wanted, bool zero) {
  if (!wanted || !t.defined()) return Tensor();
  return zero ? at::zeros(t.sizes(), t.options()) : at::empty(t.sizes(), t.options());
}

// Which of a node's inputs need a gradient; the node counts the defined tensors only.
std::vector<bool> needs(AutogradContext* ctx, const std::vector<Tensor>& inputs) {
  std::vector<bool> out;
  size_t edge = 0;
  for (const Tensor& t : inputs) {
    out.push_back(t.defined() && ctx->needs_input_grad(edge));
    edge += t.defined();
  }
  return out;
}

// Gradients of a backward pass that has none of its own: using them in another one is an error.
void once(variable_list& grads) {
  if (!at::GradMode::is_enabled()) return;
  variable_list marked;
  for (Tensor& g : grads)
    if (g.defined()) marked.push_back(g.detach().set_requires_grad(true));
  if (marked.empty()) return;
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "this operator's backward pass is not differentiable", static_cast<int>(marked.size()));
  variable_list outs = (*error)(std::move(marked));
  size_t i = 0;
  for (Tensor& g : grads)
    if (g.defined()) g = outs[i++];
}

// ---------------------------------------------------------------- causal convolution
void conv_check(const Tensor& x, const Tensor& w, const Tensor& bias, int64_t ndim) {
  activation(x, "x", ndim);
  const int64_t d = x.size(-1);
  TORCH_CHECK_VALUE(w.dim() == 2 && w.size(0) == d, "weight must have shape (", d, ", taps), got ", w.sizes());
  TORCH_CHECK_VALUE(d >= 1 && w.size(1) >= 1 && w.size(1) <= PT_CONV_MAX_TAPS, "the convolution needs channels and 1 to ",
                    PT_CONV_MAX_TAPS, " taps, got ", w.sizes());
  TORCH_CHECK_VALUE(w.scalar_type() == at::kFloat || w.scalar_type() == x.scalar_type(), "weight must be float32 or ",
                    x.scalar_type(), ", got ", w.scalar_type());
  TORCH_CHECK_VALUE(w.device() == x.device(), "weight must be on ", x.device(), ", got ", w.device());
  like(bias, "bias", {d}, w.scalar_type(), x);
}

pt_conv_args conv_args(const Tensor& x, const Tensor& w, const Tensor& bias, bool silu, int64_t batch, int64_t len) {
  pt_conv_args a{};
  a.dtype = type_code(x);
  a.param_f32 = w.scalar_type() == at::kFloat;
  a.batch = as_int(batch, "batch");
  a.len = as_int(len, "length");
  a.dim = as_int(w.size(0), "channels");
  a.taps = static_cast<int>(w.size(1));
  a.silu = silu;
  a.x = ptr(x), a.x_batch = x.stride(0), a.x_step = x.dim() == 3 ? x.stride(1) : 0;
  a.w = ptr(w), a.bias = ptr(bias);
  return a;
}

std::pair<Tensor, Tensor> conv_forward(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& state,
                                       const Tensor& lengths, bool silu, bool final) {
  Call call(x);
  Tensor y = at::empty(x.sizes(), x.options()), last;
  if (final) last = at::empty({x.size(0), w.size(1) - 1, x.size(2)}, x.options());
  pt_conv_args a = conv_args(x, w, bias, silu, x.size(0), x.size(1));
  a.state_in = ptr(state), a.lengths = as<int>(lengths);
  a.y = out_ptr(y), a.state_out = out_ptr(last);
  check(pt_causal_conv(&a, call.stream), "pt_causal_conv");
  return {y, last};
}

struct CausalConv : torch::autograd::Function<CausalConv> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& bias_,
                               const OptTensor& state_, const OptTensor& lengths_, bool silu, bool final) {
    const Tensor bias = given(bias_), state = given(state_), lengths = given(lengths_);
    ctx->set_materialize_grads(false);
    auto [y, last] = conv_forward(x, w, bias, state, lengths, silu, final);
    ctx->save_for_backward({x, w, bias, state, lengths});
    ctx->saved_data["silu"] = silu;
    return final ? variable_list{y, last} : variable_list{y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list given_grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &bias = saved[2], &state = saved[3], &lengths = saved[4];
    const auto need = needs(ctx, {x, w, bias, state, lengths});
    variable_list grads(7);
    {
      at::NoGradGuard no_grad;
      Call call(x);
      const Tensor dy = given_grads[0].defined() ? rows(given_grads[0]) : at::zeros(x.sizes(), x.options());
      const Tensor dlast = given_grads.size() > 1 ? dense(given_grads[1]) : Tensor();
      for (int i = 0; i < 4; ++i) grads[i] = grad_like(saved[i], need[i], x.size(0) == 0);
      pt_conv_args a = conv_args(x, w, bias, ctx->saved_data["silu"].toBool(), x.size(0), x.size(1));
      a.state_in = ptr(state), a.lengths = as<int>(lengths);
      a.dy = ptr(dy), a.dy_batch = dy.stride(0), a.dy_step = dy.stride(1);
      a.dstate_out = ptr(dlast);
      a.dx = out_ptr(grads[0]), a.dw = out_ptr(grads[1]), a.dbias = out_ptr(grads[2]), a.dstate_in = out_ptr(grads[3]);
      const size_t bytes = pt_causal_conv_bwd_workspace_bytes(&a);
      const Tensor ws = Call::scratch(bytes, x);
      check(pt_causal_conv_bwd(&a, out_ptr(ws), bytes, call.stream), "pt_causal_conv_bwd");
    }
    once(grads);
    return grads;
  }
};

variable_list causal_conv(const Tensor& x, const Tensor& w, const OptTensor& bias_, bool silu, const OptTensor& state_,
                          bool final, const OptTensor& lengths_) {
  const Tensor bias = given(bias_), state = given(state_), lengths = given(lengths_);
  conv_check(x, w, bias, 3);
  like(state, "initial_state", {x.size(0), w.size(1) - 1, x.size(2)}, x.scalar_type(), x);
  like(lengths, "lengths", {x.size(0)}, at::kInt, x);
  const Tensor xr = rows(x), wd = w.contiguous(), bd = dense(bias), sd = dense(state), ld = dense(lengths);
  if (wants_grad({x, w, bias, state})) return CausalConv::apply(xr, wd, maybe(bd), maybe(sd), maybe(ld), silu, final);
  auto [y, last] = conv_forward(xr, wd, bd, sd, ld, silu, final);
  return final ? variable_list{y, last} : variable_list{y};
}

Tensor causal_conv_step(const Tensor& state, const Tensor& x_, const Tensor& w_, const OptTensor& bias_, bool silu,
                        const OptTensor& slots_) {
  const Tensor bias = dense(given(bias_));
  refuse_grad("causal_conv_step", {state, x_, w_, bias});
  conv_check(x_, w_, bias, 2);
  const int64_t row = cache_row(state, w_.size(1) - 1, x_.size(1), x_.scalar_type(), x_);
  const Tensor slots = slots_of(given(slots_), x_.size(0), state.size(0), x_);
  const Tensor x = rows(x_), w = w_.contiguous();
  Call call(x);
  Tensor y = at::empty(x.sizes(), x.options());
  pt_conv_args a = conv_args(x, w, bias, silu, x.size(0), 1);
  a.cache_rows = as_int(state.size(0), "state");
  a.state_out = out_ptr(state), a.state_row = row, a.slots = as<int>(slots), a.y = out_ptr(y);
  check(pt_causal_conv_step(&a, call.stream), "pt_causal_conv_step");
  written(state);
  return y;
}

// ---------------------------------------------------------------- selective scan
struct ScanIn {
  Tensor x, dt, A, B, C, D, z, dt_bias, state, lengths;
};

// Checks the operands and gives B and C their dimension of groups.
void scan_check(ScanIn& v, int64_t ndim) {
  activation(v.x, "x", ndim);
  const Tensor& x = v.x;
  const int64_t d = x.size(-1);
  like(v.dt, "dt", x.sizes(), x.scalar_type(), x);
  like(v.z, "z", x.sizes(), x.scalar_type(), x);
  TORCH_CHECK_VALUE(v.A.dim() == 2 && v.A.size(0) == d, "A must have shape (", d, ", states), got ", v.A.sizes());
  const int64_t n = v.A.size(1);
  TORCH_CHECK_VALUE(d >= 1 && n >= 1 && n <= PT_SCAN_MAX_STATE, "the scan needs channels and 1 to ", PT_SCAN_MAX_STATE,
                    " states, got A ", v.A.sizes());
  like(v.A, "A", v.A.sizes(), at::kFloat, x);
  like(v.D, "D", {d}, at::kFloat, x);
  like(v.dt_bias, "dt_bias", {d}, at::kFloat, x);
  for (auto [t, name] : {std::pair<Tensor*, const char*>{&v.B, "B"}, {&v.C, "C"}}) {
    if (t->dim() == ndim) *t = t->unsqueeze(-2);
    TORCH_CHECK_VALUE(t->dim() == ndim + 1 && t->sizes().slice(0, ndim - 1) == x.sizes().slice(0, ndim - 1) && t->size(-1) == n,
                      name, " must have shape ", x.sizes().slice(0, ndim - 1), " + (", n, ",) or + (groups, ", n, "), got ",
                      t->sizes());
    TORCH_CHECK_VALUE(t->scalar_type() == x.scalar_type() && t->device() == x.device(), name, " must be ", x.scalar_type(),
                      " on ", x.device(), ", got ", t->scalar_type(), " on ", t->device());
  }
  const int64_t g = v.B.size(-2);
  TORCH_CHECK_VALUE(v.C.size(-2) == g && g >= 1 && d % g == 0, "B and C must have one number of groups that divides ", d,
                    " channels, got ", g, " and ", v.C.size(-2));
}

void scan_layout(ScanIn& v) {
  for (Tensor* t : {&v.x, &v.dt, &v.B, &v.C, &v.z}) *t = rows(*t);
  for (Tensor* t : {&v.A, &v.D, &v.dt_bias, &v.state, &v.lengths}) *t = dense(*t);
}

// `step` 1: [batch, length, ...] operands; 0: a single token's, without the length.
pt_scan_args scan_args(const ScanIn& v, bool softplus, int step) {
  pt_scan_args a{};
  const auto inner = [step](const Tensor& t) { return step && t.defined() ? t.stride(1) : int64_t{0}; };
  a.dtype = type_code(v.x);
  a.batch = as_int(v.x.size(0), "batch");
  a.len = step ? as_int(v.x.size(1), "length") : 1;
  a.dim = as_int(v.A.size(0), "channels");
  a.state = static_cast<int>(v.A.size(1));
  a.groups = as_int(v.B.size(-2), "groups");
  a.dt_softplus = softplus;
  a.x = ptr(v.x), a.dt = ptr(v.dt), a.z = ptr(v.z), a.B = ptr(v.B), a.C = ptr(v.C);
  a.x_batch = v.x.stride(0), a.x_step = inner(v.x);
  a.dt_batch = v.dt.stride(0), a.dt_step = inner(v.dt);
  a.z_batch = v.z.defined() ? v.z.stride(0) : 0, a.z_step = inner(v.z);
  a.B_batch = v.B.stride(0), a.B_step = inner(v.B), a.B_group = v.B.stride(-2);
  a.C_batch = v.C.stride(0), a.C_step = inner(v.C), a.C_group = v.C.stride(-2);
  a.A = as<float>(v.A), a.D = as<float>(v.D), a.dt_bias = as<float>(v.dt_bias), a.h0 = as<float>(v.state);
  a.lengths = as<int>(v.lengths);
  return a;
}

struct ScanOut {
  Tensor y, last, checkpoints;
};

ScanOut scan_forward(const ScanIn& v, bool softplus, bool final, bool train) {
  Call call(v.x);
  pt_scan_args a = scan_args(v, softplus, 1);
  const auto f32 = v.x.options().dtype(at::kFloat);
  ScanOut o;
  o.y = at::empty(v.x.sizes(), v.x.options());
  if (final) o.last = at::empty({v.x.size(0), v.A.size(0), v.A.size(1)}, f32);
  if (train) o.checkpoints = at::empty({static_cast<int64_t>(pt_scan_checkpoint_bytes(&a) / sizeof(float))}, f32);
  a.y = out_ptr(o.y), a.hlast = out_as<float>(o.last), a.checkpoints = out_as<float>(o.checkpoints);
  const size_t bytes = pt_scan_workspace_bytes(&a);
  const Tensor ws = Call::scratch(bytes, v.x);
  check(pt_scan(&a, out_ptr(ws), bytes, call.stream), "pt_scan");
  return o;
}

struct SelectiveScan : torch::autograd::Function<SelectiveScan> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B,
                               const Tensor& C, const OptTensor& D, const OptTensor& z, const OptTensor& dt_bias,
                               const OptTensor& state, const OptTensor& lengths, bool softplus, bool final) {
    ctx->set_materialize_grads(false);
    const ScanIn v{x, dt, A, B, C, given(D), given(z), given(dt_bias), given(state), given(lengths)};
    const ScanOut o = scan_forward(v, softplus, final, true);
    ctx->save_for_backward({x, dt, A, B, C, v.D, v.z, v.dt_bias, v.state, v.lengths, o.checkpoints});
    ctx->saved_data["softplus"] = softplus;
    return final ? variable_list{o.y, o.last} : variable_list{o.y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list given_grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor& x = s[0];
    const auto need = needs(ctx, {s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], s[8], s[9]});
    variable_list grads(12);
    {
      at::NoGradGuard no_grad;
      Call call(x);
      const Tensor dy = given_grads[0].defined() ? rows(given_grads[0]) : at::zeros(x.sizes(), x.options());
      const Tensor dlast = given_grads.size() > 1 ? dense(given_grads[1]) : Tensor();
      for (int i = 0; i < 9; ++i) grads[i] = grad_like(s[i], need[i], x.size(0) == 0);
      pt_scan_args a = scan_args({s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], s[8], s[9]},
                                 ctx->saved_data["softplus"].toBool(), 1);
      a.checkpoints = const_cast<float*>(as<float>(s[10]));
      a.dy = ptr(dy), a.dy_batch = dy.stride(0), a.dy_step = dy.stride(1), a.dhlast = as<float>(dlast);
      a.dx = out_ptr(grads[0]), a.ddt = out_ptr(grads[1]), a.dA = out_as<float>(grads[2]), a.dB = out_ptr(grads[3]);
      a.dC = out_ptr(grads[4]), a.dD = out_as<float>(grads[5]), a.dz = out_ptr(grads[6]);
      a.ddt_bias = out_as<float>(grads[7]), a.dh0 = out_as<float>(grads[8]);
      const size_t bytes = pt_scan_bwd_workspace_bytes(&a);
      const Tensor ws = Call::scratch(bytes, x);
      check(pt_scan_bwd(&a, out_ptr(ws), bytes, call.stream), "pt_scan_bwd");
    }
    once(grads);
    return grads;
  }
};

variable_list selective_scan(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C,
                             const OptTensor& D, const OptTensor& z, const OptTensor& dt_bias, bool softplus,
                             const OptTensor& state, bool final, const OptTensor& lengths) {
  ScanIn v{x, dt, A, B, C, given(D), given(z), given(dt_bias), given(state), given(lengths)};
  scan_check(v, 3);
  like(v.state, "initial_state", {x.size(0), x.size(2), A.size(1)}, at::kFloat, x);
  like(v.lengths, "lengths", {x.size(0)}, at::kInt, x);
  const bool grad = wants_grad({v.x, v.dt, v.A, v.B, v.C, v.D, v.z, v.dt_bias, v.state});
  scan_layout(v);
  if (grad)
    return SelectiveScan::apply(v.x, v.dt, v.A, v.B, v.C, maybe(v.D), maybe(v.z), maybe(v.dt_bias), maybe(v.state),
                                maybe(v.lengths), softplus, final);
  const ScanOut o = scan_forward(v, softplus, final, false);
  return final ? variable_list{o.y, o.last} : variable_list{o.y};
}

Tensor selective_scan_step(const Tensor& state, const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B,
                           const Tensor& C, const OptTensor& D, const OptTensor& z, const OptTensor& dt_bias,
                           bool softplus, const OptTensor& slots_) {
  ScanIn v{x, dt, A, B, C, given(D), given(z), given(dt_bias), Tensor(), Tensor()};
  refuse_grad("selective_scan_step", {state, v.x, v.dt, v.A, v.B, v.C, v.D, v.z, v.dt_bias});
  scan_check(v, 2);
  const int64_t row = cache_row(state, A.size(0), A.size(1), at::kFloat, x);
  const Tensor slots = slots_of(given(slots_), x.size(0), state.size(0), x);
  scan_layout(v);
  Call call(x);
  Tensor y = at::empty(x.sizes(), x.options());
  pt_scan_args a = scan_args(v, softplus, 0);
  a.cache_rows = as_int(state.size(0), "state");
  a.hlast = out_as<float>(state), a.h_row = row, a.slots = as<int>(slots), a.y = out_ptr(y);
  check(pt_scan_step(&a, call.stream), "pt_scan_step");
  written(state);
  return y;
}

// ---------------------------------------------------------------- norm
// t as [rows, channels], channels contiguous.
Tensor flat(const Tensor& t) { return t.defined() ? rows(t.dim() == 2 ? t : t.reshape({-1, t.size(-1)})) : t; }

pt_norm_args norm_args(const Tensor& x, const Tensor& w, const Tensor& gate, const Tensor& residual, const Tensor& scale,
                       int64_t groups, double eps) {
  pt_norm_args a{};
  a.dtype = type_code(x);
  a.param_f32 = w.scalar_type() == at::kFloat;
  a.residual_f32 = residual.defined() && residual.scalar_type() == at::kFloat;
  a.groups = as_int(groups, "groups");
  a.rows = x.size(0);
  a.dim = as_int(x.size(1), "channels");
  a.eps = static_cast<float>(eps);
  a.x = ptr(x), a.gate = ptr(gate), a.residual = ptr(residual);
  a.x_row = x.stride(0), a.gate_row = gate.defined() ? gate.stride(0) : 0;
  a.residual_row = residual.defined() ? residual.stride(0) : 0;
  a.weight = ptr(w), a.scale = ptr(scale);
  return a;
}

std::pair<Tensor, Tensor> norm_forward(const Tensor& x, const Tensor& w, const Tensor& gate, const Tensor& residual,
                                       const Tensor& scale, int64_t groups, double eps) {
  Call call(x);
  Tensor y = at::empty(x.sizes(), x.options()), r;
  if (residual.defined()) r = at::empty(x.sizes(), residual.options());
  pt_norm_args a = norm_args(x, w, gate, residual, scale, groups, eps);
  a.y = out_ptr(y), a.r = out_ptr(r);
  check(pt_fused_norm(&a, call.stream), "pt_fused_norm");
  return {y, r};
}

struct FusedNorm : torch::autograd::Function<FusedNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& gate_,
                               const OptTensor& residual_, const OptTensor& scale_, int64_t groups, double eps) {
    const Tensor gate = given(gate_), residual = given(residual_), scale = given(scale_);
    ctx->set_materialize_grads(false);
    auto [y, r] = norm_forward(x, w, gate, residual, scale, groups, eps);
    ctx->save_for_backward({x, w, gate, scale, r});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["eps"] = eps;
    return r.defined() ? variable_list{y, r} : variable_list{y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list given_grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor &x = s[0], &w = s[1], &gate = s[2], &scale = s[3], &r = s[4];
    // In the order of the inputs; r is shaped and typed like the residual that it sums up.
    const std::vector<Tensor> inputs{x, w, gate, r, scale};
    const auto need = needs(ctx, inputs);
    variable_list grads(7);
    {
      at::NoGradGuard no_grad;
      Call call(x);
      const Tensor dy = given_grads[0].defined() ? rows(given_grads[0]) : at::zeros(x.sizes(), x.options());
      const Tensor dr = given_grads.size() > 1 ? rows(given_grads[1]) : Tensor();
      for (int i = 0; i < 5; ++i) grads[i] = grad_like(inputs[i], need[i], x.size(0) == 0);
      // The kernel needs to know of a residual, and reads its sum r instead.
      pt_norm_args a = norm_args(x, w, gate, r, scale, ctx->saved_data["groups"].toInt(), ctx->saved_data["eps"].toDouble());
      a.r = const_cast<void*>(ptr(r)), a.dy = ptr(dy), a.dy_row = dy.stride(0);
      if (dr.defined()) a.dr = ptr(dr), a.dr_row = dr.stride(0);
      a.dx = out_ptr(grads[0]), a.dweight = out_ptr(grads[1]), a.dgate = out_ptr(grads[2]);
      a.dresidual = out_ptr(grads[3]), a.dscale = out_ptr(grads[4]);
      const size_t bytes = pt_fused_norm_bwd_workspace_bytes(&a);
      const Tensor ws = Call::scratch(bytes, x);
      check(pt_fused_norm_bwd(&a, out_ptr(ws), bytes, call.stream), "pt_fused_norm_bwd");
    }
    once(grads);
    return grads;
  }
};

variable_list fused_norm(const Tensor& x, const Tensor& w, const OptTensor& gate_, const OptTensor& residual_,
                         const OptTensor& scale_, int64_t groups, double eps) {
  const Tensor gate = given(gate_), residual = given(residual_), scale = given(scale_);
  TORCH_CHECK_VALUE(x.dim() >= 1, "x must have at least one dimension");
  activation(x, "x", x.dim());
  const int64_t d = x.size(-1);
  like(gate, "gate", x.sizes(), x.scalar_type(), x);
  like(residual, "residual", x.sizes(),
       residual.defined() && residual.scalar_type() == at::kFloat ? at::kFloat : x.scalar_type(), x);
  like(w, "weight", {d}, w.scalar_type() == at::kFloat ? at::kFloat : x.scalar_type(), x);
  like(scale, "scale", {d}, w.scalar_type(), x);
  TORCH_CHECK_VALUE(d >= 1 && groups >= 1 && d % groups == 0, "groups must divide the ", d, " channels, got ", groups);
  TORCH_CHECK_VALUE(d / groups <= PT_NORM_MAX_WIDTH, "a group may have up to ", PT_NORM_MAX_WIDTH, " channels, got ", d / groups);
  const Tensor xf = flat(x), wd = w.contiguous(), gf = flat(gate), rf = flat(residual), sd = dense(scale);
  variable_list out;
  if (wants_grad({x, w, gate, residual, scale})) {
    out = FusedNorm::apply(xf, wd, maybe(gf), maybe(rf), maybe(sd), groups, eps);
  } else {
    auto [y, r] = norm_forward(xf, wd, gf, rf, sd, groups, eps);
    out = r.defined() ? variable_list{y, r} : variable_list{y};
  }
  if (x.dim() != 2)
    for (Tensor& t : out) t = t.view(x.sizes());
  return out;
}

}  // namespace

PYBIND11_MODULE(_sequence, m) {
  m.doc() = "Native calls of pathtile_b200.sequence";
  m.def("causal_conv", &causal_conv);
  m.def("causal_conv_step", &causal_conv_step);
  m.def("selective_scan", &selective_scan);
  m.def("selective_scan_step", &selective_scan_step);
  m.def("fused_norm", &fused_norm);
}
