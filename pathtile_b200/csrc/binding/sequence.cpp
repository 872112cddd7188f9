// sequence.cpp -- the sequence operators' checks, autograd nodes and calls on
// torch tensors: what pathtile_b200/sequence.py documents.  A call of a single
// token takes the GPU two to three microseconds, so everything around it is
// done here and not in Python.  The kernels are behind the C ABI of
// libpathtile_b200.so.
//
// Each call is an operator of torch's dispatcher (pathtile_b200::causal_conv, ...,
// the backward passes too), so that tracers and dispatch modes record the call,
// and not the empty tensor that it fills.  An operator has two functions:
// *_kernel checks, lays out, allocates and launches (on meta tensors, which stand
// for others while shapes are traced, it launches nothing), and *_autograd in
// front of it records the node where a gradient is asked for.
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>
#include <torch/library.h>

#include <array>
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
  TORCH_CHECK_VALUE(t.is_cuda() || t.is_meta(), name, " must be a CUDA tensor");
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
// Forward mode: no operator carries tangents on, with or without gradients asked for.
void refuse_tangents(const char* what, std::initializer_list<Tensor> tensors) {
  for (const Tensor& t : tensors)
    TORCH_CHECK_VALUE(!t.defined() || !t._fw_grad(0).defined(), what, " has no derivative in forward mode");
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

// What runs behind an operator's autograd function.
using BelowAutograd = at::AutoDispatchBelowADInplaceOrView;
// The operator `name` of this library, as a call; F: its kernel's type.
template <class F>
c10::TypedOperatorHandle<F> op(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").template typed<F>();
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

// Gradients of the first N inputs, those that are wanted (of an empty batch: zeros).
template <size_t N>
struct Grads {
  std::array<Tensor, N> of;
  Grads(const std::array<Tensor, N>& inputs, const std::array<bool, N>& wanted, bool zero) {
    for (size_t i = 0; i < N; ++i)
      if (wanted[i] && inputs[i].defined())
        of[i] = zero ? at::zeros(inputs[i].sizes(), inputs[i].options()) : at::empty(inputs[i].sizes(), inputs[i].options());
  }
  // One behind the other, as a backward operator returns them.
  variable_list list() const {
    variable_list out;
    for (const Tensor& t : of)
      if (t.defined()) out.push_back(t);
    return out;
  }
};
// A node's gradients (`all` inputs, tensors or not) from that list.
template <size_t N>
variable_list spread(const variable_list& list, const std::array<bool, N>& wanted, size_t all) {
  variable_list out(all);
  size_t k = 0;
  for (size_t i = 0; i < N; ++i)
    if (wanted[i]) out[i] = list[k++];
  return out;
}

// Which of a node's inputs need a gradient; the node counts the defined tensors only.
template <size_t N>
std::array<bool, N> needs(AutogradContext* ctx, const std::array<Tensor, N>& inputs) {
  std::array<bool, N> out{};
  size_t edge = 0;
  for (size_t i = 0; i < N; ++i) {
    out[i] = inputs[i].defined() && ctx->needs_input_grad(edge);
    edge += inputs[i].defined();
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

// A backward operator as nodes call it, and its autograd function: it has no derivative itself.
template <class OP, class F = typename OP::Kernel>
struct Backward;
template <class OP, class... A>
struct Backward<OP, variable_list(A...)> {
  static variable_list call(A... args) {
    static const auto handle = op<typename OP::Kernel>(OP::kName);
    return handle.call(args...);
  }
  static variable_list autograd(A... args) {
    refuse_tangents(OP::kName, {tensor_of(args)...});
    variable_list out;
    {
      BelowAutograd below;
      out = call(args...);
    }
    if (wants_grad({tensor_of(args)...})) once(out);
    return out;
  }
  static Tensor tensor_of(const Tensor& t) { return t; }
  static Tensor tensor_of(const OptTensor& t) { return given(t); }
  template <class T>
  static Tensor tensor_of(const T&) { return Tensor(); }
};

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

// Of prompts; the step has no lengths and a state of its own.
void conv_check(const Tensor& x, const Tensor& w, const Tensor& bias, const Tensor& state, const Tensor& lengths) {
  conv_check(x, w, bias, 3);
  like(state, "initial_state", {x.size(0), w.size(1) - 1, x.size(2)}, x.scalar_type(), x);
  like(lengths, "lengths", {x.size(0)}, at::kInt, x);
}

variable_list conv_kernel(const Tensor& x_, const Tensor& w_, const OptTensor& bias_, bool silu, const OptTensor& state_,
                          bool final, const OptTensor& lengths_) {
  conv_check(x_, w_, given(bias_), given(state_), given(lengths_));
  const Tensor x = rows(x_), w = w_.contiguous(), bias = dense(given(bias_)), state = dense(given(state_));
  const Tensor lengths = dense(given(lengths_));
  variable_list out{at::empty(x.sizes(), x.options())};
  if (final) out.push_back(at::empty({x.size(0), w.size(1) - 1, x.size(2)}, x.options()));
  if (x.is_meta()) return out;
  Call call(x);
  pt_conv_args a = conv_args(x, w, bias, silu, x.size(0), x.size(1));
  a.state_in = ptr(state), a.lengths = as<int>(lengths);
  a.y = out_ptr(out[0]), a.state_out = final ? out_ptr(out[1]) : nullptr;
  check(pt_causal_conv(&a, call.stream), "pt_causal_conv");
  return out;
}

variable_list conv_backward_kernel(const OptTensor& dy_, const OptTensor& dlast_, const Tensor& x_, const Tensor& w_,
                                   const OptTensor& bias_, const OptTensor& state_, const OptTensor& lengths_, bool silu,
                                   std::array<bool, 4> wanted) {
  conv_check(x_, w_, given(bias_), given(state_), given(lengths_));
  like(given(dy_), "the gradient of y", x_.sizes(), x_.scalar_type(), x_);
  like(given(dlast_), "the gradient of the final state", {x_.size(0), w_.size(1) - 1, x_.size(2)}, x_.scalar_type(), x_);
  const Tensor x = rows(x_), w = w_.contiguous(), bias = dense(given(bias_)), state = dense(given(state_));
  const Tensor lengths = dense(given(lengths_)), dlast = dense(given(dlast_));
  const Grads<4> grads({x, w, bias, state}, wanted, x.size(0) == 0);
  if (x.is_meta()) return grads.list();
  Call call(x);
  const Tensor dy = dy_.has_value() ? rows(*dy_) : at::zeros(x.sizes(), x.options());
  pt_conv_args a = conv_args(x, w, bias, silu, x.size(0), x.size(1));
  a.state_in = ptr(state), a.lengths = as<int>(lengths);
  a.dy = ptr(dy), a.dy_batch = dy.stride(0), a.dy_step = dy.stride(1);
  a.dstate_out = ptr(dlast);
  a.dx = out_ptr(grads.of[0]), a.dw = out_ptr(grads.of[1]), a.dbias = out_ptr(grads.of[2]);
  a.dstate_in = out_ptr(grads.of[3]);
  const size_t bytes = pt_causal_conv_bwd_workspace_bytes(&a);
  const Tensor ws = Call::scratch(bytes, x);
  check(pt_causal_conv_bwd(&a, out_ptr(ws), bytes, call.stream), "pt_causal_conv_bwd");
  return grads.list();
}

variable_list causal_conv(const Tensor& x, const Tensor& w, const OptTensor& bias, bool silu, const OptTensor& state,
                          bool final, const OptTensor& lengths) {
  static const auto call = op<decltype(conv_kernel)>("pathtile_b200::causal_conv");
  return call.call(x, w, bias, silu, state, final, lengths);
}

struct ConvBackward {
  static constexpr const char* kName = "pathtile_b200::causal_conv_backward";
  using Kernel = decltype(conv_backward_kernel);
};

struct CausalConv : torch::autograd::Function<CausalConv> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& bias,
                               const OptTensor& state, const OptTensor& lengths, bool silu, bool final) {
    BelowAutograd below;
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, w, given(bias), given(state), given(lengths)});
    ctx->saved_data["silu"] = silu;
    return causal_conv(x, w, bias, silu, state, final, lengths);
  }
  static variable_list backward(AutogradContext* ctx, variable_list given_grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor dlast = given_grads.size() > 1 ? given_grads[1] : Tensor();
    const auto wanted = needs<4>(ctx, {s[0], s[1], s[2], s[3]});
    const bool silu = ctx->saved_data["silu"].toBool();
    return spread(Backward<ConvBackward>::call(maybe(given_grads[0]), maybe(dlast), s[0], s[1], maybe(s[2]), maybe(s[3]),
                                               maybe(s[4]), silu, wanted),
                  wanted, 7);
  }
};

variable_list conv_autograd(const Tensor& x, const Tensor& w, const OptTensor& bias_, bool silu, const OptTensor& state_,
                            bool final, const OptTensor& lengths_) {
  const Tensor bias = given(bias_), state = given(state_), lengths = given(lengths_);
  refuse_tangents("causal_conv", {x, w, bias, state});
  if (!wants_grad({x, w, bias, state})) {
    BelowAutograd below;
    return causal_conv(x, w, bias_, silu, state_, final, lengths_);
  }
  conv_check(x, w, bias, state, lengths);
  return CausalConv::apply(rows(x), w.contiguous(), maybe(dense(bias)), maybe(dense(state)), maybe(dense(lengths)), silu, final);
}

Tensor conv_step_kernel(const Tensor& state, const Tensor& x_, const Tensor& w_, const OptTensor& bias_, bool silu,
                        const OptTensor& slots_) {
  const Tensor bias = dense(given(bias_));
  conv_check(x_, w_, bias, 2);
  const int64_t row = cache_row(state, w_.size(1) - 1, x_.size(1), x_.scalar_type(), x_);
  const Tensor slots = slots_of(given(slots_), x_.size(0), state.size(0), x_);
  const Tensor x = rows(x_), w = w_.contiguous();
  Tensor y = at::empty(x.sizes(), x.options());
  written(state);
  if (x.is_meta()) return y;
  Call call(x);
  pt_conv_args a = conv_args(x, w, bias, silu, x.size(0), 1);
  a.cache_rows = as_int(state.size(0), "state");
  a.state_out = out_ptr(state), a.state_row = row, a.slots = as<int>(slots), a.y = out_ptr(y);
  check(pt_causal_conv_step(&a, call.stream), "pt_causal_conv_step");
  return y;
}

Tensor causal_conv_step(const Tensor& state, const Tensor& x, const Tensor& w, const OptTensor& bias, bool silu,
                        const OptTensor& slots) {
  static const auto call = op<decltype(conv_step_kernel)>("pathtile_b200::causal_conv_step");
  return call.call(state, x, w, bias, silu, slots);
}

Tensor conv_step_autograd(const Tensor& state, const Tensor& x, const Tensor& w, const OptTensor& bias, bool silu,
                          const OptTensor& slots) {
  refuse_tangents("causal_conv_step", {state, x, w, given(bias)});
  refuse_grad("causal_conv_step", {state, x, w, given(bias)});
  BelowAutograd below;
  return causal_conv_step(state, x, w, bias, silu, slots);
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

// Of prompts; the step has no lengths and a state of its own.
void scan_check(ScanIn& v) {
  scan_check(v, 3);
  like(v.state, "initial_state", {v.x.size(0), v.x.size(2), v.A.size(1)}, at::kFloat, v.x);
  like(v.lengths, "lengths", {v.x.size(0)}, at::kInt, v.x);
}

void scan_layout(ScanIn& v) {
  for (Tensor* t : {&v.x, &v.dt, &v.B, &v.C, &v.z}) *t = rows(*t);
  for (Tensor* t : {&v.A, &v.D, &v.dt_bias, &v.state, &v.lengths}) *t = dense(*t);
}

// `step` 1: [batch, length, ...] operands; 0: a single token's, without the length.
pt_scan_args scan_sizes(const ScanIn& v, bool softplus, int step) {
  pt_scan_args a{};
  a.dtype = type_code(v.x);
  a.batch = as_int(v.x.size(0), "batch");
  a.len = step ? as_int(v.x.size(1), "length") : 1;
  a.dim = as_int(v.A.size(0), "channels");
  a.state = static_cast<int>(v.A.size(1));
  a.groups = as_int(v.B.size(-2), "groups");
  a.dt_softplus = softplus;
  return a;
}

pt_scan_args scan_args(const ScanIn& v, bool softplus, int step) {
  pt_scan_args a = scan_sizes(v, softplus, step);
  const auto inner = [step](const Tensor& t) { return step && t.defined() ? t.stride(1) : int64_t{0}; };
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

int64_t checkpoint_floats(const ScanIn& v) {
  const pt_scan_args a = scan_sizes(v, false, 1);
  return static_cast<int64_t>(pt_scan_checkpoint_bytes(&a) / sizeof(float));
}

// `keep`: with the checkpoints that a backward pass starts from as the last output.
variable_list scan_kernel(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C,
                          const OptTensor& D, const OptTensor& z, const OptTensor& dt_bias, bool softplus,
                          const OptTensor& state, bool final, const OptTensor& lengths, bool keep) {
  ScanIn v{x, dt, A, B, C, given(D), given(z), given(dt_bias), given(state), given(lengths)};
  scan_check(v);
  scan_layout(v);
  const auto f32 = v.x.options().dtype(at::kFloat);
  variable_list out{at::empty(v.x.sizes(), v.x.options())};
  if (final) out.push_back(at::empty({v.x.size(0), v.A.size(0), v.A.size(1)}, f32));
  if (keep) out.push_back(at::empty({checkpoint_floats(v)}, f32));
  if (x.is_meta()) return out;
  Call call(v.x);
  pt_scan_args a = scan_args(v, softplus, 1);
  a.y = out_ptr(out[0]), a.hlast = final ? out_as<float>(out[1]) : nullptr;
  a.checkpoints = keep ? out_as<float>(out.back()) : nullptr;
  const size_t bytes = pt_scan_workspace_bytes(&a);
  const Tensor ws = Call::scratch(bytes, v.x);
  check(pt_scan(&a, out_ptr(ws), bytes, call.stream), "pt_scan");
  return out;
}

variable_list scan_backward_kernel(const OptTensor& dy_, const OptTensor& dlast_, const Tensor& x, const Tensor& dt,
                                   const Tensor& A, const Tensor& B, const Tensor& C, const OptTensor& D,
                                   const OptTensor& z, const OptTensor& dt_bias, const OptTensor& state,
                                   const OptTensor& lengths, const Tensor& checkpoints_, bool softplus,
                                   std::array<bool, 9> wanted) {
  ScanIn v{x, dt, A, B, C, given(D), given(z), given(dt_bias), given(state), given(lengths)};
  scan_check(v);
  scan_layout(v);
  like(given(dy_), "the gradient of y", x.sizes(), x.scalar_type(), x);
  like(given(dlast_), "the gradient of the final state", {x.size(0), A.size(0), A.size(1)}, at::kFloat, x);
  like(checkpoints_, "checkpoints", {checkpoint_floats(v)}, at::kFloat, x);
  const Tensor dlast = dense(given(dlast_)), checkpoints = dense(checkpoints_);
  Grads<9> grads({v.x, v.dt, v.A, v.B, v.C, v.D, v.z, v.dt_bias, v.state}, wanted, x.size(0) == 0);
  if (!x.is_meta()) {
    Call call(v.x);
    const Tensor dy = dy_.has_value() ? rows(*dy_) : at::zeros(x.sizes(), x.options());
    pt_scan_args a = scan_args(v, softplus, 1);
    a.checkpoints = const_cast<float*>(as<float>(checkpoints));
    a.dy = ptr(dy), a.dy_batch = dy.stride(0), a.dy_step = dy.stride(1), a.dhlast = as<float>(dlast);
    const auto& g = grads.of;
    a.dx = out_ptr(g[0]), a.ddt = out_ptr(g[1]), a.dA = out_as<float>(g[2]), a.dB = out_ptr(g[3]), a.dC = out_ptr(g[4]);
    a.dD = out_as<float>(g[5]), a.dz = out_ptr(g[6]), a.ddt_bias = out_as<float>(g[7]), a.dh0 = out_as<float>(g[8]);
    const size_t bytes = pt_scan_bwd_workspace_bytes(&a);
    const Tensor ws = Call::scratch(bytes, v.x);
    check(pt_scan_bwd(&a, out_ptr(ws), bytes, call.stream), "pt_scan_bwd");
  }
  if (grads.of[3].defined() && B.dim() == 3) grads.of[3] = grads.of[3].view(B.sizes());
  if (grads.of[4].defined() && C.dim() == 3) grads.of[4] = grads.of[4].view(C.sizes());
  return grads.list();
}

variable_list scan_op(const ScanIn& v, bool softplus, bool final, bool keep) {
  static const auto call = op<decltype(scan_kernel)>("pathtile_b200::selective_scan");
  return call.call(v.x, v.dt, v.A, v.B, v.C, maybe(v.D), maybe(v.z), maybe(v.dt_bias), softplus, maybe(v.state), final,
                   maybe(v.lengths), keep);
}

struct ScanBackward {
  static constexpr const char* kName = "pathtile_b200::selective_scan_backward";
  using Kernel = decltype(scan_backward_kernel);
};

struct SelectiveScan : torch::autograd::Function<SelectiveScan> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B,
                               const Tensor& C, const OptTensor& D, const OptTensor& z, const OptTensor& dt_bias,
                               const OptTensor& state, const OptTensor& lengths, bool softplus, bool final) {
    BelowAutograd below;
    ctx->set_materialize_grads(false);
    const ScanIn v{x, dt, A, B, C, given(D), given(z), given(dt_bias), given(state), given(lengths)};
    variable_list out = scan_op(v, softplus, final, true);
    ctx->save_for_backward({x, dt, A, B, C, v.D, v.z, v.dt_bias, v.state, v.lengths, out.back()});
    ctx->saved_data["softplus"] = softplus;
    out.pop_back();
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list given_grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor dlast = given_grads.size() > 1 ? given_grads[1] : Tensor();
    const auto wanted = needs<9>(ctx, {s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], s[8]});
    const bool softplus = ctx->saved_data["softplus"].toBool();
    return spread(Backward<ScanBackward>::call(maybe(given_grads[0]), maybe(dlast), s[0], s[1], s[2], s[3], s[4], maybe(s[5]),
                                               maybe(s[6]), maybe(s[7]), maybe(s[8]), maybe(s[9]), s[10], softplus, wanted),
                  wanted, 12);
  }
};

variable_list scan_autograd(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C,
                            const OptTensor& D, const OptTensor& z, const OptTensor& dt_bias, bool softplus,
                            const OptTensor& state, bool final, const OptTensor& lengths, bool keep) {
  ScanIn v{x, dt, A, B, C, given(D), given(z), given(dt_bias), given(state), given(lengths)};
  refuse_tangents("selective_scan", {v.x, v.dt, v.A, v.B, v.C, v.D, v.z, v.dt_bias, v.state});
  if (!wants_grad({v.x, v.dt, v.A, v.B, v.C, v.D, v.z, v.dt_bias, v.state})) {
    BelowAutograd below;
    return scan_op(v, softplus, final, keep);
  }
  TORCH_CHECK_VALUE(!keep, "selective_scan: keep_checkpoints is for calls that record no gradient");
  scan_check(v);
  scan_layout(v);
  return SelectiveScan::apply(v.x, v.dt, v.A, v.B, v.C, maybe(v.D), maybe(v.z), maybe(v.dt_bias), maybe(v.state),
                              maybe(v.lengths), softplus, final);
}

variable_list selective_scan(const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C,
                             const OptTensor& D, const OptTensor& z, const OptTensor& dt_bias, bool softplus,
                             const OptTensor& state, bool final, const OptTensor& lengths) {
  return scan_op({x, dt, A, B, C, given(D), given(z), given(dt_bias), given(state), given(lengths)}, softplus, final, false);
}

Tensor scan_step_kernel(const Tensor& state, const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B,
                        const Tensor& C, const OptTensor& D, const OptTensor& z, const OptTensor& dt_bias, bool softplus,
                        const OptTensor& slots_) {
  ScanIn v{x, dt, A, B, C, given(D), given(z), given(dt_bias), Tensor(), Tensor()};
  scan_check(v, 2);
  const int64_t row = cache_row(state, A.size(0), A.size(1), at::kFloat, x);
  const Tensor slots = slots_of(given(slots_), x.size(0), state.size(0), x);
  scan_layout(v);
  Tensor y = at::empty(x.sizes(), x.options());
  written(state);
  if (x.is_meta()) return y;
  Call call(x);
  pt_scan_args a = scan_args(v, softplus, 0);
  a.cache_rows = as_int(state.size(0), "state");
  a.hlast = out_as<float>(state), a.h_row = row, a.slots = as<int>(slots), a.y = out_ptr(y);
  check(pt_scan_step(&a, call.stream), "pt_scan_step");
  return y;
}

Tensor selective_scan_step(const Tensor& state, const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B,
                           const Tensor& C, const OptTensor& D, const OptTensor& z, const OptTensor& dt_bias,
                           bool softplus, const OptTensor& slots) {
  static const auto call = op<decltype(scan_step_kernel)>("pathtile_b200::selective_scan_step");
  return call.call(state, x, dt, A, B, C, D, z, dt_bias, softplus, slots);
}

Tensor scan_step_autograd(const Tensor& state, const Tensor& x, const Tensor& dt, const Tensor& A, const Tensor& B,
                          const Tensor& C, const OptTensor& D, const OptTensor& z, const OptTensor& dt_bias, bool softplus,
                          const OptTensor& slots) {
  refuse_tangents("selective_scan_step", {state, x, dt, A, B, C, given(D), given(z), given(dt_bias)});
  refuse_grad("selective_scan_step", {state, x, dt, A, B, C, given(D), given(z), given(dt_bias)});
  BelowAutograd below;
  return selective_scan_step(state, x, dt, A, B, C, D, z, dt_bias, softplus, slots);
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

void norm_check(const Tensor& x, const Tensor& w, const Tensor& gate, const Tensor& residual, const Tensor& scale,
                int64_t groups) {
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
}

// y, and r with a residual.
variable_list norm_kernel(const Tensor& x_, const Tensor& w_, const OptTensor& gate_, const OptTensor& residual_,
                          const OptTensor& scale_, int64_t groups, double eps) {
  norm_check(x_, w_, given(gate_), given(residual_), given(scale_), groups);
  const Tensor x = flat(x_), w = w_.contiguous(), gate = flat(given(gate_)), residual = flat(given(residual_));
  const Tensor scale = dense(given(scale_));
  variable_list out{at::empty(x_.sizes(), x.options())};
  if (residual.defined()) out.push_back(at::empty(x_.sizes(), residual.options()));
  if (x.is_meta()) return out;
  Call call(x);
  pt_norm_args a = norm_args(x, w, gate, residual, scale, groups, eps);
  a.y = out_ptr(out[0]), a.r = residual.defined() ? out_ptr(out[1]) : nullptr;
  check(pt_fused_norm(&a, call.stream), "pt_fused_norm");
  return out;
}

// r: the forward pass' own, in the residual's place, whose shape and type it has.
variable_list norm_backward_kernel(const OptTensor& dy_, const OptTensor& dr_, const Tensor& x_, const Tensor& w_,
                                   const OptTensor& gate_, const OptTensor& scale_, const OptTensor& r_, int64_t groups,
                                   double eps, std::array<bool, 5> wanted) {
  norm_check(x_, w_, given(gate_), given(r_), given(scale_), groups);
  like(given(dy_), "the gradient of y", x_.sizes(), x_.scalar_type(), x_);
  TORCH_CHECK_VALUE(!dr_.has_value() || r_.has_value(), "no residual, so there is no gradient of r");
  if (r_.has_value()) like(given(dr_), "the gradient of r", x_.sizes(), r_->scalar_type(), x_);
  const Tensor x = flat(x_), w = w_.contiguous(), gate = flat(given(gate_)), scale = dense(given(scale_));
  const Tensor r = dense(flat(given(r_))), dr = flat(given(dr_));
  // In the order of the forward pass' inputs.
  Grads<5> grads({x, w, gate, r, scale}, wanted, x.size(0) == 0);
  if (!x.is_meta()) {
    Call call(x);
    const Tensor dy = dy_.has_value() ? flat(*dy_) : at::zeros(x.sizes(), x.options());
    // The kernel needs to know of a residual, and reads its sum r instead.
    pt_norm_args a = norm_args(x, w, gate, r, scale, groups, eps);
    a.r = const_cast<void*>(ptr(r)), a.dy = ptr(dy), a.dy_row = dy.stride(0);
    if (dr.defined()) a.dr = ptr(dr), a.dr_row = dr.stride(0);
    a.dx = out_ptr(grads.of[0]), a.dweight = out_ptr(grads.of[1]), a.dgate = out_ptr(grads.of[2]);
    a.dresidual = out_ptr(grads.of[3]), a.dscale = out_ptr(grads.of[4]);
    const size_t bytes = pt_fused_norm_bwd_workspace_bytes(&a);
    const Tensor ws = Call::scratch(bytes, x);
    check(pt_fused_norm_bwd(&a, out_ptr(ws), bytes, call.stream), "pt_fused_norm_bwd");
  }
  if (x_.dim() != 2)
    for (const int i : {0, 2, 3})
      if (grads.of[i].defined()) grads.of[i] = grads.of[i].view(x_.sizes());
  return grads.list();
}

variable_list fused_norm(const Tensor& x, const Tensor& w, const OptTensor& gate, const OptTensor& residual,
                         const OptTensor& scale, int64_t groups, double eps) {
  static const auto call = op<decltype(norm_kernel)>("pathtile_b200::fused_norm");
  return call.call(x, w, gate, residual, scale, groups, eps);
}

struct NormBackward {
  static constexpr const char* kName = "pathtile_b200::fused_norm_backward";
  using Kernel = decltype(norm_backward_kernel);
};

struct FusedNorm : torch::autograd::Function<FusedNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& gate,
                               const OptTensor& residual, const OptTensor& scale, int64_t groups, double eps) {
    BelowAutograd below;
    ctx->set_materialize_grads(false);
    variable_list out = fused_norm(x, w, gate, residual, scale, groups, eps);
    ctx->save_for_backward({x, w, given(gate), given(scale), residual.has_value() ? out[1] : Tensor()});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["eps"] = eps;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list given_grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor &x = s[0], &w = s[1], &gate = s[2], &scale = s[3], &r = s[4];
    const Tensor dr = given_grads.size() > 1 ? given_grads[1] : Tensor();
    const auto wanted = needs<5>(ctx, {x, w, gate, r, scale});
    const int64_t groups = ctx->saved_data["groups"].toInt();
    const double eps = ctx->saved_data["eps"].toDouble();
    return spread(Backward<NormBackward>::call(maybe(given_grads[0]), maybe(dr), x, w, maybe(gate), maybe(scale), maybe(r),
                                               groups, eps, wanted),
                  wanted, 7);
  }
};

variable_list norm_autograd(const Tensor& x, const Tensor& w, const OptTensor& gate_, const OptTensor& residual_,
                            const OptTensor& scale_, int64_t groups, double eps) {
  const Tensor gate = given(gate_), residual = given(residual_), scale = given(scale_);
  refuse_tangents("fused_norm", {x, w, gate, residual, scale});
  if (!wants_grad({x, w, gate, residual, scale})) {
    BelowAutograd below;
    return fused_norm(x, w, gate_, residual_, scale_, groups, eps);
  }
  norm_check(x, w, gate, residual, scale, groups);
  variable_list out = FusedNorm::apply(flat(x), w.contiguous(), maybe(flat(gate)), maybe(flat(residual)), maybe(dense(scale)),
                                       groups, eps);
  if (x.dim() != 2)
    for (Tensor& t : out) t = t.view(x.sizes());
  return out;
}

}  // namespace

TORCH_LIBRARY(pathtile_b200, m) {
  m.def("causal_conv(Tensor x, Tensor weight, Tensor? bias, bool silu, Tensor? initial_state, bool return_final_state, "
        "Tensor? lengths) -> Tensor[]");
  m.def("causal_conv_backward(Tensor? dy, Tensor? dstate, Tensor x, Tensor weight, Tensor? bias, Tensor? initial_state, "
        "Tensor? lengths, bool silu, bool[4] wanted) -> Tensor[]");
  m.def("causal_conv_step(Tensor(a!) state, Tensor x, Tensor weight, Tensor? bias, bool silu, Tensor? slots) -> Tensor");
  m.def("selective_scan(Tensor x, Tensor dt, Tensor A, Tensor B, Tensor C, Tensor? D, Tensor? z, Tensor? dt_bias, "
        "bool dt_softplus, Tensor? initial_state, bool return_final_state, Tensor? lengths, bool keep_checkpoints) -> Tensor[]");
  m.def("selective_scan_backward(Tensor? dy, Tensor? dstate, Tensor x, Tensor dt, Tensor A, Tensor B, Tensor C, Tensor? D, "
        "Tensor? z, Tensor? dt_bias, Tensor? initial_state, Tensor? lengths, Tensor checkpoints, bool dt_softplus, "
        "bool[9] wanted) -> Tensor[]");
  m.def("selective_scan_step(Tensor(a!) state, Tensor x, Tensor dt, Tensor A, Tensor B, Tensor C, Tensor? D, Tensor? z, "
        "Tensor? dt_bias, bool dt_softplus, Tensor? slots) -> Tensor");
  m.def("fused_norm(Tensor x, Tensor weight, Tensor? gate, Tensor? residual, Tensor? scale, int groups, float eps) "
        "-> Tensor[]");
  m.def("fused_norm_backward(Tensor? dy, Tensor? dr, Tensor x, Tensor weight, Tensor? gate, Tensor? scale, Tensor? r, "
        "int groups, float eps, bool[5] wanted) -> Tensor[]");
}

// For every device: what the kernels do not take, their checks refuse.
TORCH_LIBRARY_IMPL(pathtile_b200, CompositeExplicitAutograd, m) {
  m.impl("causal_conv", &conv_kernel);
  m.impl("causal_conv_backward", &conv_backward_kernel);
  m.impl("causal_conv_step", &conv_step_kernel);
  m.impl("selective_scan", &scan_kernel);
  m.impl("selective_scan_backward", &scan_backward_kernel);
  m.impl("selective_scan_step", &scan_step_kernel);
  m.impl("fused_norm", &norm_kernel);
  m.impl("fused_norm_backward", &norm_backward_kernel);
}

TORCH_LIBRARY_IMPL(pathtile_b200, Autograd, m) {
  m.impl("causal_conv", &conv_autograd);
  m.impl("causal_conv_step", &conv_step_autograd);
  m.impl("selective_scan", &scan_autograd);
  m.impl("selective_scan_step", &scan_step_autograd);
  m.impl("fused_norm", &norm_autograd);
  m.impl("causal_conv_backward", &Backward<ConvBackward>::autograd);
  m.impl("selective_scan_backward", &Backward<ScanBackward>::autograd);
  m.impl("fused_norm_backward", &Backward<NormBackward>::autograd);
}

PYBIND11_MODULE(_sequence, m) {
  m.doc() = "Native calls of pathtile_b200.sequence";
  m.def("causal_conv", &causal_conv);
  m.def("causal_conv_step", &causal_conv_step);
  m.def("selective_scan", &selective_scan);
  m.def("selective_scan_step", &selective_scan_step);
  m.def("fused_norm", &fused_norm);
}
