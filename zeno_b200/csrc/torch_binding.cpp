// The memory operators (linear attention with decays, layer norm) as PyTorch functions: checks of arguments, allocation, the autograd
// nodes, and the calls of the C entries on the current stream.  Small calls cost what the host takes for them, and
// a gradient call passes through here twice: in Python this was 85 us of layer norm's 135, the kernels being 10.
// zeno_b200/operators.py is what users call.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>

#include <array>
#include <cmath>
#include <optional>
#include <string>

#include "../../include/zeno.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Maybe = std::optional<Tensor>;

namespace {

constexpr int64_t kMaxDim = 128, kMaxHeads = 65535, kMaxStates = 1 << 27, kMaxTokens = 1 << 30;  // linear attention
constexpr int64_t kMaxWidth = 1 << 30, kMaxRows = int64_t(1) << 31;                                 // layer norm

std::string shape_of(at::IntArrayRef s) {
  std::string r = "(";
  for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
  return r + (s.size() == 1 ? ",)" : ")");
}
std::string type_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return "torch.float32";
    case at::kBFloat16: return "torch.bfloat16";
    case at::kHalf: return "torch.float16";
    case at::kDouble: return "torch.float64";
    case at::kByte: return "torch.uint8";
    case at::kBool: return "torch.bool";
    default: return c10::toString(t);
  }
}
[[noreturn]] void bad_value(const std::string& why) { throw py::value_error(why); }
[[noreturn]] void bad_type(const std::string& why) { throw py::type_error(why); }

Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : std::nullopt; }

uint32_t dtype_of(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? ZENO_DTYPE_BF16 : ZENO_DTYPE_F32; }
bool is_ours(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16; }

void check(int code, const char* what) {
  if (code != 0)
    throw std::runtime_error(std::string(what) + " failed with error code " + std::to_string(code) + ": " + zeno_last_error());
}

// The kernels see values alone: a tangent would be lost without a word.
void refuse_tangents(const char* what, std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors)
    if (t->defined() && t->_fw_grad(0).defined()) throw std::runtime_error(std::string(what) + " has no forward-mode derivatives");
}

void expect_on(const char* name, const Tensor& t, const char* other, const Tensor& x) {
  if (t.device() != x.device()) bad_value(std::string(name) + " is on " + t.device().str() + ", " + other + " on " + x.device().str());
}
void expect(const char* name, const Tensor& t, at::IntArrayRef shape, at::ScalarType type, const Tensor& q) {
  if (t.sizes() != shape) bad_value(std::string(name) + " must have shape " + shape_of(shape) + ", got " + shape_of(t.sizes()));
  if (t.scalar_type() != type) bad_type(std::string(name) + " must be " + type_of(type) + ", got " + type_of(t.scalar_type()));
  expect_on(name, t, "q", q);
}

// t, or a copy of it where it is negative by a flag alone (part of a conjugated complex tensor): its memory holds other values.
Tensor held(const Tensor& t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }
// The same where its last axis is not contiguous.
Tensor rows(const Tensor& t_) {
  const Tensor t = held(t_);
  return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous();
}

// An empty tensor of t's shape, and of its order where that leaves the last axis contiguous.
Tensor dense_like(const Tensor& t) {
  if (t.is_contiguous()) return at::empty(t.sizes(), t.options());
  Tensor y = at::empty_like(t);
  return y.stride(-1) == 1 ? y : at::empty(t.sizes(), t.options());
}

Tensor bytes(uint64_t n, const Tensor& like) { return n ? at::empty({int64_t(n)}, like.options().dtype(at::kByte)) : Tensor(); }
void* address(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* floats(const Tensor& t) { return static_cast<float*>(address(t)); }
cudaStream_t stream_of(const Tensor& t) { return at::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// What a backward pass returns; `again`: a graph of it is asked for, which says so once it is differentiated.
variable_list once(variable_list grads, bool again, const char* what) {
  if (!again) return grads;
  const at::AutoGradMode on(true);
  variable_list there;
  for (Tensor& g : grads)
    if (g.defined()) there.push_back(g.set_requires_grad(true));
  auto error = std::make_shared<torch::autograd::DelayedError>(std::string(what) + " can be differentiated once", int64_t(there.size()));
  there = (*error)(std::move(there));
  size_t i = 0;
  for (Tensor& g : grads)
    if (g.defined()) g = there[i++];
  return grads;
}

bool wants_gradient(std::initializer_list<const Tensor*> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : tensors)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// ---------------------------------------------------------------- linear attention
// [batch, tokens, ...], or [batch, ...] of one token
ZenoTensor tensor_of(const Tensor& t, bool one) {
  ZenoTensor z{};
  if (!t.defined()) return z;
  z.data = t.data_ptr();
  int64_t at = 0;
  z.stride[0] = t.stride(at++);
  z.stride[1] = one ? 0 : t.stride(at++);
  z.stride[2] = t.dim() > at ? t.stride(at) : 0;
  return z;
}

ZenoLinearAttention linear_of(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& reset, const Tensor& initial,
                              const Tensor& out, double scale, bool one) {
  ZenoLinearAttention p{};
  p.batch = uint32_t(q.size(0)), p.tokens = one ? 1 : uint32_t(q.size(1));
  p.key_heads = uint32_t(q.size(-2)), p.value_heads = uint32_t(v.size(-2));
  p.key_dim = uint32_t(q.size(-1)), p.value_dim = uint32_t(v.size(-1));
  p.dtype = dtype_of(q), p.scale = float(scale);
  p.q = tensor_of(q, one), p.k = tensor_of(k, one), p.v = tensor_of(v, one);
  if (g.dim() == 1) p.g.data = g.data_ptr(), p.g.stride[2] = g.stride(0);
  else p.g = tensor_of(g, one);
  p.reset = tensor_of(reset, one);
  p.initial_state = floats(initial);
  p.out = tensor_of(out, one);
  return p;
}

// `lead`: the axes in front of the heads (2: batch and tokens, 1: batch).  Returns the state's shape.
std::array<int64_t, 4> check_linear(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& reset, int64_t lead) {
  if (q.dim() != lead + 2 || v.dim() != lead + 2)
    bad_value(std::string("q, k and v must be ") + (lead == 2 ? "[batch, tokens, heads, width]" : "[batch, heads, width]") + ", got " +
              shape_of(q.sizes()) + " and " + shape_of(v.sizes()));
  if (!q.is_cuda()) bad_value("expected CUDA tensors, got q on " + q.device().str());
  if (!is_ours(q.scalar_type())) bad_type("q must be float32 or bfloat16, got " + type_of(q.scalar_type()));
  const int64_t key_heads = q.size(lead), dk = q.size(lead + 1), heads = v.size(lead), dv = v.size(lead + 1);
  if (dk < 1 || dk > kMaxDim || dv < 1 || dv > kMaxDim)
    bad_value("head widths must be 1 to " + std::to_string(kMaxDim) + ", got " + std::to_string(dk) + " and " + std::to_string(dv));
  if (key_heads < 1 || heads < 1 || heads % key_heads)
    bad_value("the " + std::to_string(heads) + " value heads must be a multiple of the " + std::to_string(key_heads) + " key heads");
  // what the C entries take, before anything is allocated or cut to their types
  if (heads > kMaxHeads || q.size(0) > kMaxStates / heads || (lead == 2 && q.size(1) > kMaxTokens))
    bad_value("at most 65535 value heads, 2^27 states and 2^30 tokens, got q " + shape_of(q.sizes()) + " and " + std::to_string(heads) + " value heads");
  expect("k", k, q.sizes(), q.scalar_type(), q);
  const int64_t front[4] = {q.size(0), lead == 2 ? q.size(1) : heads, lead == 2 ? heads : dv, dv};
  expect("v", v, at::IntArrayRef(front, size_t(lead + 2)), q.scalar_type(), q);
  expect("g", g, g.dim() == 1 ? at::IntArrayRef(&heads, 1) : v.sizes().slice(0, size_t(lead + 1)), at::kFloat, q);
  if (reset.defined()) {
    if (reset.sizes() != q.sizes().slice(0, size_t(lead)))
      bad_value("reset must have shape " + shape_of(q.sizes().slice(0, size_t(lead))) + ", got " + shape_of(reset.sizes()));
    if (reset.scalar_type() != at::kByte && reset.scalar_type() != at::kBool)
      bad_type("reset must be torch.uint8 or torch.bool, got " + type_of(reset.scalar_type()));
    expect_on("reset", reset, "q", q);
  }
  return {q.size(0), heads, dk, dv};
}

struct Forward {
  Tensor out, final, saved;
};
Forward run_linear(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& reset, const Tensor& initial, double scale,
                   bool save) {
  Forward r;
  r.out = dense_like(v);
  const auto state = v.options().dtype(at::kFloat);
  r.final = at::empty({v.size(0), v.size(2), q.size(3), v.size(3)}, state);
  ZenoLinearAttention p = linear_of(q, k, v, g, reset, initial, r.out, scale, false);
  p.final_state = floats(r.final);
  const c10::cuda::CUDAGuard guard(q.device());
  if (save) {
    const uint64_t n = zeno_linear_attention_saved_bytes(&p);
    if (n) r.saved = at::empty({int64_t(n / 4)}, state), p.saved = floats(r.saved);
  }
  const uint64_t n = zeno_linear_attention_workspace_bytes(&p, ZENO_LINEAR_FORWARD);
  const Tensor w = bytes(n, q);
  check(zeno_linear_attention_forward(&p, address(w), n, stream_of(q)), "linear_attention");
  return r;
}

struct LinearAttention : torch::autograd::Function<LinearAttention> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Maybe& maybe_initial,
                               const Maybe& maybe_reset, double scale) {
    const Tensor initial = maybe_initial.value_or(Tensor()), reset = maybe_reset.value_or(Tensor());
    Forward r = run_linear(q, k, v, g, reset, initial, scale, true);
    ctx->save_for_backward({q, k, v, g, initial, reset, r.saved});
    ctx->saved_data["scale"] = scale;
    ctx->set_materialize_grads(false);
    return {r.out, r.final};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const Tensor &q = s[0], &k = s[1], &v = s[2], &g = s[3], &initial = s[4];
    const bool again = at::GradMode::is_enabled();
    const at::AutoGradMode off(false);
    const c10::cuda::CUDAGuard guard(q.device());
    const Tensor d_out = grads[0].defined() ? rows(grads[0]) : at::zeros(v.sizes(), v.options());
    const Tensor d_final = grads[1].defined() ? held(grads[1]).contiguous() : Tensor();
    ZenoLinearAttention p = linear_of(q, k, v, g, s[5], initial, d_out, ctx->saved_data["scale"].toDouble(), false);
    p.saved = floats(s[6]);
    const Tensor d_q = dense_like(q), d_k = dense_like(k), d_v = dense_like(v);
    const Tensor d_g = ctx->needs_input_grad(3) ? at::empty_like(g) : Tensor();
    const Tensor d_initial = initial.defined() && ctx->needs_input_grad(4) ? at::empty_like(initial) : Tensor();
    ZenoLinearAttentionGrads d{};
    d.d_out = p.out;
    d.d_final = floats(d_final);
    d.d_q = tensor_of(d_q, false), d.d_k = tensor_of(d_k, false), d.d_v = tensor_of(d_v, false);
    if (g.dim() == 1) d.d_decay = floats(d_g);
    else d.d_g = tensor_of(d_g, false);
    d.d_initial = floats(d_initial);
    const uint64_t n = zeno_linear_attention_workspace_bytes(&p, ZENO_LINEAR_BACKWARD);
    const Tensor w = bytes(n, q);
    check(zeno_linear_attention_backward(&p, &d, address(w), n, stream_of(q)), "linear_attention backward");
    return once({d_q, d_k, d_v, d_g, d_initial, Tensor(), Tensor()}, again, "linear_attention");
  }
};

py::tuple linear_attention(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& g_, const Maybe& reset_, const Maybe& initial_,
                           const std::optional<double>& scale_) {
  const Tensor reset = reset_.value_or(Tensor());
  Tensor initial = held(initial_.value_or(Tensor()));
  const Tensor g = held(g_);
  const auto state = check_linear(q_, k_, v_, g, reset, 2);
  if (initial.defined()) {
    expect("initial_state", initial, state, at::kFloat, q_);
    initial = initial.contiguous();
  }
  refuse_tangents("linear_attention", {&q_, &k_, &v_, &g, &initial});
  const double scale = scale_ ? *scale_ : 1.0 / std::sqrt(double(q_.size(3)));
  const Tensor q = rows(q_), k = rows(k_), v = rows(v_);
  if (wants_gradient({&q, &k, &v, &g, &initial})) {
    const variable_list r = LinearAttention::apply(q, k, v, g, maybe(initial), maybe(reset), scale);
    return py::make_tuple(r[0], r[1]);
  }
  const at::AutoGradMode off(false);
  const Forward r = run_linear(q, k, v, g, reset, initial, scale, false);
  return py::make_tuple(r.out, r.final);
}

Tensor linear_attention_step(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& g_, const Tensor& state, const Maybe& reset_,
                             const std::optional<double>& scale_) {
  const Tensor reset = reset_.value_or(Tensor()), g = held(g_);
  expect("state", state, check_linear(q_, k_, v_, g, reset, 1), at::kFloat, q_);
  if (!state.is_contiguous()) bad_value("state must be contiguous: it is updated in place");
  if (state.is_neg()) bad_value("state must hold its own values, not those of a conjugated tensor: it is updated in place");
  if (wants_gradient({&q_, &k_, &v_, &g, &state}))
    throw std::runtime_error("linear_attention_step has no gradients: call it under torch.no_grad(), and linear_attention to learn");
  refuse_tangents("linear_attention_step", {&q_, &k_, &v_, &g, &state});
  const double scale = scale_ ? *scale_ : 1.0 / std::sqrt(double(q_.size(2)));
  const at::AutoGradMode off(false);
  const Tensor q = rows(q_), k = rows(k_), v = rows(v_), out = at::empty(v.sizes(), v.options());
  ZenoLinearAttention p = linear_of(q, k, v, g, reset, state, out, scale, true);
  p.final_state = floats(state);
  const c10::cuda::CUDAGuard guard(q.device());
  check(zeno_linear_attention_step(&p, stream_of(q)), "linear_attention_step");
  if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();  // (those have no version, and are never saved for a backward pass)
  return out;
}

// ---------------------------------------------------------------- layer norm
// Rows of up to three leading axes, padded to three.
ZenoTensor rows_of(const Tensor& t) {
  ZenoTensor z{};
  if (!t.defined()) return z;
  z.data = t.data_ptr();
  const int64_t axes = t.dim() - 1;
  for (int64_t i = 0; i < axes; ++i) z.stride[3 - axes + i] = t.stride(i);
  return z;
}

ZenoLayerNorm norm_of(const Tensor& x, const Tensor& weight, at::ScalarType affine, const Tensor& bias, double eps, const Tensor& out, const Tensor& saved) {
  ZenoLayerNorm p{};
  const int64_t axes = x.dim() - 1;
  for (int64_t i = 0; i < 3; ++i) p.rows[i] = i < 3 - axes ? 1 : uint64_t(x.size(i - 3 + axes));
  p.width = uint32_t(x.size(-1));
  p.dtype = dtype_of(x);
  p.affine_dtype = affine == at::kBFloat16 ? ZENO_DTYPE_BF16 : ZENO_DTYPE_F32;
  p.eps = float(eps);
  p.x = rows_of(x), p.out = rows_of(out);
  p.weight = address(weight), p.bias = address(bias);
  p.saved = floats(saved);
  return p;
}

at::ScalarType affine_of(const Tensor& x, const Tensor& weight, const Tensor& bias) {
  return weight.defined() ? weight.scalar_type() : bias.defined() ? bias.scalar_type() : x.scalar_type();
}

Tensor run_norm(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps, Tensor* saved) {
  const Tensor out = dense_like(x);
  if (saved) *saved = at::empty({3, x.numel() / x.size(-1)}, x.options().dtype(at::kFloat));
  const ZenoLayerNorm p = norm_of(x, weight, affine_of(x, weight, bias), bias, eps, out, saved ? *saved : Tensor());
  const c10::cuda::CUDAGuard guard(x.device());
  check(zeno_layer_norm_forward(&p, stream_of(x)), "layer_norm");
  return out;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& maybe_weight, const Maybe& maybe_bias, double eps) {
    const Tensor weight = maybe_weight.value_or(Tensor()), bias = maybe_bias.value_or(Tensor());
    Tensor saved;
    const Tensor out = run_norm(x, weight, bias, eps, &saved);
    ctx->save_for_backward({x, weight, saved});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["affine"] = int64_t(affine_of(x, weight, bias));
    ctx->saved_data["bias"] = bias.defined();
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const Tensor &x = s[0], &weight = s[1];
    const bool again = at::GradMode::is_enabled();
    const at::AutoGradMode off(false);
    const c10::cuda::CUDAGuard guard(x.device());
    const auto affine = at::ScalarType(ctx->saved_data["affine"].toInt());
    const Tensor d_out = rows(grads[0]);
    const Tensor d_x = ctx->needs_input_grad(0) ? dense_like(x) : Tensor();
    const auto sums = x.options().dtype(affine);
    const Tensor d_weight = weight.defined() && ctx->needs_input_grad(1) ? at::empty({x.size(-1)}, sums) : Tensor();
    // (tensors that are not there are not counted)
    const Tensor d_bias = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(weight.defined() ? 2 : 1) ? at::empty({x.size(-1)}, sums) : Tensor();
    const ZenoLayerNorm p = norm_of(x, weight, affine, Tensor(), ctx->saved_data["eps"].toDouble(), Tensor(), s[2]);
    ZenoLayerNormGrads d{};
    d.d_out = rows_of(d_out), d.d_x = rows_of(d_x);
    d.d_weight = address(d_weight), d.d_bias = address(d_bias);
    const uint64_t n = d.d_weight || d.d_bias ? zeno_layer_norm_workspace_bytes(&p) : 0;
    const Tensor w = bytes(n, x);
    check(zeno_layer_norm_backward(&p, &d, address(w), n, stream_of(x)), "layer_norm backward");
    return once({d_x, d_weight, d_bias, Tensor()}, again, "layer_norm");
  }
};

Tensor layer_norm(const Tensor& x_, const Maybe& weight_, const Maybe& bias_, double eps) {
  Tensor weight = weight_.value_or(Tensor()), bias = bias_.value_or(Tensor());
  if (!x_.is_cuda()) bad_value("expected a CUDA tensor, got x on " + x_.device().str());
  if (!is_ours(x_.scalar_type())) bad_type("x must be float32 or bfloat16, got " + type_of(x_.scalar_type()));
  if (x_.dim() < 1 || x_.size(-1) < 1) bad_value("x needs a last axis to be normalised over, got shape " + shape_of(x_.sizes()));
  const int64_t width = x_.size(-1);
  if (width > kMaxWidth || x_.numel() / width > kMaxRows) bad_value("at most 2^31 rows of 2^30 values, got shape " + shape_of(x_.sizes()));
  const std::pair<const char*, Tensor*> both[] = {{"weight", &weight}, {"bias", &bias}};
  for (const auto& [name, t] : both) {
    if (!t->defined()) continue;
    if (t->dim() != 1 || t->size(0) != width)
      bad_value(std::string(name) + " must have shape " + shape_of(at::IntArrayRef(&width, 1)) + ", got " + shape_of(t->sizes()));
    if (t->scalar_type() != at::kFloat && t->scalar_type() != x_.scalar_type())
      bad_type(std::string(name) + " must be torch.float32 or " + type_of(x_.scalar_type()) + ", got " + type_of(t->scalar_type()));
    expect_on(name, *t, "x", x_);
    *t = held(*t).contiguous();
  }
  if (weight.defined() && bias.defined() && weight.scalar_type() != bias.scalar_type())
    bad_type("weight and bias must be of one type, got " + type_of(weight.scalar_type()) + " and " + type_of(bias.scalar_type()));
  if (!(eps >= 0.0)) bad_value("eps must not be negative, got " + std::to_string(eps));
  refuse_tangents("layer_norm", {&x_, &weight, &bias});
  Tensor x = rows(x_);
  if (x.dim() > 4) x = x.reshape({-1, width});
  Tensor out;
  if (wants_gradient({&x, &weight, &bias})) {
    out = LayerNorm::apply(x, maybe(weight), maybe(bias), eps);
  } else {
    const at::AutoGradMode off(false);
    out = run_norm(x, weight, bias, eps, nullptr);
  }
  return x.dim() == x_.dim() ? out : out.reshape(x_.sizes());
}

}  // namespace

PYBIND11_MODULE(zeno_torch, m) {
  m.def("linear_attention", &linear_attention);
  m.def("linear_attention_step", &linear_attention_step);
  m.def("layer_norm", &layer_norm);
}
