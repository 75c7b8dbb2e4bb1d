// C entries of the policy operators (declared in include/zeno.h): the checks of their
// arguments, then the launches.
#include "policy_ops.h"

#include <string>

namespace zb {
// Defined in capi.cpp: records the message returned by zeno_last_error().
void set_last_error(const std::string& msg);

namespace {

int refuse(const char* what, const std::string& why) {
  set_last_error(std::string(what) + ": " + why);
  return ZENO_INVALID_ARGUMENT;
}

int status(const char* what, cudaError_t e) {
  if (e == cudaSuccess) return ZENO_SUCCESS;
  set_last_error(std::string(what) + ": " + cudaGetErrorString(e));
  return ZENO_METAL_ERROR;
}

size_t item(uint32_t dtype) { return dtype == ZENO_DTYPE_BF16 ? 2 : 4; }

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// The sizes and types of a call; "" if they can be computed.
std::string shape_fault(const ZenoDeltaRule& p) {
  if (p.dtype != ZENO_DTYPE_F32 && p.dtype != ZENO_DTYPE_BF16) return "dtype must be float32 or bfloat16";
  if (p.key_dim < 1 || p.key_dim > kDeltaMaxDim || p.value_dim < 1 || p.value_dim > kDeltaMaxDim)
    return "key_dim and value_dim must be 1 to " + std::to_string(kDeltaMaxDim) + ", got " +
           std::to_string(p.key_dim) + " and " + std::to_string(p.value_dim);
  if (p.key_heads < 1 || p.value_heads < 1 || p.value_heads % p.key_heads)
    return "value_heads must be a multiple of key_heads, got " + std::to_string(p.value_heads) + " and " +
           std::to_string(p.key_heads);
  if (p.value_heads > 65535) return "more than 65535 value heads";
  // one block for each environment and head (and a few slices of a state) in a grid's first dimension
  if (uint64_t(p.batch) * p.value_heads > (uint64_t(1) << 27)) return "batch * value_heads exceeds 2^27";
  if (p.tokens > (1u << 30)) return "more than 2^30 tokens";
  return "";
}

std::string tensor_fault(const char* name, const ZenoTensor& t, size_t size) {
  if (!t.data) return std::string(name) + " is NULL";
  if (!aligned(t.data, size)) return std::string(name) + " is not aligned to its elements";
  return "";
}

std::string data_fault(const ZenoDeltaRule& p) {
  std::string why = shape_fault(p);
  if (!why.empty()) return why;
  if (!aligned(p.initial_state, 4) || !aligned(p.final_state, 4)) return "a state is not aligned to its elements";
  if (!p.batch || !p.tokens) return "";
  const size_t size = item(p.dtype);
  const struct { const char* name; const ZenoTensor* t; size_t size; } all[] = {
      {"q", &p.q, size}, {"k", &p.k, size}, {"v", &p.v, size}, {"out", &p.out, size}, {"g", &p.g, 4}, {"beta", &p.beta, 4}};
  for (const auto& x : all) {
    why = tensor_fault(x.name, *x.t, x.size);
    if (!why.empty()) return why;
  }
  return "";
}

// The sizes and types of a call; "" if they can be computed.
std::string shape_fault(const ZenoLinearAttention& p) {
  ZenoDeltaRule same{};
  same.batch = p.batch, same.tokens = p.tokens, same.key_heads = p.key_heads, same.value_heads = p.value_heads;
  same.key_dim = p.key_dim, same.value_dim = p.value_dim, same.dtype = p.dtype;
  return shape_fault(same);
}

// `out`: the tensor that takes out's place.
std::string data_fault(const ZenoLinearAttention& p, const char* out_name, const ZenoTensor& out) {
  std::string why = shape_fault(p);
  if (!why.empty()) return why;
  if (!aligned(p.initial_state, 4) || !aligned(p.final_state, 4)) return "a state is not aligned to its elements";
  if (!p.batch || !p.tokens) return "";
  const size_t size = item(p.dtype);
  const struct { const char* name; const ZenoTensor* t; size_t size; } all[] = {
      {"q", &p.q, size}, {"k", &p.k, size}, {"v", &p.v, size}, {out_name, &out, size}, {"g", &p.g, 4}};
  for (const auto& x : all) {
    why = tensor_fault(x.name, *x.t, x.size);
    if (!why.empty()) return why;
  }
  return "";
}

std::string norm_fault(const ZenoLayerNorm& p) {
  if (p.dtype != ZENO_DTYPE_F32 && p.dtype != ZENO_DTYPE_BF16) return "dtype must be float32 or bfloat16";
  if (p.affine_dtype != ZENO_DTYPE_F32 && p.affine_dtype != p.dtype) return "affine_dtype must be float32 or dtype";
  if (p.width < 1 || p.width > (1u << 30)) return "width must be 1 to 2^30";
  uint64_t rows = 1;
  bool none = false;
  for (uint64_t r : p.rows) none |= r == 0;
  for (uint64_t r : p.rows) {
    if (!none && (r > (uint64_t(1) << 31) || rows * r > (uint64_t(1) << 31))) return "more than 2^31 rows";
    rows *= none ? 1 : r;
  }
  return "";
}

bool no_rows(const ZenoLayerNorm& p) { return !p.rows[0] || !p.rows[1] || !p.rows[2]; }

std::string norm_data_fault(const ZenoLayerNorm& p, const char* out_name, const ZenoTensor& out) {
  std::string why = norm_fault(p);
  if (!why.empty()) return why;
  if (!aligned(p.weight, item(p.affine_dtype)) || !aligned(p.bias, item(p.affine_dtype))) return "weight or bias is not aligned to its elements";
  if (!aligned(p.saved, 4)) return "saved is not aligned to its elements";
  if (no_rows(p)) return "";
  why = tensor_fault("x", p.x, item(p.dtype));
  return why.empty() ? tensor_fault(out_name, out, item(p.dtype)) : why;
}

std::string matrix_fault(uint32_t count, uint32_t rows, uint32_t cols, uint32_t dtype) {
  if (dtype != ZENO_DTYPE_F32 && dtype != ZENO_DTYPE_BF16) return "dtype must be float32 or bfloat16";
  if (count > 65535) return "more than 65535 matrices";
  if (rows > (1u << 20) || cols > (1u << 20) || (rows < cols ? rows : cols) > (1u << 15))
    return "a matrix has at most 2^20 rows and columns, and 2^15 of one of them";
  return "";
}

}  // namespace
}  // namespace zb

extern "C" {

int zeno_delta_rule_step(const ZenoDeltaRule* p, void* cuda_stream) {
  constexpr const char* what = "zeno_delta_rule_step";
  if (!p) return zb::refuse(what, "NULL arguments");
  const std::string why = zb::data_fault(*p);
  if (!why.empty()) return zb::refuse(what, why);
  if (!p->batch) return ZENO_SUCCESS;
  return zb::status(what, zb::launch_delta_recurrent(*p, static_cast<cudaStream_t>(cuda_stream)));
}

uint64_t zeno_delta_rule_saved_bytes(const ZenoDeltaRule* p) {
  return p && zb::shape_fault(*p).empty() ? zb::delta_saved_bytes(*p) : 0;
}

uint64_t zeno_delta_rule_workspace_bytes(const ZenoDeltaRule* p, uint32_t pass) {
  if (!p || !zb::shape_fault(*p).empty()) return 0;
  return pass == ZENO_DELTA_BACKWARD ? zb::delta_backward_workspace(*p) : zb::delta_forward_workspace(*p);
}

int zeno_delta_rule_forward(const ZenoDeltaRule* p, void* workspace, uint64_t workspace_bytes, void* cuda_stream) {
  constexpr const char* what = "zeno_delta_rule_forward";
  if (!p) return zb::refuse(what, "NULL arguments");
  const std::string why = zb::data_fault(*p);
  if (!why.empty()) return zb::refuse(what, why);
  const uint64_t need = zeno_delta_rule_workspace_bytes(p, ZENO_DELTA_FORWARD);
  if (workspace_bytes < need) return zb::refuse(what, "workspace is too small");
  if (need && !workspace) return zb::refuse(what, "workspace is NULL");
  if (!zb::aligned(p->saved, 16) || !zb::aligned(workspace, 16)) return zb::refuse(what, "saved and workspace must be aligned to 16 bytes");
  if (!p->batch) return ZENO_SUCCESS;
  return zb::status(what, zb::launch_delta_forward(*p, workspace, static_cast<cudaStream_t>(cuda_stream)));
}

int zeno_delta_rule_backward(const ZenoDeltaRule* p, const ZenoDeltaRuleGrads* d, void* workspace, uint64_t workspace_bytes,
                             void* cuda_stream) {
  constexpr const char* what = "zeno_delta_rule_backward";
  if (!p || !d) return zb::refuse(what, "NULL arguments");
  ZenoDeltaRule inputs = *p;
  inputs.out = d->d_out;  // out itself is not read
  std::string why = zb::data_fault(inputs);
  if (!why.empty()) return zb::refuse(what, why);
  const size_t size = zb::item(p->dtype);
  const struct { const char* name; const ZenoTensor* t; size_t size; } all[] = {
      {"d_q", &d->d_q, size}, {"d_k", &d->d_k, size}, {"d_v", &d->d_v, size}, {"d_g", &d->d_g, 4}, {"d_beta", &d->d_beta, 4}};
  for (const auto& x : all) {
    why = p->batch && p->tokens ? zb::tensor_fault(x.name, *x.t, x.size) : "";
    if (!why.empty()) return zb::refuse(what, why);
  }
  if (!zb::aligned(d->d_final, 4) || !zb::aligned(d->d_initial, 4)) return zb::refuse(what, "a state is not aligned to its elements");
  if (!zb::aligned(p->saved, 16) || !zb::aligned(workspace, 16)) return zb::refuse(what, "saved and workspace must be aligned to 16 bytes");
  if (!p->saved && zb::delta_saved_bytes(*p)) return zb::refuse(what, "saved is NULL");
  const uint64_t need = zeno_delta_rule_workspace_bytes(p, ZENO_DELTA_BACKWARD);
  if (workspace_bytes < need) return zb::refuse(what, "workspace is too small");
  if (need && !workspace) return zb::refuse(what, "workspace is NULL");
  if (!p->batch) return ZENO_SUCCESS;
  return zb::status(what, zb::launch_delta_backward(*p, *d, workspace, static_cast<cudaStream_t>(cuda_stream)));
}

int zeno_linear_attention_step(const ZenoLinearAttention* p, void* cuda_stream) {
  constexpr const char* what = "zeno_linear_attention_step";
  if (!p) return zb::refuse(what, "NULL arguments");
  if (p->tokens != 1) return zb::refuse(what, "tokens must be 1");
  const std::string why = zb::data_fault(*p, "out", p->out);
  if (!why.empty()) return zb::refuse(what, why);
  if (!p->batch) return ZENO_SUCCESS;
  return zb::status(what, zb::launch_linear_step(*p, static_cast<cudaStream_t>(cuda_stream)));
}

uint64_t zeno_linear_attention_wait_limit(uint64_t nanoseconds) { return zb::linear_wait_limit(nanoseconds); }

uint64_t zeno_linear_attention_saved_bytes(const ZenoLinearAttention* p) {
  return p && zb::shape_fault(*p).empty() ? zb::linear_saved_bytes(*p) : 0;
}

uint64_t zeno_linear_attention_workspace_bytes(const ZenoLinearAttention* p, uint32_t pass) {
  if (!p || !zb::shape_fault(*p).empty()) return 0;
  return pass == ZENO_LINEAR_BACKWARD ? zb::linear_backward_workspace(*p) : zb::linear_forward_workspace(*p);
}

int zeno_linear_attention_forward(const ZenoLinearAttention* p, void* workspace, uint64_t workspace_bytes, void* cuda_stream) {
  constexpr const char* what = "zeno_linear_attention_forward";
  if (!p) return zb::refuse(what, "NULL arguments");
  const std::string why = zb::data_fault(*p, "out", p->out);
  if (!why.empty()) return zb::refuse(what, why);
  const uint64_t need = zeno_linear_attention_workspace_bytes(p, ZENO_LINEAR_FORWARD);
  if (workspace_bytes < need) return zb::refuse(what, "workspace is too small");
  if (need && !workspace) return zb::refuse(what, "workspace is NULL");
  if (!zb::aligned(p->saved, 16) || !zb::aligned(workspace, 16)) return zb::refuse(what, "saved and workspace must be aligned to 16 bytes");
  if (!p->batch) return ZENO_SUCCESS;
  return zb::status(what, zb::launch_linear_forward(*p, workspace, static_cast<cudaStream_t>(cuda_stream)));
}

int zeno_linear_attention_backward(const ZenoLinearAttention* p, const ZenoLinearAttentionGrads* d, void* workspace,
                                   uint64_t workspace_bytes, void* cuda_stream) {
  constexpr const char* what = "zeno_linear_attention_backward";
  if (!p || !d) return zb::refuse(what, "NULL arguments");
  std::string why = zb::data_fault(*p, "d_out", d->d_out);
  if (!why.empty()) return zb::refuse(what, why);
  const size_t size = zb::item(p->dtype);
  const struct { const char* name; const ZenoTensor* t; } all[] = {{"d_q", &d->d_q}, {"d_k", &d->d_k}, {"d_v", &d->d_v}};
  for (const auto& x : all) {
    why = p->batch && p->tokens ? zb::tensor_fault(x.name, *x.t, size) : "";
    if (!why.empty()) return zb::refuse(what, why);
  }
  if (!zb::aligned(d->d_g.data, 4) || !zb::aligned(d->d_decay, 4)) return zb::refuse(what, "d_g or d_decay is not aligned to its elements");
  if (!zb::aligned(d->d_final, 4) || !zb::aligned(d->d_initial, 4)) return zb::refuse(what, "a state is not aligned to its elements");
  if (!zb::aligned(p->saved, 16) || !zb::aligned(workspace, 16)) return zb::refuse(what, "saved and workspace must be aligned to 16 bytes");
  if (!p->saved && p->batch && zb::linear_saved_bytes(*p)) return zb::refuse(what, "saved is NULL");
  const uint64_t need = zeno_linear_attention_workspace_bytes(p, ZENO_LINEAR_BACKWARD);
  if (workspace_bytes < need) return zb::refuse(what, "workspace is too small");
  if (need && !workspace) return zb::refuse(what, "workspace is NULL");
  if (!p->batch && !d->d_decay) return ZENO_SUCCESS;
  return zb::status(what, zb::launch_linear_backward(*p, *d, workspace, static_cast<cudaStream_t>(cuda_stream)));
}

int zeno_layer_norm_forward(const ZenoLayerNorm* p, void* cuda_stream) {
  constexpr const char* what = "zeno_layer_norm_forward";
  if (!p) return zb::refuse(what, "NULL arguments");
  const std::string why = zb::norm_data_fault(*p, "out", p->out);
  if (!why.empty()) return zb::refuse(what, why);
  if (zb::no_rows(*p)) return ZENO_SUCCESS;
  return zb::status(what, zb::launch_layer_norm_forward(*p, static_cast<cudaStream_t>(cuda_stream)));
}

uint64_t zeno_layer_norm_workspace_bytes(const ZenoLayerNorm* p) {
  return p && zb::norm_fault(*p).empty() ? zb::layer_norm_workspace(*p) : 0;
}

int zeno_layer_norm_backward(const ZenoLayerNorm* p, const ZenoLayerNormGrads* d, void* workspace, uint64_t workspace_bytes,
                             void* cuda_stream) {
  constexpr const char* what = "zeno_layer_norm_backward";
  if (!p || !d) return zb::refuse(what, "NULL arguments");
  const std::string why = zb::norm_data_fault(*p, "d_out", d->d_out);
  if (!why.empty()) return zb::refuse(what, why);
  if (!zb::aligned(d->d_x.data, zb::item(p->dtype))) return zb::refuse(what, "d_x is not aligned to its elements");
  if (!zb::aligned(d->d_weight, zb::item(p->affine_dtype)) || !zb::aligned(d->d_bias, zb::item(p->affine_dtype)))
    return zb::refuse(what, "d_weight or d_bias is not aligned to its elements");
  if (!p->saved && !zb::no_rows(*p)) return zb::refuse(what, "saved is NULL");
  const uint64_t need = d->d_weight || d->d_bias ? zeno_layer_norm_workspace_bytes(p) : 0;
  if (workspace_bytes < need) return zb::refuse(what, "workspace is too small");
  if (need && !workspace) return zb::refuse(what, "workspace is NULL");
  if (!zb::aligned(workspace, 16)) return zb::refuse(what, "workspace must be aligned to 16 bytes");
  return zb::status(what, zb::launch_layer_norm_backward(*p, *d, workspace, static_cast<cudaStream_t>(cuda_stream)));
}

uint64_t zeno_orthogonalize_wait_limit(uint64_t nanoseconds) { return zb::orthogonalize_wait_limit(nanoseconds); }

uint64_t zeno_orthogonalize_workspace_bytes(uint32_t count, uint32_t rows, uint32_t cols, uint32_t dtype) {
  return zb::matrix_fault(count, rows, cols, dtype).empty() ? zb::orthogonalize_workspace(count, rows, cols, dtype) : 0;
}

int zeno_orthogonalize(const void* update, const int64_t* strides, void* out, uint32_t count, uint32_t rows, uint32_t cols,
                       uint32_t dtype, uint32_t steps, void* workspace, uint64_t workspace_bytes, void* cuda_stream) {
  constexpr const char* what = "zeno_orthogonalize";
  const std::string why = zb::matrix_fault(count, rows, cols, dtype);
  if (!why.empty()) return zb::refuse(what, why);
  if (steps > 100) return zb::refuse(what, "more than 100 steps");
  if (!count || !rows || !cols) return ZENO_SUCCESS;
  const uint64_t need = zeno_orthogonalize_workspace_bytes(count, rows, cols, dtype);
  if (!update || !strides || !out || (need && !workspace)) return zb::refuse(what, "NULL arguments");
  if (!zb::aligned(update, zb::item(dtype)) || !zb::aligned(out, zb::item(dtype))) return zb::refuse(what, "update or out is not aligned to its elements");
  if (!zb::aligned(workspace, 256)) return zb::refuse(what, "workspace must be aligned to 256 bytes");
  if (workspace_bytes < need) return zb::refuse(what, "workspace is too small");
  return zb::status(what, zb::launch_orthogonalize(update, strides, out, count, rows, cols, dtype, steps, workspace,
                                                   static_cast<cudaStream_t>(cuda_stream)));
}

}  // extern "C"
