// The bfloat16 instances without shared key heads of the gated delta rule's backward pass, and its workspace.
#include "delta_backward.cuh"

namespace zb {

cudaError_t launch_delta_backward_f32(const ZenoDeltaRule& p, const ZenoDeltaRuleGrads& d, void* workspace, cudaStream_t stream);
cudaError_t launch_delta_backward_shared(const ZenoDeltaRule& p, const ZenoDeltaRuleGrads& d, void* workspace, cudaStream_t stream);

// A split rollout's states; for shared key heads, 32-bit rows of dq and dk for each value head.
uint64_t delta_backward_workspace(const ZenoDeltaRule& p) {
  const uint64_t shared = p.key_heads == p.value_heads ? 0 : 2 * uint64_t(p.batch) * p.tokens * p.value_heads * p.key_dim * 4;
  return delta::split_bytes(p) + shared;
}

cudaError_t launch_delta_backward(const ZenoDeltaRule& p, const ZenoDeltaRuleGrads& d, void* workspace, cudaStream_t stream) {
  if (p.dtype != ZENO_DTYPE_BF16) return launch_delta_backward_f32(p, d, workspace, stream);
  if (p.key_heads != p.value_heads) return launch_delta_backward_shared(p, d, workspace, stream);
  return delta::own_heads<__nv_bfloat16>(p, d, workspace, stream);
}

}  // namespace zb
