// The bfloat16 instances of the gated delta rule's backward pass for shared key heads.
#include "delta_backward.cuh"

namespace zb {

cudaError_t launch_delta_backward_shared(const ZenoDeltaRule& p, const ZenoDeltaRuleGrads& d, void* workspace, cudaStream_t stream) {
  return delta::shared_heads<__nv_bfloat16>(p, d, workspace, stream);
}

}  // namespace zb
