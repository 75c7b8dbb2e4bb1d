// The 32-bit instances of the gated delta rule's backward pass.
#include "delta_backward.cuh"

namespace zb {

cudaError_t launch_delta_backward_f32(const ZenoDeltaRule& p, const ZenoDeltaRuleGrads& d, void* workspace, cudaStream_t stream) {
  return p.key_heads == p.value_heads ? delta::own_heads<float>(p, d, workspace, stream)
                                      : delta::shared_heads<float>(p, d, workspace, stream);
}

}  // namespace zb
