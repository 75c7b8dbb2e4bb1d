// Gradients of the linear attention, of bfloat16 calls.
#include "linear_backward_impl.cuh"

namespace zb {
namespace linear {
template cudaError_t backward<bf16>(const ZenoLinearAttention&, const ZenoLinearAttentionGrads&, void*, cudaStream_t);
extern template cudaError_t backward<float>(const ZenoLinearAttention&, const ZenoLinearAttentionGrads&, void*, cudaStream_t);
}  // namespace linear

uint64_t linear_backward_workspace(const ZenoLinearAttention& p) {
  const linear::BackwardLayout l = linear::backward_layout(p);
  return l.cut + 2 * l.shared + l.decay;
}

cudaError_t launch_linear_backward(const ZenoLinearAttention& p, const ZenoLinearAttentionGrads& d, void* workspace, cudaStream_t stream) {
  return p.dtype == ZENO_DTYPE_BF16 ? linear::backward<linear::bf16>(p, d, workspace, stream) : linear::backward<float>(p, d, workspace, stream);
}

}  // namespace zb
