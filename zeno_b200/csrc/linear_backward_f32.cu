// Gradients of the linear attention, of 32-bit calls.
#include "linear_backward_impl.cuh"

namespace zb {
namespace linear {
template cudaError_t backward<float>(const ZenoLinearAttention&, const ZenoLinearAttentionGrads&, void*, cudaStream_t);
}
}  // namespace zb
