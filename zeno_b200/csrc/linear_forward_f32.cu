// Linear attention, forward, of 32-bit calls.
#include "linear_forward_impl.cuh"

namespace zb {
namespace linear {
template cudaError_t forward<float>(const ZenoLinearAttention&, void*, cudaStream_t);
}
}  // namespace zb
