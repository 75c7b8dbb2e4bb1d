// Gradients of the linear attention, of bfloat16 calls.
#include "linear_backward_impl.cuh"

namespace zb {
namespace linear {
template cudaError_t backward<bf16>(const ZenoLinearAttention&, const ZenoLinearAttentionGrads&, void*, cudaStream_t);
extern template cudaError_t backward<float>(const ZenoLinearAttention&, const ZenoLinearAttentionGrads&, void*, cudaStream_t);
}  // namespace linear

namespace linear {
cudaError_t backward_by_warps(const ZenoLinearAttention& p, const ZenoLinearAttentionGrads& d, const BackwardOut& extra, uint32_t vec, cudaStream_t stream) {
  return with_warp_shape(p, [&](auto shape, auto full) {
    using S = decltype(shape);
    constexpr int WARPS = 1, BLOCKS = S::D == 128 ? 6 : 11;  // as shared memory has room for
    constexpr int bytes = WARPS * (int(sizeof(WarpGates)) + 4 * 2 * S::PLANE);
    auto kernel = linear_warp_backward_kernel<S::D, decltype(full)::value, WARPS, BLOCKS>;
    static std::atomic<uint64_t> devices{0};
    const cudaError_t e = allow_smem(kernel, bytes, devices);
    if (e != cudaSuccess) return e;
    kernel<<<(p.batch * p.value_heads + WARPS - 1) / WARPS, WARPS * 32, bytes, stream>>>(p, d, vec, extra);
    return cudaGetLastError();
  });
}
}  // namespace linear

uint64_t linear_backward_workspace(const ZenoLinearAttention& p) {
  const linear::BackwardLayout l = linear::backward_layout(p);
  return l.cut + 2 * l.shared + l.decay;
}

cudaError_t launch_linear_backward(const ZenoLinearAttention& p, const ZenoLinearAttentionGrads& d, void* workspace, cudaStream_t stream) {
  return p.dtype == ZENO_DTYPE_BF16 ? linear::backward<linear::bf16>(p, d, workspace, stream) : linear::backward<float>(p, d, workspace, stream);
}

}  // namespace zb
