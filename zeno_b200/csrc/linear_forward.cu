// Linear attention, forward, of bfloat16 calls, and the sizes of all.
#include "linear_forward_impl.cuh"

namespace zb {
namespace linear {
template cudaError_t forward<bf16>(const ZenoLinearAttention&, void*, cudaStream_t);
extern template cudaError_t forward<float>(const ZenoLinearAttention&, void*, cudaStream_t);
}  // namespace linear

namespace linear {
cudaError_t forward_by_warps(const ZenoLinearAttention& p, cudaStream_t stream) {
  return with_warp_shape(p, [&](auto shape, auto full) {
    using S = decltype(shape);
    constexpr int WARPS = S::D == 128 ? 1 : 2, BLOCKS = S::D == 128 ? 8 : 6;  // 12 warps an SM, 8 of wide heads: registers, shared memory
    constexpr int bytes = WARPS * (int(sizeof(Gates<32>)) + 3 * 2 * S::PLANE);
    auto kernel = linear_warp_forward_kernel<S::D, decltype(full)::value, WARPS, BLOCKS>;
    static std::atomic<uint64_t> devices{0};
    const cudaError_t e = allow_smem(kernel, bytes, devices);
    if (e != cudaSuccess) return e;
    kernel<<<(p.batch * p.value_heads + WARPS - 1) / WARPS, WARPS * 32, bytes, stream>>>(p, vec_of(p, p.out));
    return cudaGetLastError();
  });
}
}  // namespace linear

uint64_t linear_saved_bytes(const ZenoLinearAttention& p) {
  const uint64_t C = uint64_t(linear::chunk_of(p)), chunks = (p.tokens + C - 1) / C;
  return chunks < 2 ? 0 : (chunks - 1) * p.batch * p.value_heads * p.key_dim * p.value_dim * 4;
}

uint64_t linear_forward_workspace(const ZenoLinearAttention& p) { return linear::cut_of(p).total; }

cudaError_t launch_linear_forward(const ZenoLinearAttention& p, void* workspace, cudaStream_t stream) {
  if (linear::warp_a_head(p)) return linear::forward_by_warps(p, stream);
  return p.dtype == ZENO_DTYPE_BF16 ? linear::forward<linear::bf16>(p, workspace, stream) : linear::forward<float>(p, workspace, stream);
}

}  // namespace zb
