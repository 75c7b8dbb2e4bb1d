// Launches of the backward pass for one element type.
#pragma once
#include "linear_launch.h"

namespace zb {
namespace linear {

struct BackwardLayout {  // bytes of a workspace's parts, in this order
  uint64_t cut, shared, decay;
};
inline BackwardLayout backward_layout(const ZenoLinearAttention& p) {
  const Cut c = cut_of(p);
  BackwardLayout l{c.total, 0, 0};
  if (p.value_heads != p.key_heads) l.shared = (uint64_t(p.batch) * p.tokens * p.value_heads * p.key_dim * 4 + 15) / 16 * 16;
  l.decay = uint64_t(p.batch) * p.value_heads * c.count * 8;
  return l;
}

cudaError_t backward_by_warps(const ZenoLinearAttention& p, const ZenoLinearAttentionGrads& d, const BackwardOut& extra, uint32_t vec, cudaStream_t stream);

template <class T>
cudaError_t backward(const ZenoLinearAttention& p, const ZenoLinearAttentionGrads& d, void* workspace, cudaStream_t stream) {
  return with_shape<T>(p, [&](auto shape) {
    using S = decltype(shape);
    const Cut c = cut_of(p);
    const BackwardLayout l = backward_layout(p);
    char* at = static_cast<char*>(workspace);
    const uint32_t vec = vec_of(p, d.d_out) | vec_of(d.d_q, p.key_dim, p.dtype, kVecDq) | vec_of(d.d_k, p.key_dim, p.dtype, kVecDk) |
                         vec_of(d.d_v, p.value_dim, p.dtype, kVecDv);
    Segments sg{c.count, c.chunks, vec, reinterpret_cast<float*>(at), reinterpret_cast<float*>(at + c.state)};
    BackwardOut extra{};
    if (l.shared) {
      extra.shared_q = reinterpret_cast<float*>(at + l.cut);
      extra.shared_k = reinterpret_cast<float*>(at + l.cut + l.shared);
    }
    if (d.d_decay) extra.decay = reinterpret_cast<double*>(at + l.cut + 2 * l.shared);
    if (!p.batch) return launch_linear_decay(nullptr, 0, p.value_heads, d.d_decay, stream);
    cudaError_t e;
    if (c.count > 1) {
      e = cut_states<S>(p, p.q, d.d_out, sg, d.d_final, true, stream);
      if (e != cudaSuccess) return e;
    }
    if (sizeof(T) == 2 && warp_a_head(p) && !d.d_final) {
      e = backward_by_warps(p, d, extra, vec, stream);
    } else if constexpr (kTensor<S>) {
      static std::atomic<uint64_t> devices{0};
      auto kernel = tensor::linear_tensor_backward_kernel<S>;
      e = allow_smem(kernel, tensor::kBackwardBytes, devices);
      if (e != cudaSuccess) return e;
      e = launch_main(kernel, grid_of(p, c.count), S::THREADS, tensor::kBackwardBytes, c.count > 1, stream, p, d, sg, extra, linear_patience());
    } else {
      constexpr int BLOCKS = S::D == 128 ? 1 : 512 / S::THREADS;
      auto kernel = linear_backward_kernel<S, BLOCKS>;
      const int bytes = BackwardSmem<S>::bytes(p.initial_state || d.d_final || p.tokens > uint32_t(S::C));
      static std::atomic<uint64_t> devices{0};
      e = allow_smem(kernel, BackwardSmem<S>::bytes(true), devices);
      if (e != cudaSuccess) return e;
      static_assert(sizeof(T) == 4 || S::C * S::P <= 2 * S::PL * S::CPLANE, "dV is staged where P and D were");
      static_assert(BackwardSmem<S>::front + 2 * (4 * S::L * S::PLANE + 2 * S::PL * S::CPLANE + 3 * S::SPLANE) <= 232448, "shared memory of a block");
      e = launch_main(kernel, grid_of(p, c.count), S::THREADS, bytes, c.count > 1, stream, p, d, sg, extra);
    }
    if (e != cudaSuccess) return e;
    if (l.shared) {
      const uint32_t group = p.value_heads / p.key_heads;
      e = launch_linear_shared(LinearShared{extra.shared_q, d.d_q, p.tokens, p.key_heads, group, p.key_dim},
                               LinearShared{extra.shared_k, d.d_k, p.tokens, p.key_heads, group, p.key_dim}, p.batch, p.dtype, stream);
      if (e != cudaSuccess) return e;
    }
    return d.d_decay ? launch_linear_decay(extra.decay, uint64_t(p.batch) * c.count, p.value_heads, d.d_decay, stream) : cudaSuccess;
  });
}

}  // namespace linear
}  // namespace zb
