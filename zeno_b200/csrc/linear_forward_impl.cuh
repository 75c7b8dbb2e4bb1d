// Launches of the forward pass for one element type.
#pragma once
#include "linear_launch.h"

namespace zb {
namespace linear {

template <class T>
cudaError_t forward(const ZenoLinearAttention& p, void* workspace, cudaStream_t stream) {
  return with_shape<T>(p, [&](auto shape) {
    using S = decltype(shape);
    const Cut c = cut_of(p);
    Segments sg{c.count, c.chunks, vec_of(p, p.out), static_cast<float*>(workspace), nullptr};
    cudaError_t e;
    if (c.count > 1) {
      sg.keep = reinterpret_cast<float*>(static_cast<char*>(workspace) + c.state);
      e = cut_states<S>(p, p.k, p.v, sg, p.initial_state, false, stream);
      if (e != cudaSuccess) return e;
    }
    static std::atomic<uint64_t> devices{0};
    if constexpr (kTensor<S>) {
      auto kernel = tensor::linear_tensor_forward_kernel<S>;
      e = allow_smem(kernel, tensor::kForwardBytes, devices);
      if (e != cudaSuccess) return e;
      return launch_main(kernel, grid_of(p, c.count), S::THREADS, tensor::kForwardBytes, c.count > 1, stream, p, sg, linear_patience());
    } else {
      constexpr int BLOCKS = S::D == 128 ? 1 : 512 / S::THREADS;
      auto kernel = linear_forward_kernel<S, BLOCKS>;
      // the first chunk of a rollout from nothing has no state in front of it
      const int bytes = ForwardSmem<S>::bytes(p.initial_state || c.count > 1 || p.tokens > uint32_t(S::C));
      e = allow_smem(kernel, ForwardSmem<S>::bytes(true), devices);
      if (e != cudaSuccess) return e;
      return launch_main(kernel, grid_of(p, c.count), S::THREADS, bytes, c.count > 1, stream, p, sg);
    }
  });
}

}  // namespace linear
}  // namespace zb
