// Launchers of the policy operators (gated delta rule, Newton-Schulz orthogonalisation),
// shared by the kernels' files and the C entries in policy_ops.cpp.
#pragma once
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "../../include/zeno.h"

namespace zb {

constexpr int kDeltaMaxDim = 128;  // largest key or value width of a head
constexpr int kDeltaChunk = 32;    // tokens of one chunk (one lane each in the gate scan)
constexpr float kNormEps = 1e-6f;  // under the root of the norms of q and k
constexpr uint32_t kSms = 148;     // of a B200

// Lets a kernel use `bytes` of dynamic shared memory, once for each device.
template <class Kernel>
cudaError_t allow_smem(Kernel kernel, int bytes, std::atomic<uint64_t>& devices) {
  if (bytes <= 48 * 1024) return cudaSuccess;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (dev < 64 && (devices.load(std::memory_order_relaxed) & bit)) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev < 64) devices.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

// Launches a kernel whose blocks may start while the one in front of it in the stream still runs, where that one lets them
// (let_next_start); each waits for its end (wait_for_previous) before it reads what it wrote, or writes anything.
template <class... Params, class... Args>
cudaError_t launch_early(void (*kernel)(Params...), dim3 grid, int threads, int smem, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t c{};
  c.gridDim = grid, c.blockDim = dim3(threads), c.dynamicSmemBytes = size_t(smem), c.stream = stream;
  cudaLaunchAttribute a{};
  a.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  a.val.programmaticStreamSerializationAllowed = 1;
  c.attrs = &a, c.numAttrs = 1;
  return cudaLaunchKernelEx(&c, kernel, args...);
}
#ifdef __CUDACC__
namespace early {
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
}  // namespace early
#endif

// A rollout in segments: what takes the state over a segment is M S + N.
struct DeltaWalk {
  const float* m;      // [rows][segments][dk][dk]: M, in the forward walk M^T
  const float* n;      // [rows][segments][dk][dv]
  float* state;        // written, same shape: in front of each segment (behind it in reverse)
  const int* cleared;  // [rows][segments]: the segment drops the state
  const float* initial;  // [rows][dk][dv] or NULL
  uint32_t segments, dk, dv;
  bool reverse;
};
struct DeltaSplitLayout {  // bytes of m, of n and of state, and of all with cleared behind them
  uint64_t m, n, total;
  DeltaSplitLayout(const ZenoDeltaRule& p, uint32_t segments);
};
cudaError_t launch_delta_walk(const DeltaWalk& w, uint32_t rows, cudaStream_t stream);
cudaError_t launch_delta_transitions(const ZenoDeltaRule& p, float* m, int* cleared, uint32_t segments, uint32_t chunks,
                                     cudaStream_t stream);

uint64_t delta_saved_bytes(const ZenoDeltaRule& p);
uint64_t delta_backward_workspace(const ZenoDeltaRule& p);
cudaError_t launch_delta_recurrent(const ZenoDeltaRule& p, cudaStream_t stream);
uint64_t delta_forward_workspace(const ZenoDeltaRule& p);
cudaError_t launch_delta_forward(const ZenoDeltaRule& p, void* workspace, cudaStream_t stream);
cudaError_t launch_delta_backward(const ZenoDeltaRule& p, const ZenoDeltaRuleGrads& d, void* workspace, cudaStream_t stream);

// Linear attention over the segments of few long rollouts: S <- keep S + what the segment adds.
struct LinearWalk {
  float* state;          // [rows][segments][size]: read as what a segment adds, written as the state in front of it
  const float* keep;     // [rows][segments]
  const float* initial;  // [rows][size] or NULL
  uint32_t segments, size;
  bool reverse;          // from the last segment back; written is the state behind a segment
};
struct LinearShared {  // gradients of a key head's rows from those of its value heads
  const float* from;   // [batch][tokens][key_heads * group][width]
  ZenoTensor to;
  uint32_t tokens, key_heads, group, width;
};
cudaError_t launch_linear_walk(const LinearWalk& w, uint32_t rows, cudaStream_t stream);
cudaError_t launch_linear_shared(const LinearShared& q, const LinearShared& k, uint32_t batch, uint32_t dtype, cudaStream_t stream);
cudaError_t launch_linear_decay(const double* from, uint64_t count, uint32_t heads, float* to, cudaStream_t stream);
uint64_t linear_wait_limit(uint64_t nanoseconds);  // sets it, returns the one before
uint64_t linear_patience();
uint64_t linear_saved_bytes(const ZenoLinearAttention& p);
uint64_t linear_forward_workspace(const ZenoLinearAttention& p);
uint64_t linear_backward_workspace(const ZenoLinearAttention& p);
cudaError_t launch_linear_forward(const ZenoLinearAttention& p, void* workspace, cudaStream_t stream);
cudaError_t launch_linear_backward(const ZenoLinearAttention& p, const ZenoLinearAttentionGrads& d, void* workspace, cudaStream_t stream);
cudaError_t launch_linear_step(const ZenoLinearAttention& p, cudaStream_t stream);

uint64_t layer_norm_workspace(const ZenoLayerNorm& p);
cudaError_t launch_layer_norm_forward(const ZenoLayerNorm& p, cudaStream_t stream);
cudaError_t launch_layer_norm_backward(const ZenoLayerNorm& p, const ZenoLayerNormGrads& d, void* workspace, cudaStream_t stream);

uint64_t orthogonalize_wait_limit(uint64_t nanoseconds);
uint64_t orthogonalize_workspace(uint32_t count, uint32_t rows, uint32_t cols, uint32_t dtype);
cudaError_t launch_orthogonalize(const void* update, const int64_t* strides, void* out, uint32_t count, uint32_t rows, uint32_t cols,
                                 uint32_t dtype, uint32_t steps, void* workspace, cudaStream_t stream);

}  // namespace zb
