// The state over the segments of a rollout, element by element: S <- keep S + what the segment adds.  In place: what a
// segment adds is read, the state in front of it (in reverse, behind it) is written.  Bound by the latency of the loads, kAhead of which are under way
// (16 heads of 128 x 128 in 8 segments, 8.4 MB in L2 both ways: a few us between the kernels that write and read them).
#include <cuda_bf16.h>

#include "policy_ops.h"

namespace zb {
namespace {

// kAhead: segments whose sums are under way at once.
template <uint32_t kAhead>
__global__ void __launch_bounds__(256) linear_walk_kernel(const LinearWalk w) {
  const uint64_t i = uint64_t(blockIdx.x) * 256 + threadIdx.x;
  const uint64_t row = blockIdx.y;
  early::wait_for_previous();
  early::let_next_start();
  if (i >= w.size) return;
  float run = w.initial ? w.initial[row * w.size + i] : 0.0f;
  float* state = w.state + row * w.segments * w.size + i;
  const float* keep = w.keep + row * w.segments;
  for (uint32_t first = 0; first < w.segments; first += kAhead) {
    float add[kAhead], kept[kAhead];
#pragma unroll
    for (uint32_t u = 0; u < kAhead; ++u) {
      const uint32_t step = first + u, seg = w.reverse ? w.segments - 1 - step : step;
      add[u] = 0.0f, kept[u] = 1.0f;
      // (the last one's sum is not asked for, and was not taken)
      if (step + 1 < w.segments) add[u] = state[seg * uint64_t(w.size)], kept[u] = keep[seg];
    }
#pragma unroll
    for (uint32_t u = 0; u < kAhead; ++u) {
      const uint32_t step = first + u, seg = w.reverse ? w.segments - 1 - step : step;
      if (step >= w.segments) break;
      state[seg * uint64_t(w.size)] = run;
      run = kept[u] == 0.0f ? add[u] : fmaf(kept[u], run, add[u]);
    }
  }
}

// out[t][kh][c] = sum over the value heads that share key head kh, in their order, rounded once.
template <class T>
__device__ __forceinline__ T rounded(float x);
template <>
__device__ __forceinline__ float rounded<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 rounded<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// blockIdx.y is the environment, blockIdx.z the gradient; a thread takes V neighbouring channels of a token's key head.
struct SharedPair {
  LinearShared of[2];
  uint32_t batch, turn;  // turn: tokens of a block
};
template <class T, int V>
__global__ void __launch_bounds__(256) linear_shared_kernel(const SharedPair pair) {
  const LinearShared s = blockIdx.z ? pair.of[1] : pair.of[0];
  early::wait_for_previous();
  early::let_next_start();
  const uint32_t pieces = s.width / V, row = pieces * s.key_heads;
  for (uint32_t j = threadIdx.x; j < pair.turn * row; j += 256) {
    const uint32_t t = blockIdx.x * pair.turn + j / row, kh = j % row / pieces, c = j % pieces * V;
    if (t >= s.tokens) return;
    for (uint32_t b = blockIdx.y; b < pair.batch; b += gridDim.y) {
      const float* from = s.from + ((uint64_t(b) * s.tokens + t) * (s.key_heads * s.group) + kh * s.group) * s.width + c;
      T* to = static_cast<T*>(s.to.data) + int64_t(b) * s.to.stride[0] + int64_t(t) * s.to.stride[1] + int64_t(kh) * s.to.stride[2] + c;
      float sum[V] = {};
      for (uint32_t g = 0; g < s.group; ++g) {
        if constexpr (V == 4) {
          const float4 x = *reinterpret_cast<const float4*>(from + uint64_t(g) * s.width);
          sum[0] += x.x, sum[1] += x.y, sum[2] += x.z, sum[3] += x.w;
        } else {
          sum[0] += from[uint64_t(g) * s.width];
        }
      }
#pragma unroll
      for (int e = 0; e < V; ++e) to[e] = rounded<T>(sum[e]);
    }
  }
}

// One block a head: its decay's gradient from those of the environments and segments, [heads][count], in a fixed order, in 64 bits.
__global__ void __launch_bounds__(1024) linear_decay_kernel(const double* from, uint64_t count, float* to) {
  __shared__ double part[32];
  from += blockIdx.x * count;
  early::wait_for_previous();
  double sum = 0.0;
#pragma unroll 8
  for (uint64_t i = threadIdx.x; i < count; i += 1024) sum += from[i];
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x >= 32) return;
  sum = part[threadIdx.x];
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  if (threadIdx.x == 0) to[blockIdx.x] = float(sum);
}

std::atomic<uint64_t> wait_limit{2000000000};  // nanoseconds that a block waits for its own products

}  // namespace

uint64_t linear_wait_limit(uint64_t nanoseconds) { return wait_limit.exchange(nanoseconds); }
uint64_t linear_patience() { return wait_limit.load(); }

cudaError_t launch_linear_walk(const LinearWalk& w, uint32_t rows, cudaStream_t stream) {
  // at most a few hundred rows are cut into segments
  const dim3 grid((w.size + 255) / 256, rows);
  return launch_early(w.segments <= 2 ? linear_walk_kernel<2> : linear_walk_kernel<8>, grid, 256, 0, stream, w);
}

cudaError_t launch_linear_shared(const LinearShared& q, const LinearShared& k, uint32_t batch, uint32_t dtype, cudaStream_t stream) {
  if (!batch || !q.tokens) return cudaSuccess;
  const bool four = q.width % 4 == 0;
  const uint32_t row = q.key_heads * (four ? q.width / 4 : q.width), turn = row < 1024 ? 1024 / row : 1;
  const SharedPair pair{{q, k}, batch, turn};
  const dim3 grid((q.tokens + turn - 1) / turn, batch < 65535 ? batch : 65535, 2);
  const auto kernel = dtype == ZENO_DTYPE_BF16 ? (four ? linear_shared_kernel<__nv_bfloat16, 4> : linear_shared_kernel<__nv_bfloat16, 1>)
                                               : (four ? linear_shared_kernel<float, 4> : linear_shared_kernel<float, 1>);
  return launch_early(kernel, grid, 256, 0, stream, pair);
}

cudaError_t launch_linear_decay(const double* from, uint64_t count, uint32_t heads, float* to, cudaStream_t stream) {
  return launch_early(linear_decay_kernel, dim3(heads), 1024, 0, stream, from, count, to);
}

}  // namespace zb
