// The states between the segments of a split rollout.
#include "policy_ops.h"

namespace zb {
namespace {

// Forward: the state in front of every segment, S <- M S + N.  Backward: the gradient behind every
// segment, R <- M^T R + N, from the last.  Where a segment drops the state, N alone: M is zero, and
// what it would be multiplied with need not be finite.  A block has 16 columns of one environment
// and head; 8 threads share a row's columns, two each.
constexpr int kCols = 16;

__global__ void __launch_bounds__(1024) walk_kernel(DeltaWalk w) {
  extern __shared__ float shared[];
  const int dk = int(w.dk), dv = int(w.dv);
  float* m = shared;                  // [dk][dk + 1]
  float* s = shared + dk * (dk + 1);  // [dk][16]
  const int c0 = int(blockIdx.y) * kCols, cols = min(kCols, dv - c0);
  const int r = threadIdx.x >> 3, c = (threadIdx.x & 7) * 2;
  const int64_t size = int64_t(dk) * dv;
  for (uint32_t g = 0; g < w.segments; ++g) {
    const int64_t at = int64_t(blockIdx.x) * w.segments + (w.reverse ? w.segments - 1 - g : g);
    const int64_t from = w.reverse ? at + 1 : at - 1;  // the segment that leads here
    float x[2] = {0.0f, 0.0f};
    if (g == 0) {
      for (int q = 0; q < 2; ++q)
        if (w.initial && r < dk && c + q < cols) x[q] = w.initial[int64_t(blockIdx.x) * size + int64_t(r) * dv + c0 + c + q];
    } else {
      for (int q = 0; q < 2; ++q)
        if (r < dk && c + q < cols) x[q] = w.n[from * size + int64_t(r) * dv + c0 + c + q];
      if (g > 1 && !w.cleared[from]) {  // the first segment's N starts from the initial state already
        for (int e = threadIdx.x; e < dk * dk; e += blockDim.x) m[e / dk * (dk + 1) + e % dk] = w.m[from * dk * dk + e];
        __syncthreads();
        if (r < dk) {
          const float* row = m + (w.reverse ? r : r * (dk + 1));
          const int step = w.reverse ? dk + 1 : 1;
          float y[2] = {0.0f, 0.0f};
#pragma unroll 4
          for (int j = 0; j < dk; ++j) {
            const float a = row[j * step];
            y[0] = fmaf(a, s[j * kCols + c], y[0]), y[1] = fmaf(a, s[j * kCols + c + 1], y[1]);
          }
          x[0] += y[0], x[1] += y[1];
        }
      }
    }
    __syncthreads();
    if (r < dk) {
      s[r * kCols + c] = x[0], s[r * kCols + c + 1] = x[1];
      for (int q = 0; q < 2; ++q)
        if (c + q < cols) w.state[at * size + int64_t(r) * dv + c0 + c + q] = x[q];
    }
    __syncthreads();
  }
}

}  // namespace

DeltaSplitLayout::DeltaSplitLayout(const ZenoDeltaRule& p, uint32_t segments) {
  const uint64_t rows = uint64_t(p.batch) * p.value_heads * segments;
  const auto align = [](uint64_t x) { return (x + 255) / 256 * 256; };
  m = align(rows * p.key_dim * p.key_dim * 4), n = align(rows * p.key_dim * p.value_dim * 4);
  total = m + 2 * n + align(rows * 4);
}

cudaError_t launch_delta_walk(const DeltaWalk& w, uint32_t rows, cudaStream_t stream) {
  static std::atomic<uint64_t> allowed{0};
  const cudaError_t e = allow_smem(walk_kernel, 80 * 1024, allowed);
  if (e != cudaSuccess) return e;
  const int smem = int(w.dk * (w.dk + 1) + w.dk * kCols) * 4;
  walk_kernel<<<dim3(rows, (w.dv + kCols - 1) / kCols), (8 * w.dk + 31) / 32 * 32, smem, stream>>>(w);
  return cudaGetLastError();
}

}  // namespace zb
