// The states between the segments of a split rollout.
#include "policy_ops.h"

namespace zb {
namespace {

// Forward: the state in front of every segment, S <- M S + N.  Backward: the gradient behind every
// segment, R <- M^T R + N, from the last.  Where a segment drops the state, N alone: M is zero, and
// what it would be multiplied with need not be finite.
//
// A block has 16 columns of one environment and head.  m comes as [j][r] with row r of the result the
// sum over j, so a thread takes 4 rows x 4 columns with two 16-byte reads of shared memory for 16
// multiplications; four groups of threads share the sum.  (12 steps of 128 x 128, 16 rows, cold caches: 77 us;
// one thread a row and two columns, M not fetched ahead: 120.)
constexpr int kCols = 16, kGroups = 4, kThreads = 128 * kGroups;

__global__ void __launch_bounds__(kThreads) walk_kernel(DeltaWalk w) {
  extern __shared__ __align__(16) float shared[];
  const int dk = int(w.dk), dv = int(w.dv), pitch = (dk + 3) / 4 * 4 + 4;
  float* m = shared;                // [dk][pitch]
  float* s = m + dk * pitch;        // [128][16]
  float* part = s + 128 * kCols;    // [kGroups - 1][128][16]
  const int c0 = int(blockIdx.y) * kCols, cols = min(kCols, dv - c0);
  const int group = threadIdx.x >> 7, r = (threadIdx.x & 31) * 4, c = ((threadIdx.x >> 5) & 3) * 4;
  const int64_t size = int64_t(dk) * dv;
  // the next step's M is on its way while this one's sum is made (widths that are a multiple of 4)
  constexpr int kAhead = 128 * 128 / 4 / kThreads;
  const bool vec = dk % 4 == 0;
  float4 ahead[kAhead];
  const auto fetch = [&](uint32_t g) {
    if (!vec || g < 2 || g >= w.segments) return;
    const int64_t row = int64_t(blockIdx.x) * w.segments;
    const float* in = w.m + (row + (w.reverse ? w.segments - g : g - 1)) * dk * dk;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int e = threadIdx.x + u * kThreads;
      if (e < dk * (dk / 4)) ahead[u] = reinterpret_cast<const float4*>(in)[e];
    }
  };
  for (uint32_t g = 0; g < w.segments; ++g) {
    const int64_t at = int64_t(blockIdx.x) * w.segments + (w.reverse ? w.segments - 1 - g : g);
    const int64_t from = w.reverse ? at + 1 : at - 1;  // the segment that leads here
    float x[4][4] = {};
    if (group == 0) {
      const float* n = g == 0 ? (w.initial ? w.initial + int64_t(blockIdx.x) * size : nullptr) : w.n + from * size;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (n && r + i < dk && c + q < cols) x[i][q] = n[int64_t(r + i) * dv + c0 + c + q];
    }
    const bool product = g > 1 && !w.cleared[from];
    if (product && vec) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int e = threadIdx.x + u * kThreads;
        if (e < dk * (dk / 4)) *reinterpret_cast<float4*>(m + e / (dk / 4) * pitch + e % (dk / 4) * 4) = ahead[u];
      }
    }
    fetch(g + 1);
    if (product) {  // the first segment's N starts from the initial state already
      if (!vec) {
        const float* in = w.m + from * dk * dk;
        for (int e = threadIdx.x; e < dk * (pitch - 4); e += kThreads) {
          const int j = e / (pitch - 4), i = e % (pitch - 4);
          m[j * pitch + i] = i < dk ? in[j * dk + i] : 0.0f;
        }
      }
      __syncthreads();
      if (r < dk) {
        const int each = (dk + kGroups - 1) / kGroups, last = min(dk, (group + 1) * each);
#pragma unroll 4
        for (int j = group * each; j < last; ++j) {
          const float4 a4 = *reinterpret_cast<const float4*>(m + j * pitch + r), b4 = *reinterpret_cast<const float4*>(s + j * kCols + c);
          const float a[4] = {a4.x, a4.y, a4.z, a4.w}, b[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) x[i][q] = fmaf(a[i], b[q], x[i][q]);
        }
        if (group > 0) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<float4*>(part + ((group - 1) * 128 + r + i) * kCols + c) = make_float4(x[i][0], x[i][1], x[i][2], x[i][3]);
        }
      }
      __syncthreads();
      if (group == 0 && r < dk) {
#pragma unroll
        for (int u = 0; u < kGroups - 1; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float4 y = *reinterpret_cast<const float4*>(part + (u * 128 + r + i) * kCols + c);
            x[i][0] += y.x, x[i][1] += y.y, x[i][2] += y.z, x[i][3] += y.w;
          }
      }
    }
    if (group == 0 && r < dk) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        *reinterpret_cast<float4*>(s + (r + i) * kCols + c) = make_float4(x[i][0], x[i][1], x[i][2], x[i][3]);
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (r + i < dk && c + q < cols) w.state[at * size + int64_t(r + i) * dv + c0 + c + q] = x[i][q];
      }
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
  const cudaError_t e = allow_smem(walk_kernel, (128 * 132 + kGroups * 128 * kCols) * 4, allowed);
  if (e != cudaSuccess) return e;
  const int dk = int(w.dk), smem = (dk * ((dk + 3) / 4 * 4 + 4) + kGroups * 128 * kCols) * 4;
  walk_kernel<<<dim3(rows, (w.dv + kCols - 1) / kCols), kThreads, smem, stream>>>(w);
  return cudaGetLastError();
}

}  // namespace zb
