// What the two Newton-Schulz kernels (tiled and one-block) share.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "policy_ops.h"

namespace zb {
namespace ns {

constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;
constexpr double kEps = 1e-7;
constexpr float kScale = 4096.0f, kUnscale = 1.0f / 4096.0f;

struct Matrix {  // the call's matrices as the wide X [m][n]
  uint32_t count, m, n;
  int64_t matrix, row, col;  // strides of X's element (i, j) in the caller's array
};

template <class T>
__device__ __forceinline__ float up(T x) { return float(x); }
template <>
__device__ __forceinline__ float up(__nv_bfloat16 x) { return __bfloat162float(x); }

// The extra exponent of X in front of the first step: 2^-E >= |X|_F = |M| / (|M| + 1e-7).  At most
// 125, for the least 32-bit number (B X has long left the 32-bit range then, a X is what counts).
__device__ __forceinline__ int first_extra(double norm) {
  const double size = norm / (norm + kEps);
  if (!(size > 0.0)) return 0;
  return max(0, -ilogb(size) - 1);
}
// ... and in front of step k
__device__ __forceinline__ int extra_at(int first, uint32_t k) { return max(0, first - 2 * int(k)); }

constexpr uint32_t kSmallRows = 64, kSmallCols = 4096;
cudaError_t launch_small(const void* update, const Matrix& s, bool transposed, void* out, uint32_t dtype, uint32_t steps,
                         cudaStream_t stream);

}  // namespace ns
}  // namespace zb
