// Newton-Schulz orthogonalisation of update matrices.
//
//   X = M / (|M|_F + 1e-7) (transposed so that it is wide), then `steps` times
//   A = X X^T,  B = b A + c A A,  X <- a X + B X
//
// Each singular value s of X goes through the odd polynomial a s + b s^3 + c s^5, which takes
// (0, 1] towards 1.
#include <cuda_bf16.h>

#include "policy_ops.h"

namespace zb {
namespace ns {
namespace {

constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f, kEps = 1e-7f;
constexpr int kTile = 64, kDeep = 16, kNormBlocks = 64;

template <class T>
__device__ __forceinline__ float up(T x) { return float(x); }
template <>
__device__ __forceinline__ float up(__nv_bfloat16 x) { return __bfloat162float(x); }

struct Matrix {  // one matrix of the call as the wide X [m][n]
  uint32_t count, m, n;
  int64_t matrix, row, col;  // strides of X's element (i, j) in the caller's array
};

// Partial sums of squares: block y of matrix x.
template <class T>
__global__ void __launch_bounds__(256) norm_kernel(const T* from, Matrix s, float* part) {
  __shared__ float sum[8];
  const T* at = from + int64_t(blockIdx.x) * s.matrix;
  const uint64_t n = uint64_t(s.m) * s.n;
  float x = 0.0f;
  for (uint64_t i = blockIdx.y * 256ull + threadIdx.x; i < n; i += 256ull * gridDim.y) {
    const float y = up(at[int64_t(i / s.n) * s.row + int64_t(i % s.n) * s.col]);
    x = fmaf(y, y, x);
  }
  for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
  if ((threadIdx.x & 31) == 0) sum[threadIdx.x >> 5] = x;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; ++i) x += sum[i];
    part[blockIdx.x * gridDim.y + blockIdx.y] = x;
  }
}

template <class T>
__global__ void __launch_bounds__(256) scale_kernel(const T* from, Matrix s, const float* part, uint32_t parts, float* x) {
  float sum = 0.0f;
  for (uint32_t i = 0; i < parts; ++i) sum += part[blockIdx.x * parts + i];
  const float f = 1.0f / (sqrtf(sum) + kEps);
  const T* at = from + int64_t(blockIdx.x) * s.matrix;
  const uint64_t n = uint64_t(s.m) * s.n;
  for (uint64_t i = blockIdx.y * 256ull + threadIdx.x; i < n; i += 256ull * gridDim.y)
    x[blockIdx.x * n + i] = up(at[int64_t(i / s.n) * s.row + int64_t(i % s.n) * s.col]) * f;
}

// out = p L R + q add, all [rows][cols] of one matrix a grid plane; R is [depth][cols], or its transpose (BT).
template <bool BT>
__global__ void __launch_bounds__(256) product_kernel(const float* l, const float* r, const float* add, float* out, uint32_t rows,
                                                      uint32_t cols, uint32_t depth, float p, float q) {
  __shared__ float sl[kDeep][kTile + 4], sr[kDeep][kTile + 4];
  const uint64_t z = blockIdx.z;
  l += z * rows * depth, r += z * cols * depth, add += z * rows * cols, out += z * rows * cols;
  const uint32_t i0 = blockIdx.y * kTile, j0 = blockIdx.x * kTile;
  const int ti = threadIdx.x / 16 * 4, tj = threadIdx.x % 16 * 4;
  float acc[4][4] = {};
  for (uint32_t k0 = 0; k0 < depth; k0 += kDeep) {
    for (int e = threadIdx.x; e < kTile * kDeep; e += 256) {
      const uint32_t i = e / kDeep, k = e % kDeep;
      sl[k][i] = i0 + i < rows && k0 + k < depth ? l[uint64_t(i0 + i) * depth + k0 + k] : 0.0f;
      if (BT) {
        sr[k][i] = j0 + i < cols && k0 + k < depth ? r[uint64_t(j0 + i) * depth + k0 + k] : 0.0f;
      } else {
        const uint32_t j = e % kTile, kk = e / kTile;
        sr[kk][j] = j0 + j < cols && k0 + kk < depth ? r[uint64_t(k0 + kk) * cols + j0 + j] : 0.0f;
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kDeep; ++k) {
      float a[4], b[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) a[x] = sl[k][ti + x], b[x] = sr[k][tj + x];
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int y = 0; y < 4; ++y) acc[x][y] = fmaf(a[x], b[y], acc[x][y]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int x = 0; x < 4; ++x)
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const uint32_t i = i0 + ti + x, j = j0 + tj + y;
      if (i < rows && j < cols) {
        const uint64_t at = uint64_t(i) * cols + j;
        out[at] = fmaf(p, acc[x][y], q == 0.0f ? 0.0f : q * add[at]);
      }
    }
}

template <class T>
__global__ void __launch_bounds__(256) store_kernel(const float* x, T* out, uint32_t m, uint32_t n, bool transposed) {
  const uint64_t size = uint64_t(m) * n;
  for (uint64_t i = blockIdx.y * 256ull + threadIdx.x; i < size; i += 256ull * gridDim.y) {
    const uint64_t from = transposed ? (i % m) * n + i / m : i;
    const float y = x[blockIdx.x * size + from];
    if constexpr (sizeof(T) == 2) out[blockIdx.x * size + i] = __float2bfloat16_rn(y);
    else out[blockIdx.x * size + i] = y;
  }
}

uint64_t align(uint64_t x) { return (x + 255) / 256 * 256; }

template <class T>
cudaError_t run(const void* update, const Matrix& s, bool transposed, void* out, uint32_t steps, void* workspace, cudaStream_t stream) {
  const uint64_t xs = align(uint64_t(s.count) * s.m * s.n * 4), as = align(uint64_t(s.count) * s.m * s.m * 4);
  char* at = static_cast<char*>(workspace);
  float* x = reinterpret_cast<float*>(at);
  float* y = reinterpret_cast<float*>(at + xs);
  float* a = reinterpret_cast<float*>(at + 2 * xs);
  float* b = reinterpret_cast<float*>(at + 2 * xs + as);
  float* part = reinterpret_cast<float*>(at + 2 * xs + 2 * as);
  const T* from = static_cast<const T*>(update);
  const dim3 grid(s.count, kNormBlocks);
  norm_kernel<T><<<grid, 256, 0, stream>>>(from, s, part);
  scale_kernel<T><<<grid, 256, 0, stream>>>(from, s, part, kNormBlocks, x);
  const uint32_t mt = (s.m + kTile - 1) / kTile, nt = (s.n + kTile - 1) / kTile;
  for (uint32_t i = 0; i < steps; ++i) {
    product_kernel<true><<<dim3(mt, mt, s.count), 256, 0, stream>>>(x, x, a, a, s.m, s.m, s.n, 1.0f, 0.0f);
    product_kernel<true><<<dim3(mt, mt, s.count), 256, 0, stream>>>(a, a, a, b, s.m, s.m, s.m, kC, kB);
    product_kernel<false><<<dim3(nt, mt, s.count), 256, 0, stream>>>(b, x, x, y, s.m, s.n, s.m, 1.0f, kA);
    float* t = x;
    x = y, y = t;
  }
  store_kernel<T><<<grid, 256, 0, stream>>>(x, static_cast<T*>(out), s.m, s.n, transposed);
  return cudaGetLastError();
}

}  // namespace
}  // namespace ns

uint64_t orthogonalize_workspace(uint32_t count, uint32_t rows, uint32_t cols, uint32_t) {
  const uint64_t m = rows < cols ? rows : cols, n = rows < cols ? cols : rows;
  return 2 * ns::align(count * m * n * 4) + 2 * ns::align(count * m * m * 4) + ns::align(uint64_t(count) * ns::kNormBlocks * 4);
}

cudaError_t launch_orthogonalize(const void* update, const int64_t* strides, void* out, uint32_t count, uint32_t rows, uint32_t cols,
                                 uint32_t dtype, uint32_t steps, void* workspace, cudaStream_t stream) {
  const bool t = rows > cols;
  const ns::Matrix s{count, t ? cols : rows, t ? rows : cols, strides[0], t ? strides[2] : strides[1], t ? strides[1] : strides[2]};
  return dtype == ZENO_DTYPE_BF16 ? ns::run<__nv_bfloat16>(update, s, t, out, steps, workspace, stream)
                                  : ns::run<float>(update, s, t, out, steps, workspace, stream);
}

}  // namespace zb
