// Layer norm and its gradients.  With xhat = (x - mean) rstd and dh = dy w:
//   y = xhat w + b
//   dx = rstd (dh - mean(dh) - xhat mean(dh xhat)),  dw = sum over rows of dy xhat,  db = sum over rows of dy
// The time is the bytes of the rows: each is read once, held in registers, and written once.  A row of up to
// 512 values belongs to a part of a warp or a warp, a longer one to a block.  Backward, every thread keeps the
// sums of its own columns over the rows it sees; a block's sums go to the workspace and a second kernel adds them in a
// fixed order.  Sums are 32-bit (the last ones over blocks too), the variance is taken from the differences to the mean.
#include <cuda_bf16.h>

#include <algorithm>

#include "policy_ops.h"

namespace zb {
namespace {

using bf16 = __nv_bfloat16;
constexpr unsigned kAll = 0xffffffffu;
constexpr uint32_t kWide = 8192;  // longest row that a block holds in registers

// Where the rows of a tensor are.
struct RowsAt {
  int64_t stride[3];
  bool flat;  // row r is at r * stride[2]
};
struct Norm {
  const void *x, *weight, *bias, *dy;
  void *y, *dx;
  RowsAt at_x, at_y, at_dy, at_dx;
  float* saved;    // [3][rows]: the mean as summed, what that sum's rounding left of it, rstd
  float* partial;  // [blocks][2][width]: sums of dy xhat and of dy
  uint32_t rows, rows1, rows2, width;
  float eps;
};

__device__ __forceinline__ int64_t offset(const RowsAt& a, uint32_t row, const Norm& p) {
  if (a.flat) return int64_t(row) * a.stride[2];
  const uint32_t i2 = row % p.rows2, rest = row / p.rows2;
  return int64_t(rest / p.rows1) * a.stride[0] + int64_t(rest % p.rows1) * a.stride[1] + int64_t(i2) * a.stride[2];
}

// Two 32-bit values at once: sm_100 adds, multiplies and multiply-adds pairs of registers in one instruction, and the
// arithmetic of a value is what the vector units can just keep up with.
struct Two {
  uint64_t bits;
};
__device__ __forceinline__ Two two(float x, float y) {
  Two r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.bits) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 apart(Two a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.bits));
  return r;
}
__device__ __forceinline__ Two operator+(Two a, Two b) {
  Two r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits));
  return r;
}
__device__ __forceinline__ Two operator*(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits));
  return r;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits), "l"(c.bits));
  return r;
}

// V neighbouring values as 32-bit ones: one 16-byte vector, or a single value.
template <class T, int V>
__device__ __forceinline__ void fetch(float (&x)[V], const T* at) {
  if constexpr (V == 1) {
    x[0] = float(*at);
  } else if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int h = 0; h < V; h += 8) {
      const uint4 w = *reinterpret_cast<const uint4*>(at + h);
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) x[h + 2 * i] = __uint_as_float(u[i] << 16), x[h + 2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int h = 0; h < V; h += 4) {
      const float4 w = *reinterpret_cast<const float4*>(at + h);
      x[h] = w.x, x[h + 1] = w.y, x[h + 2] = w.z, x[h + 3] = w.w;
    }
  }
}
template <class T, int V>
__device__ __forceinline__ void put(T* at, const float (&x)[V]) {
  if constexpr (V == 1) {
    if constexpr (sizeof(T) == 2) *at = __float2bfloat16_rn(x[0]);
    else *at = x[0];
  } else if constexpr (sizeof(T) == 2) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      u[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(at) = make_uint4(u[0], u[1], u[2], u[3]);
  } else {
    *reinterpret_cast<float4*>(at) = make_float4(x[0], x[1], x[2], x[3]);
  }
}

// Sums over the lanes of a row.  A block's pass through `box` ([2][32], taken in turns so that one barrier is enough).
template <bool BLOCK>
__device__ __forceinline__ float row_sum(float s, int lanes, float2 (*box)[32], int& turn) {
  if (BLOCK) lanes = 32;
  for (int d = 1; d < lanes; d <<= 1) s += __shfl_xor_sync(kAll, s, d);
  if (BLOCK) {
    const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) box[turn][warp].x = s;
    __syncthreads();
    const int i = threadIdx.x & 31;
    s = i < warps ? box[turn][i].x : 0.0f;
    turn ^= 1;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) s += __shfl_xor_sync(kAll, s, d);
  }
  return s;
}
template <bool BLOCK>
__device__ __forceinline__ float2 row_sum(float2 s, int lanes, float2 (*box)[32], int& turn) {
  if (BLOCK) lanes = 32;
  for (int d = 1; d < lanes; d <<= 1) {
    s.x += __shfl_xor_sync(kAll, s.x, d);
    s.y += __shfl_xor_sync(kAll, s.y, d);
  }
  if (BLOCK) {
    const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) box[turn][warp] = s;
    __syncthreads();
    const int i = threadIdx.x & 31;
    s = i < warps ? box[turn][i] : make_float2(0.0f, 0.0f);
    turn ^= 1;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      s.x += __shfl_xor_sync(kAll, s.x, d);
      s.y += __shfl_xor_sync(kAll, s.y, d);
    }
  }
  return s;
}

// N vectors of V values a lane, K rows at once.  `lanes` of a warp (or the block) share a row.
template <class T, class W, int V, int N, int K, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? 512 : 256) norm_forward_kernel(const __grid_constant__ Norm p, const int lanes, const int lanes_log) {
  constexpr int M = N * V / 2;  // pairs of values of a lane
  __shared__ float2 box[2][32];
  int turn = 0;
  const int lane = BLOCK ? threadIdx.x : threadIdx.x & (lanes - 1);
  const uint32_t per = BLOCK ? 1 : 256u >> lanes_log;  // rows side by side in a block
  const int stride = BLOCK ? blockDim.x : lanes;
  const uint32_t row0 = blockIdx.x * (per * K) + (BLOCK ? 0 : threadIdx.x >> lanes_log);  // (below 2^31 + 2^10)
  float x[K][N][V];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const uint32_t row = row0 + k * per;
    const T* from = static_cast<const T*>(p.x) + (row < p.rows ? offset(p.at_x, row, p) : 0);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t c = uint32_t(lane + i * stride) * V;
      if (row < p.rows && c < p.width) {
        fetch(x[k][i], from + c);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) x[k][i][e] = 0.0f;
      }
    }
  }
  float mean[K], rest[K], rstd[K];
  const float inverse = 1.0f / float(p.width);
  Two y[K][M];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const float* values = &x[k][0][0];
#pragma unroll
    for (int m = 0; m < M; ++m) y[k][m] = two(values[2 * m], values[2 * m + 1]);
    Two s = y[k][0];
#pragma unroll
    for (int m = 1; m < M; ++m) s = s + y[k][m];
    const float2 t = apart(s);
    mean[k] = row_sum<BLOCK>(t.x + t.y, lanes, box, turn) * inverse;
  }
  // where a lane's values are not all there, what is not stays zero
  const bool whole = uint32_t(lane + (N - 1) * stride + 1) * V <= p.width;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const Two minus = two(-mean[k], -mean[k]);
    Two s = two(0.0f, 0.0f), q = s;
#pragma unroll
    for (int m = 0; m < M; ++m) {
      Two d = y[k][m] + minus;
      if (!whole) {
        const float2 a = apart(d);
        d = two(uint32_t(lane + 2 * m / V * stride) * V < p.width ? a.x : 0.0f, uint32_t(lane + (2 * m + 1) / V * stride) * V < p.width ? a.y : 0.0f);
      }
      y[k][m] = d, s = s + d, q = fma2(d, d, q);
    }
    const float2 a = apart(s), b = apart(q);
    const float2 t = row_sum<BLOCK>(make_float2(a.x + a.y, b.x + b.y), lanes, box, turn);
    // what the sum's rounding left of the mean
    rest[k] = t.x * inverse;
    rstd[k] = 1.0f / sqrtf(fmaxf(fmaf(-rest[k], rest[k], t.y * inverse), 0.0f) + p.eps);
    if (t.y != t.y) rstd[k] = t.y;
    const Two r = two(-rest[k], -rest[k]), f = two(rstd[k], rstd[k]);
#pragma unroll
    for (int m = 0; m < M; ++m) y[k][m] = (y[k][m] + r) * f;
  }
  // one pair for all of a lane's rows at a time; 1 and 0 where there is no weight or bias
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t c = uint32_t(lane + i * stride) * V;
    if (c >= p.width) continue;
    float w[V], b[V];
#pragma unroll
    for (int e = 0; e < V; ++e) w[e] = 1.0f, b[e] = 0.0f;
    if (p.weight) fetch(w, static_cast<const W*>(p.weight) + c);
    if (p.bias) fetch(b, static_cast<const W*>(p.bias) + c);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const uint32_t row = row0 + k * per;
      if (row >= p.rows) continue;
      float z[V];
      if constexpr (V == 1) {
        const float2 a = apart(y[k][i / 2]);
        z[0] = fmaf(i % 2 ? a.y : a.x, w[0], b[0]);
      } else {
#pragma unroll
        for (int m = 0; m < V / 2; ++m) {
          const float2 a = apart(fma2(y[k][i * V / 2 + m], two(w[2 * m], w[2 * m + 1]), two(b[2 * m], b[2 * m + 1])));
          z[2 * m] = a.x, z[2 * m + 1] = a.y;
        }
      }
      put(static_cast<T*>(p.y) + offset(p.at_y, row, p) + c, z);
    }
  }
  if (p.saved && lane == 0) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const uint32_t row = row0 + k * per;
      if (row < p.rows) p.saved[row] = mean[k], p.saved[uint64_t(p.rows) + row] = rest[k], p.saved[2 * uint64_t(p.rows) + row] = rstd[k];
    }
  }
}

// Rows from blockIdx.x on in steps of the grid; a thread's sums over its columns end in the block's line of the workspace.
template <class T, class W, int V, int N, int K, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? 512 : 256) norm_backward_kernel(const __grid_constant__ Norm p, const int lanes, const int lanes_log) {
  constexpr int M = N * V / 2;
  __shared__ float2 box[2][32];
  extern __shared__ float side[];  // sums of the rows side by side
  int turn = 0;
  const int lane = BLOCK ? threadIdx.x : threadIdx.x & (lanes - 1);
  const uint32_t per = BLOCK ? 1 : 256u >> lanes_log;
  const int stride = BLOCK ? blockDim.x : lanes;
  const uint32_t own = BLOCK ? 0 : threadIdx.x >> lanes_log;
  const float inverse = 1.0f / float(p.width);
  Two dw[M], db[M], w[M];
#pragma unroll
  for (int m = 0; m < M; ++m) dw[m] = db[m] = two(0.0f, 0.0f);
  {
    float v[N][V];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t c = uint32_t(lane + i * stride) * V;
#pragma unroll
      for (int e = 0; e < V; ++e) v[i][e] = 1.0f;
      if (p.weight && c < p.width) fetch(v[i], static_cast<const W*>(p.weight) + c);
    }
    const float* values = &v[0][0];
#pragma unroll
    for (int m = 0; m < M; ++m) w[m] = two(values[2 * m], values[2 * m + 1]);
  }
  for (uint64_t first = uint64_t(blockIdx.x) * (per * K); first < p.rows; first += uint64_t(gridDim.x) * (per * K)) {
    Two x[K][M], g[K][M];
    float mean[K], rest[K], rstd[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const uint32_t row = uint32_t(first) + own + k * per;
      const bool here = row < p.rows;
      const T* from = static_cast<const T*>(p.x) + (here ? offset(p.at_x, row, p) : 0);
      const T* grad = static_cast<const T*>(p.dy) + (here ? offset(p.at_dy, row, p) : 0);
      float a[N][V], b[N][V];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint32_t c = uint32_t(lane + i * stride) * V;
        if (here && c < p.width) {
          fetch(a[i], from + c);
          fetch(b[i], grad + c);
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) a[i][e] = b[i][e] = 0.0f;
        }
      }
      const float *va = &a[0][0], *vb = &b[0][0];
#pragma unroll
      for (int m = 0; m < M; ++m) x[k][m] = two(va[2 * m], va[2 * m + 1]), g[k][m] = two(vb[2 * m], vb[2 * m + 1]);
      mean[k] = here ? p.saved[row] : 0.0f;
      rest[k] = here ? p.saved[uint64_t(p.rows) + row] : 0.0f;
      rstd[k] = here ? p.saved[2 * uint64_t(p.rows) + row] : 0.0f;
    }
    float2 s[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const Two minus = two(-mean[k], -mean[k]), r = two(-rest[k], -rest[k]), f = two(rstd[k], rstd[k]);
      Two s0 = two(0.0f, 0.0f), s1 = s0;
#pragma unroll
      for (int m = 0; m < M; ++m) {  // (what is not there has no gradient: it adds nothing)
        const Two hat = (x[k][m] + minus + r) * f, dy = g[k][m], dh = dy * w[m];
        dw[m] = fma2(dy, hat, dw[m]), db[m] = db[m] + dy;
        s0 = s0 + dh, s1 = fma2(dh, hat, s1);
        x[k][m] = hat, g[k][m] = dh;
      }
      const float2 a = apart(s0), b = apart(s1);
      s[k] = make_float2(a.x + a.y, b.x + b.y);
    }
    if (!p.dx) continue;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const uint32_t row = uint32_t(first) + own + k * per;
      const float2 t = row_sum<BLOCK>(s[k], lanes, box, turn);
      if (row >= p.rows) continue;
      const Two m0 = two(-t.x * inverse, -t.x * inverse), m1 = two(-t.y * inverse, -t.y * inverse), f = two(rstd[k], rstd[k]);
      T* to = static_cast<T*>(p.dx) + offset(p.at_dx, row, p);
      float z[N][V];
#pragma unroll
      for (int m = 0; m < M; ++m) {
        const float2 a = apart((g[k][m] + fma2(x[k][m], m1, m0)) * f);
        (&z[0][0])[2 * m] = a.x, (&z[0][0])[2 * m + 1] = a.y;
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint32_t c = uint32_t(lane + i * stride) * V;
        if (c < p.width) put(to + c, z[i]);
      }
    }
  }
  if (!p.partial) return;
  float* line = p.partial + uint64_t(blockIdx.x) * 2 * p.width;
  const int cols = lanes * N * V;
#pragma unroll
  for (int pass = 0; pass < 2; ++pass) {
    if (!BLOCK) __syncthreads();
#pragma unroll
    for (int m = 0; m < M; ++m) {
      const float2 a = apart(pass ? db[m] : dw[m]);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t c = uint32_t(lane + (2 * m + h) / V * stride) * V + (2 * m + h) % V;
        if (!BLOCK) side[own * cols + c] = h ? a.y : a.x;
        else if (c < p.width) line[pass * p.width + c] = h ? a.y : a.x;
      }
    }
    if (BLOCK) continue;
    __syncthreads();
    for (uint32_t c = threadIdx.x; c < p.width; c += 256) {
      float sum = 0.0f;
      for (uint32_t r = 0; r < per; ++r) sum += side[r * cols + c];
      line[pass * p.width + c] = sum;
    }
  }
}

// Rows too long for registers: one block a row, which is read three times forward (from L2 after the first).
template <class T, class W>
__global__ void __launch_bounds__(1024) norm_wide_forward_kernel(const __grid_constant__ Norm p) {
  __shared__ float2 box[2][32];
  int turn = 0;
  const float inverse = 1.0f / float(p.width);
  for (uint32_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* from = static_cast<const T*>(p.x) + offset(p.at_x, row, p);
    T* to = static_cast<T*>(p.y) + offset(p.at_y, row, p);
    float2 s = make_float2(0.0f, 0.0f);
    for (uint32_t c = threadIdx.x; c < p.width; c += 1024) s.x += float(from[c]);
    const float mean = row_sum<true>(s, 32, box, turn).x * inverse;
    s = make_float2(0.0f, 0.0f);
    for (uint32_t c = threadIdx.x; c < p.width; c += 1024) {
      const float d = float(from[c]) - mean;
      s.x += d, s.y = fmaf(d, d, s.y);
    }
    s = row_sum<true>(s, 32, box, turn);
    const float rest = s.x * inverse;
    float rstd = 1.0f / sqrtf(fmaxf(fmaf(-rest, rest, s.y * inverse), 0.0f) + p.eps);
    if (s.y != s.y) rstd = s.y;
    for (uint32_t c = threadIdx.x; c < p.width; c += 1024) {
      float y[1] = {(float(from[c]) - mean - rest) * rstd};
      if (p.weight) y[0] *= float(static_cast<const W*>(p.weight)[c]);
      if (p.bias) y[0] += float(static_cast<const W*>(p.bias)[c]);
      put(to + c, y);
    }
    if (p.saved && threadIdx.x == 0) p.saved[row] = mean, p.saved[uint64_t(p.rows) + row] = rest, p.saved[2 * uint64_t(p.rows) + row] = rstd;
  }
}
template <class T, class W>
__global__ void __launch_bounds__(1024) norm_wide_backward_kernel(const __grid_constant__ Norm p) {
  __shared__ float2 box[2][32];
  int turn = 0;
  const float inverse = 1.0f / float(p.width);
  float* line = p.partial ? p.partial + uint64_t(blockIdx.x) * 2 * p.width : nullptr;
  if (line)
    for (uint32_t c = threadIdx.x; c < p.width; c += 1024) line[c] = 0.0f, line[p.width + c] = 0.0f;
  for (uint32_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* from = static_cast<const T*>(p.x) + offset(p.at_x, row, p);
    const T* grad = static_cast<const T*>(p.dy) + offset(p.at_dy, row, p);
    const float mean = p.saved[row], rest = p.saved[uint64_t(p.rows) + row], rstd = p.saved[2 * uint64_t(p.rows) + row];
    float2 s = make_float2(0.0f, 0.0f);
    for (uint32_t c = threadIdx.x; c < p.width; c += 1024) {  // a thread comes back to its own columns of the line
      const float hat = (float(from[c]) - mean - rest) * rstd, dy = float(grad[c]);
      const float dh = p.weight ? dy * float(static_cast<const W*>(p.weight)[c]) : dy;
      s.x += dh, s.y = fmaf(dh, hat, s.y);
      if (line) line[c] = fmaf(dy, hat, line[c]), line[p.width + c] += dy;
    }
    if (!p.dx) continue;
    s = row_sum<true>(s, 32, box, turn);
    const float m0 = s.x * inverse, m1 = s.y * inverse;
    T* to = static_cast<T*>(p.dx) + offset(p.at_dx, row, p);
    for (uint32_t c = threadIdx.x; c < p.width; c += 1024) {
      const float hat = (float(from[c]) - mean - rest) * rstd, dy = float(grad[c]);
      const float dh = p.weight ? dy * float(static_cast<const W*>(p.weight)[c]) : dy;
      const float y[1] = {(dh - fmaf(hat, m1, m0)) * rstd};
      put(to + c, y);
    }
  }
}

// dw and db from the blocks' sums: 32 columns a block, its warps over the lines.
template <class W>
__global__ void __launch_bounds__(1024) norm_reduce_kernel(const float* partial, uint32_t lines, uint32_t width, W* dw, W* db) {
  __shared__ float part[32][33];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t c = blockIdx.x * 32 + lane;
  W* to = blockIdx.y ? db : dw;
  if (!to) return;
  float sum = 0.0f;
  if (c < width)
#pragma unroll 4
    for (uint32_t l = warp; l < lines; l += 32) sum += partial[(uint64_t(l) * 2 + blockIdx.y) * width + c];
  part[warp][lane] = sum;
  __syncthreads();
  sum = part[lane][warp];  // line `lane` of column `warp`
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(kAll, sum, d);
  const uint32_t column = blockIdx.x * 32 + warp;
  if (lane == 0 && column < width) {
    const float y[1] = {sum};
    put(to + column, y);
  }
}

// ---------------------------------------------------------------- which kernel
RowsAt rows_at(const ZenoTensor& t, const ZenoLayerNorm& p) {
  RowsAt a{};
  for (int i = 0; i < 3; ++i) a.stride[i] = t.stride[i];
  // axes of one row have no stride; the rest fold into one where each is the next one's span
  int64_t step = 0, span = 0;
  a.flat = true;
  for (int i = 2; i >= 0; --i) {
    if (p.rows[i] == 1) continue;
    if (span == 0) step = t.stride[i], span = t.stride[i] * int64_t(p.rows[i]);
    else if (t.stride[i] == span) span *= int64_t(p.rows[i]);
    else a.flat = false;
    if (span == 0) a.flat = false;  // stride 0
  }
  if (a.flat) a.stride[2] = step;
  return a;
}

// Up to 16 values a lane (backward holds four of each: x, dy and the two sums).  Short rows, a part of a warp each, are
// taken several at a time, so that enough loads are under way.
constexpr int kValues = 16;
constexpr int rows_at_once(int values, bool block, bool backward) {
  return block ? 1 : (values <= 8 ? 4 : 2) / (backward ? 2 : 1);
}

struct Choice {
  bool vec, block;
  int lanes;    // of a row (a power of two); threads where a block takes one
  int lanes_log;
  int vectors;  // of a lane, as one of the instances
  int values() const { return vec ? vectors * width : vectors; }
  int width;    // values of a vector
};

bool vec_ok(const void* data, const ZenoTensor& t, size_t item) {
  const int64_t n = int64_t(16 / item);
  return reinterpret_cast<uintptr_t>(data) % 16 == 0 && t.stride[0] % n == 0 && t.stride[1] % n == 0 && t.stride[2] % n == 0;
}

size_t item_of(uint32_t dtype) { return dtype == ZENO_DTYPE_BF16 ? 2 : 4; }

Choice choose(const ZenoLayerNorm& p, bool vec) {
  Choice c{};
  c.vec = vec;
  c.width = vec ? int(16 / item_of(p.dtype)) : 1;
  const uint32_t v = uint32_t(c.width), pieces = (p.width + v - 1) / v, most = kValues / v;
  if (pieces <= 32 * most) {
    c.lanes = 1;
    while (uint32_t(c.lanes) < pieces && c.lanes < 32) c.lanes *= 2;
    // scalars: two of a lane, so that a warp takes several short rows
    if (!vec && c.lanes > 4 && pieces <= uint32_t(c.lanes)) c.lanes /= 2;
    while (1 << c.lanes_log < c.lanes) ++c.lanes_log;
    const uint32_t n = (pieces + c.lanes - 1) / c.lanes;
    c.vectors = vec ? (n <= 1 ? 1 : n <= 2 ? 2 : 4) : (n <= 2 ? 2 : n <= 8 ? 8 : 16);
    return c;
  }
  c.block = true;
  c.lanes = int(std::max(((pieces + most - 1) / most + 31) / 32 * 32, 64u));
  c.vectors = int(most);
  return c;
}

template <class T, class W, int V, int N, bool BLOCK>
cudaError_t run(const Norm& p, const Choice& c, bool backward, unsigned blocks, cudaStream_t stream) {
  const int threads = BLOCK ? c.lanes : 256;
  if (!backward) {
    norm_forward_kernel<T, W, V, N, rows_at_once(V * N, BLOCK, false), BLOCK><<<blocks, threads, 0, stream>>>(p, c.lanes, c.lanes_log);
  } else {
    const size_t side = BLOCK || !p.partial ? 0 : size_t(256) * N * V * 4;
    norm_backward_kernel<T, W, V, N, rows_at_once(V * N, BLOCK, true), BLOCK><<<blocks, threads, side, stream>>>(p, c.lanes, c.lanes_log);
  }
  return cudaGetLastError();
}

template <class T, class W>
cudaError_t by_values(const Norm& p, const Choice& c, bool backward, unsigned blocks, cudaStream_t stream) {
  constexpr int V = 16 / int(sizeof(T));
  if (c.block) return c.vec ? run<T, W, V, kValues / V, true>(p, c, backward, blocks, stream) : run<T, W, 1, kValues, true>(p, c, backward, blocks, stream);
  if (c.vec) {
    if (c.vectors == 1) return run<T, W, V, 1, false>(p, c, backward, blocks, stream);
    if constexpr (V == 4)
      if (c.vectors == 2) return run<T, W, V, 2, false>(p, c, backward, blocks, stream);
    return run<T, W, V, kValues / V, false>(p, c, backward, blocks, stream);
  }
  if (c.vectors == 2) return run<T, W, 1, 2, false>(p, c, backward, blocks, stream);
  if (c.vectors == 8) return run<T, W, 1, 8, false>(p, c, backward, blocks, stream);
  return run<T, W, 1, 16, false>(p, c, backward, blocks, stream);
}

Norm norm_of(const ZenoLayerNorm& p) {
  Norm n{};
  n.x = p.x.data, n.weight = p.weight, n.bias = p.bias, n.y = p.out.data, n.saved = p.saved;
  n.at_x = rows_at(p.x, p), n.at_y = rows_at(p.out, p);
  n.rows = uint32_t(p.rows[0] * p.rows[1] * p.rows[2]);
  n.rows1 = uint32_t(std::max<uint64_t>(p.rows[1], 1)), n.rows2 = uint32_t(std::max<uint64_t>(p.rows[2], 1));
  n.width = p.width, n.eps = p.eps;
  return n;
}

bool affine_ok(const ZenoLayerNorm& p) {
  return ((reinterpret_cast<uintptr_t>(p.weight) | reinterpret_cast<uintptr_t>(p.bias)) & 15) == 0;
}

bool is_vec(const ZenoLayerNorm& p, const ZenoTensor& out) {
  const size_t item = item_of(p.dtype);
  return p.width % (16 / item) == 0 && vec_ok(p.x.data, p.x, item) && vec_ok(out.data, out, item) && affine_ok(p);
}

// Blocks of the backward pass: enough to fill the GPU, and no more lines of sums than the rows are worth.
unsigned backward_blocks(const ZenoLayerNorm& p, uint32_t rows, bool vec) {
  if (p.width > kWide) return unsigned(std::min<uint32_t>(rows, kSms));
  const Choice c = choose(p, vec);
  const uint64_t per = c.block ? 1 : uint64_t(256 / c.lanes) * rows_at_once(c.values(), c.block, true);
  const uint64_t threads = c.block ? uint64_t(c.lanes) : 256;
  return unsigned(std::min<uint64_t>((rows + per - 1) / per, uint64_t(kSms) * std::max<uint64_t>(1, 1024 / threads)));
}

template <class T, class W>
cudaError_t forward(const ZenoLayerNorm& p, cudaStream_t stream) {
  const Norm n = norm_of(p);
  if (p.width > kWide) {
    norm_wide_forward_kernel<T, W><<<std::min(n.rows, 2 * kSms), 1024, 0, stream>>>(n);
    return cudaGetLastError();
  }
  const bool vec = is_vec(p, p.out);
  const Choice c = choose(p, vec);
  const uint64_t per = c.block ? 1 : uint64_t(256 / c.lanes) * rows_at_once(c.values(), c.block, false);
  return by_values<T, W>(n, c, false, unsigned((n.rows + per - 1) / per), stream);
}

template <class T, class W>
cudaError_t backward(const ZenoLayerNorm& p, const ZenoLayerNormGrads& d, void* workspace, cudaStream_t stream) {
  Norm n = norm_of(p);
  n.dy = d.d_out.data, n.dx = d.d_x.data;
  n.at_dy = rows_at(d.d_out, p), n.at_dx = rows_at(d.d_x, p);
  n.partial = d.d_weight || d.d_bias ? static_cast<float*>(workspace) : nullptr;
  unsigned blocks = 0;
  if (n.rows && (n.dx || n.partial)) {
    const bool vec = is_vec(p, d.d_out) && (!n.dx || vec_ok(d.d_x.data, d.d_x, sizeof(T)));
    blocks = backward_blocks(p, n.rows, vec);
    cudaError_t e;
    if (p.width > kWide) {
      norm_wide_backward_kernel<T, W><<<blocks, 1024, 0, stream>>>(n);
      e = cudaGetLastError();
    } else {
      e = by_values<T, W>(n, choose(p, vec), true, blocks, stream);
    }
    if (e != cudaSuccess) return e;
  }
  if (!d.d_weight && !d.d_bias) return cudaSuccess;
  norm_reduce_kernel<W><<<dim3((p.width + 31) / 32, 2), 1024, 0, stream>>>(n.partial, blocks, p.width, static_cast<W*>(d.d_weight),
                                                                          static_cast<W*>(d.d_bias));
  return cudaGetLastError();
}

}  // namespace

uint64_t layer_norm_workspace(const ZenoLayerNorm& p) {
  const uint32_t rows = uint32_t(p.rows[0] * p.rows[1] * p.rows[2]);
  if (!rows) return 0;
  // alignment decides on the vectors only when the gradients are known: room for either
  const unsigned blocks = std::max(backward_blocks(p, rows, false), p.width % (16 / item_of(p.dtype)) == 0 ? backward_blocks(p, rows, true) : 0u);
  return uint64_t(blocks) * 2 * p.width * 4;
}

cudaError_t launch_layer_norm_forward(const ZenoLayerNorm& p, cudaStream_t stream) {
  if (p.dtype == ZENO_DTYPE_F32) return forward<float, float>(p, stream);
  return p.affine_dtype == ZENO_DTYPE_F32 ? forward<bf16, float>(p, stream) : forward<bf16, bf16>(p, stream);
}

cudaError_t launch_layer_norm_backward(const ZenoLayerNorm& p, const ZenoLayerNormGrads& d, void* workspace, cudaStream_t stream) {
  if (p.dtype == ZENO_DTYPE_F32) return backward<float, float>(p, d, workspace, stream);
  return p.affine_dtype == ZENO_DTYPE_F32 ? backward<bf16, float>(p, d, workspace, stream) : backward<bf16, bf16>(p, d, workspace, stream);
}

}  // namespace zb
