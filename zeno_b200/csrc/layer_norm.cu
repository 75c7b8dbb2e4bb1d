// Layer norm and its gradients.  With xhat = (x - mean) rstd and dh = dy w:
//   y = xhat w + b
//   dx = rstd (dh - mean(dh) - xhat mean(dh xhat)),  dw = sum over rows of dy xhat,  db = sum over rows of dy
// The time is the bytes of the rows: each is read once, held in registers, and written once.  A row of up to
// 512 values belongs to a part of a warp or a warp, a longer one to a block.  Backward, every thread keeps the
// sums of its own columns over the rows it sees; a block's sums go to the workspace and a second kernel adds them in a
// fixed order.  Sums are 32-bit (the last ones over blocks too), the variance is taken from the differences to the mean.
//
// Rows whose squares leave a float's range are taken again in units that they fit in, once a thread's rows are through: rows of spreads past 1e19 (or
// whose plain sum overflows) in units of 2^96, and differences below 2^-50, which count where eps is below 2^-100, times 2^96.  Powers of two round
// nothing.  In the loops over the rows this costs a comparison of each (branches there cost 3 to 8 %, the registers of the other side included).
//
// 131072 rows of 256 bfloat16: 29 us forward, 40 us backward (20 and 31 us of bytes), 4 us for the sums over blocks; 524288 rows of 64: 26.5 us (20 us).
// Nothing is full there: forward an SM issues in 65 % of its cycles, has 30 of 40 warps on average and is without work for 14 % of the time (start and
// end of one round of blocks); a warp waits for its row's loads and for two sums across lanes, one behind the other.
// 2047 rows of 4099 floats, whose rows are not aligned: 26 and 37 us, value by value.  2000 rows of 20000 floats, past what a block holds: 93 us
// forward, 410 us with gradients (24 and 73 us of bytes), value by value from L2 and with the block's sums in memory.
#include <cuda_bf16.h>

#include <algorithm>
#include <type_traits>

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
  float* saved;    // [3][rows]: the mean as summed, what that sum's rounding left of it, rstd; rstd negative: all three are of x in units of 2^96
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

// V neighbouring values (one 16-byte vector, or a single value) as they are in memory.
template <class T, int V>
struct Raw {
  using type = uint4;
};
template <class T>
struct Raw<T, 1> {
  using type = T;
};
template <class T, int V>
__device__ __forceinline__ typename Raw<T, V>::type fetch_raw(const T* at) {
  return *reinterpret_cast<const typename Raw<T, V>::type*>(at);
}
__device__ __forceinline__ void unpack(float (&x)[1], float w) { x[0] = w; }
__device__ __forceinline__ void unpack(float (&x)[1], bf16 w) { x[0] = __bfloat162float(w); }
__device__ __forceinline__ void unpack(float (&x)[4], const uint4& w) {
  x[0] = __uint_as_float(w.x), x[1] = __uint_as_float(w.y), x[2] = __uint_as_float(w.z), x[3] = __uint_as_float(w.w);
}
__device__ __forceinline__ void unpack(float (&x)[8], const uint4& w) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(u[i] << 16), x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
}
// V values of a weight, of its own type.
template <class W, int V>
__device__ __forceinline__ void fetch(float (&x)[V], const W* at) {
  if constexpr (V == 1) {
    unpack(x, *at);
  } else if constexpr (sizeof(W) == 2) {
    unpack(x, *reinterpret_cast<const uint4*>(at));
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

// 1 / sqrt(x): the approximation and one Newton step
__device__ __forceinline__ float inverse_sqrt(float x) {
  const float y = rsqrtf(x);
  return x < INFINITY ? fmaf(0.5f * y, fmaf(-x * y, y, 1.0f), y) : y;
}

constexpr float kUp = 79228162514264337593543950336.0f, kDown = 1.0f / kUp;  // 2^96
// x where it is above 0 or not a number
__device__ __forceinline__ float positive(float x) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(x), "f"(0.0f));
  return y;
}
// variance + eps, from the sums of the differences and of their squares and 1 / n; not a number where a difference is not finite.
// rest: what the sum's rounding left of the mean
__device__ __forceinline__ float spread(float2 sums, float inverse, float eps, float& rest) {
  rest = sums.x * inverse;
  return positive(fmaf(-rest, rest, sums.y * inverse)) + eps;
}
// Whether the squares kept 24 bits: above 2^-100.
__device__ __forceinline__ bool in_range(float v) { return v > 7.888609e-31f && v < INFINITY; }

// Sums over the LANES lanes of a row, or over a block.  A block's pass through `box` (taken in turns so that one barrier is enough).
template <int LANES, bool BLOCK>
__device__ __forceinline__ float row_sum(float s, float2 (*box)[32], int& turn) {
#pragma unroll
  for (int d = 1; d < LANES; d <<= 1) s += __shfl_xor_sync(kAll, s, d);
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
template <int LANES, bool BLOCK>
__device__ __forceinline__ float2 row_sum(float2 s, float2 (*box)[32], int& turn) {
#pragma unroll
  for (int d = 1; d < LANES; d <<= 1) {
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

// A row belongs to LANES lanes, or with BLOCK to all warps of a block, 32 N V neighbouring values to each.  A lane has N vectors of V
// values, LANES V apart.
template <class T_, class W_, int V_, int N_, int LANES_, bool BLOCK_>
struct Shape {
  using T = T_;
  using W = W_;
  static constexpr int V = V_, N = N_, LANES = LANES_, M = N * V / 2;  // M: pairs of values of a lane
  static constexpr bool BLOCK = BLOCK_;
  static constexpr int PER = BLOCK ? 1 : 256 / LANES;  // rows side by side in a block
  static constexpr bool AHEAD = N * V <= 8;
  // blocks that an SM has registers for, where the compiler would take a few more than leave place for them (0: as it likes)
  static constexpr int FORWARD_RESIDENT = V == 8 && N == 2 && !BLOCK ? 4 : 0, BACKWARD_RESIDENT = V == 8 && N == 1 ? 4 : 0;
  static constexpr int COLS = LANES * N * V;  // columns that there is room for (BLOCK: for each warp)
  int first;   // first column
  bool full;   // no column of this row (this warp) is past the width
  __device__ __forceinline__ explicit Shape(uint32_t width) {
    const int lane = BLOCK ? threadIdx.x & 31 : threadIdx.x & (LANES - 1), warp = BLOCK ? threadIdx.x >> 5 : 0;
    first = warp * COLS + lane * V;
    full = uint32_t((warp + 1) * COLS) <= width;
  }
  __device__ __forceinline__ int column(int i) const { return first + i * LANES * V; }
};

// One row value by value, in ordinary units and, where its squares leave the range there, in others; such a row is written.  All lanes of a warp
// come here, where a block has the row all of its threads.  columns(f): f of each column that is this thread's.
template <int LANES, bool BLOCK, class T, class W, class F>
__device__ __forceinline__ void norm_again(const Norm& p, uint32_t row, bool first_lane, float2 (*box)[32], F&& columns) {
  int turn = 0;  // (the sums are even in number)
  const bool here = row < p.rows;
  const T* from = static_cast<const T*>(p.x) + (here ? offset(p.at_x, row, p) : 0);
  const float inverse = 1.0f / float(p.width);
  float unit = 1.0f, times = 1.0f, mean, rest, v;  // x times `unit`, its differences times `times`
  auto difference = [&](uint32_t c) { return fmaf(float(from[c]), unit, -mean) * times; };
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    float sum = 0.0f;
    if (here) columns([&](uint32_t c) { sum = fmaf(float(from[c]), unit, sum); });
    mean = row_sum<LANES, BLOCK>(sum, box, turn) * inverse;
    float2 sums = make_float2(0.0f, 0.0f);
    if (here) columns([&](uint32_t c) {
      const float d = difference(c);
      sums.x += d, sums.y = fmaf(d, d, sums.y);
    });
    v = spread(row_sum<LANES, BLOCK>(sums, box, turn), inverse, p.eps * (unit * times) * (unit * times), rest);
    if (pass == 0 && !in_range(v)) (v < INFINITY ? times : unit) = v < INFINITY ? kUp : kDown;
  }
  if (!here || unit * times == 1.0f) return;
  const float rstd = inverse_sqrt(v);
  T* to = static_cast<T*>(p.y) + offset(p.at_y, row, p);
  columns([&](uint32_t c) {
    float y[1] = {(difference(c) - rest) * rstd};
    if (p.weight) y[0] *= float(static_cast<const W*>(p.weight)[c]);
    if (p.bias) y[0] += float(static_cast<const W*>(p.bias)[c]);
    put(to + c, y);
  });
  if (!p.saved || !first_lane) return;
  p.saved[row] = mean, p.saved[uint64_t(p.rows) + row] = times == 1.0f ? rest : rest * kDown;
  p.saved[2 * uint64_t(p.rows) + row] = unit == 1.0f ? fminf(rstd * times, 3.402823e38f) + (rstd - rstd) : -rstd;
}
// The rows of a thread.
template <class S>
__device__ __noinline__ void norm_forward_again(const Norm& p, float2 (*box)[32]) {
  const S at(p.width);
  for (uint64_t first = uint64_t(blockIdx.x) * S::PER; first < p.rows; first += uint64_t(gridDim.x) * S::PER)
    norm_again<S::LANES, S::BLOCK, typename S::T, typename S::W>(p, uint32_t(first) + (S::BLOCK ? 0 : threadIdx.x / S::LANES), at.first == 0, box, [&](auto&& f) {
#pragma unroll 1
      for (int i = 0; i < S::N * S::V; ++i) {
        const uint32_t c = uint32_t(at.column(i / S::V)) + i % S::V;
        if (c < p.width) f(c);
      }
    });
}

// Rows from blockIdx.x on in steps of the grid; the next one is on its way while one is worked on.  Where a lane has 16 values
// there are more blocks instead (of 4099 values: 25 us against 28).
template <class S>
__global__ void __launch_bounds__(S::BLOCK ? 512 : 256, S::FORWARD_RESIDENT) norm_forward_kernel(const __grid_constant__ Norm p) {
  using T = typename S::T;
  using W = typename S::W;
  constexpr int V = S::V, N = S::N, M = S::M;
  constexpr bool AHEAD = S::AHEAD, HELD = AHEAD;  // weight and bias stay in registers
  __shared__ float2 box[2][32];
  int turn = 0;
  const S at(p.width);
  const uint32_t own = S::BLOCK ? 0 : threadIdx.x / S::LANES;
  typename Raw<T, V>::type raw[N];
  auto fetch_row = [&](uint32_t row) {
    const bool here = row < p.rows;
    const T* from = static_cast<const T*>(p.x) + (here ? offset(p.at_x, row, p) : 0) + at.first;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      raw[i] = typename Raw<T, V>::type{};
      if (here && (at.full || uint32_t(at.column(i)) < p.width)) raw[i] = fetch_raw<T, V>(from + i * S::LANES * V);
    }
  };
  if (AHEAD) fetch_row(blockIdx.x * S::PER + own);
  float w[N][V], b[N][V];
  auto fetch_affine = [&](int i) {  // 1 and 0 where there is none
#pragma unroll
    for (int e = 0; e < V; ++e) w[i][e] = 1.0f, b[i][e] = 0.0f;
    if (!at.full && uint32_t(at.column(i)) >= p.width) return;
    if (p.weight) fetch(w[i], static_cast<const W*>(p.weight) + at.column(i));
    if (p.bias) fetch(b[i], static_cast<const W*>(p.bias) + at.column(i));
  };
  if (HELD) {
#pragma unroll
    for (int i = 0; i < N; ++i) fetch_affine(i);
  }
  const float inverse = 1.0f / float(p.width);
  bool again = false;  // (where a block has the rows, the same in all of its threads)
  for (uint64_t first = uint64_t(blockIdx.x) * S::PER; first < p.rows; first += uint64_t(gridDim.x) * S::PER) {
    const uint32_t row = uint32_t(first) + own;
    if (!AHEAD) fetch_row(row);
    Two y[M];
    {
      float x[N][V];
#pragma unroll
      for (int i = 0; i < N; ++i) unpack(x[i], raw[i]);
      const float* values = &x[0][0];
#pragma unroll
      for (int m = 0; m < M; ++m) y[m] = two(values[2 * m], values[2 * m + 1]);
    }
    const uint64_t ahead = first + uint64_t(gridDim.x) * S::PER;
    if (AHEAD && ahead < p.rows) fetch_row(uint32_t(ahead) + own);
    Two s = y[0];
#pragma unroll
    for (int m = 1; m < M; ++m) s = s + y[m];
    const float2 t = apart(s);
    const float mean = row_sum<S::LANES, S::BLOCK>(t.x + t.y, box, turn) * inverse;
    const Two minus = two(-mean, -mean);
#pragma unroll
    for (int m = 0; m < M; ++m) y[m] = y[m] + minus;
    if (!at.full) {  // what is not there stays zero
#pragma unroll
      for (int m = 0; m < M; ++m) {
        const float2 a = apart(y[m]);
        y[m] = two(uint32_t(at.column(2 * m / V)) < p.width ? a.x : 0.0f, uint32_t(at.column((2 * m + 1) / V)) < p.width ? a.y : 0.0f);
      }
    }
    s = y[0];
    Two q = y[0] * y[0];
#pragma unroll
    for (int m = 1; m < M; ++m) s = s + y[m], q = fma2(y[m], y[m], q);
    const float2 c = apart(s), d = apart(q);
    float rest;
    const float v = spread(row_sum<S::LANES, S::BLOCK>(make_float2(c.x + c.y, d.x + d.y), box, turn), inverse, p.eps, rest);
    const float rstd = inverse_sqrt(v);
    again |= !in_range(v);
    if (row >= p.rows) continue;
    const float less = -rest * rstd;
    const Two f = two(rstd, rstd), r = two(less, less);
    T* to = static_cast<T*>(p.y) + offset(p.at_y, row, p) + at.first;
    float z[N][V];
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (!HELD) fetch_affine(i);
#pragma unroll
    for (int m = 0; m < M; ++m) {
      const float *vw = &w[0][0] + 2 * m, *vb = &b[0][0] + 2 * m;
      const float2 a = apart(fma2(fma2(y[m], f, r), two(vw[0], vw[1]), two(vb[0], vb[1])));
      (&z[0][0])[2 * m] = a.x, (&z[0][0])[2 * m + 1] = a.y;
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (at.full || uint32_t(at.column(i)) < p.width) put(to + i * S::LANES * V, z[i]);
    if (p.saved && (S::BLOCK ? threadIdx.x : threadIdx.x & (S::LANES - 1)) == 0)
      p.saved[row] = mean, p.saved[uint64_t(p.rows) + row] = rest, p.saved[2 * uint64_t(p.rows) + row] = rstd;
  }
  if (S::BLOCK ? again : __any_sync(kAll, again)) norm_forward_again<S>(p, box);
}

// A row of x and dy, and what is known of it.
template <class S>
struct Fetched {
  typename Raw<typename S::T, S::V>::type x[S::N], g[S::N];
  float mean, rest, rstd;
  __device__ __forceinline__ void fetch(const Norm& p, const S& at, uint32_t row) {
    using T = typename S::T;
    const bool here = row < p.rows;
    const T* from = static_cast<const T*>(p.x) + (here ? offset(p.at_x, row, p) : 0) + at.first;
    const T* grad = static_cast<const T*>(p.dy) + (here ? offset(p.at_dy, row, p) : 0) + at.first;
#pragma unroll
    for (int i = 0; i < S::N; ++i) {
      x[i] = g[i] = typename Raw<T, S::V>::type{};
      if (here && (at.full || uint32_t(at.column(i)) < p.width)) {
        x[i] = fetch_raw<T, S::V>(from + i * S::LANES * S::V);
        g[i] = fetch_raw<T, S::V>(grad + i * S::LANES * S::V);
      }
    }
    mean = here ? p.saved[row] : 0.0f;
    rest = here ? p.saved[uint64_t(p.rows) + row] : 0.0f;
    rstd = here ? p.saved[2 * uint64_t(p.rows) + row] : 0.0f;
  }
};

// Rows from blockIdx.x on in steps of the grid; a thread's sums over its columns end in the block's line of the workspace.  The next row is
// on its way while one is worked on, where there are registers for it.
template <class S>
__device__ __forceinline__ void norm_backward(const Norm& p) {
  using T = typename S::T;
  using W = typename S::W;
  constexpr int V = S::V, N = S::N, M = S::M;
  constexpr bool AHEAD = S::AHEAD;
  __shared__ float2 box[2][32];
  extern __shared__ float side[];  // sums of the rows side by side
  int turn = 0;
  const S at(p.width);
  const uint32_t own = S::BLOCK ? 0 : threadIdx.x / S::LANES;
  const float inverse = 1.0f / float(p.width);
  early::let_next_start();
  Two dw[M], db[M];
#pragma unroll
  for (int m = 0; m < M; ++m) dw[m] = db[m] = two(0.0f, 0.0f);
  Fetched<S> next;
  if (AHEAD) next.fetch(p, at, blockIdx.x * S::PER + own);
  bool again = false;
  // A row; its sums over dy xhat are zero where x is in other units (`large`: the rows that are, and those sums alone).
  auto take = [&](auto large, const Fetched<S>& now, uint32_t row) {
    constexpr bool LARGE = decltype(large)::value;
    Two x[M], g[M];
    {
      float a[N][V], b[N][V];
#pragma unroll
      for (int i = 0; i < N; ++i) unpack(a[i], now.x[i]), unpack(b[i], now.g[i]);
      const float *va = &a[0][0], *vb = &b[0][0];
#pragma unroll
      for (int m = 0; m < M; ++m) x[m] = two(va[2 * m], va[2 * m + 1]), g[m] = two(vb[2 * m], vb[2 * m + 1]);
    }
    const bool other = now.rstd < 0.0f;
    const float rstd = LARGE ? -now.rstd : positive(now.rstd), less = -now.rest * rstd;
    const Two minus = two(-now.mean, -now.mean), r = two(less, less), f = two(rstd, rstd);
#pragma unroll
    for (int m = 0; m < M; ++m) {  // (what is not there has no gradient: it adds nothing)
      if (LARGE) x[m] = other ? x[m] * two(kDown, kDown) : two(0.0f, 0.0f);
      x[m] = fma2(x[m] + minus, f, r);
      if (!LARGE) dw[m] = fma2(g[m], x[m], dw[m]), db[m] = db[m] + g[m];
      else if (other) dw[m] = fma2(g[m], x[m], dw[m]);
    }
    if (!LARGE) again |= other;
    if (!p.dx) return;
    if (p.weight) {
      float w[N][V];
#pragma unroll
      for (int i = 0; i < N; ++i) {
#pragma unroll
        for (int e = 0; e < V; ++e) w[i][e] = 0.0f;
        if (at.full || uint32_t(at.column(i)) < p.width) fetch(w[i], static_cast<const W*>(p.weight) + at.column(i));
      }
      const float* values = &w[0][0];
#pragma unroll
      for (int m = 0; m < M; ++m) g[m] = g[m] * two(values[2 * m], values[2 * m + 1]);
    }
    Two s0 = g[0], s1 = g[0] * x[0];
#pragma unroll
    for (int m = 1; m < M; ++m) s0 = s0 + g[m], s1 = fma2(g[m], x[m], s1);
    const float2 a = apart(s0), b = apart(s1);
    const float2 t = row_sum<S::LANES, S::BLOCK>(make_float2(a.x + a.y, b.x + b.y), box, turn);
    if (row >= p.rows || (LARGE && !other)) return;
    const Two m0 = two(-t.x * inverse, -t.x * inverse), m1 = two(-t.y * inverse, -t.y * inverse);
    T* to = static_cast<T*>(p.dx) + offset(p.at_dx, row, p) + at.first;
    float z[N][V];
#pragma unroll
    for (int m = 0; m < M; ++m) {
      Two y = (g[m] + fma2(x[m], m1, m0)) * f;
      if (LARGE) y = y * two(kDown, kDown);
      const float2 c = apart(y);
      (&z[0][0])[2 * m] = c.x, (&z[0][0])[2 * m + 1] = c.y;
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (at.full || uint32_t(at.column(i)) < p.width) put(to + i * S::LANES * V, z[i]);
  };
  for (uint64_t first = uint64_t(blockIdx.x) * S::PER; first < p.rows; first += uint64_t(gridDim.x) * S::PER) {
    const uint32_t row = uint32_t(first) + own;
    if (!AHEAD) next.fetch(p, at, row);
    Fetched<S> now = next;
    const uint64_t ahead = first + uint64_t(gridDim.x) * S::PER;
    if (AHEAD && ahead < p.rows) next.fetch(p, at, uint32_t(ahead) + own);
    take(std::false_type{}, now, row);
  }
  if (S::BLOCK ? again : __any_sync(kAll, again)) {
#pragma unroll 1
    for (uint64_t first = uint64_t(blockIdx.x) * S::PER; first < p.rows; first += uint64_t(gridDim.x) * S::PER) {
      next.fetch(p, at, uint32_t(first) + own);
      take(std::true_type{}, next, uint32_t(first) + own);
    }
  }
  if (!p.partial) return;
  float* line = p.partial + uint64_t(blockIdx.x) * 2 * p.width;
#pragma unroll
  for (int pass = 0; pass < 2; ++pass) {
    if (!S::BLOCK) __syncthreads();
#pragma unroll
    for (int m = 0; m < M; ++m) {
      const float2 a = apart(pass ? db[m] : dw[m]);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t c = uint32_t(at.column((2 * m + h) / V)) + (2 * m + h) % V;
        if (!S::BLOCK) side[own * S::COLS + c] = h ? a.y : a.x;
        else if (c < p.width) line[pass * p.width + c] = h ? a.y : a.x;
      }
    }
    if (S::BLOCK) continue;
    __syncthreads();
    for (uint32_t c = threadIdx.x; c < p.width; c += 256) {
      float sum = 0.0f;
      for (int r = 0; r < S::PER; ++r) sum += side[r * S::COLS + c];
      line[pass * p.width + c] = sum;
    }
  }
}
template <class S>
__global__ void __launch_bounds__(256, S::BACKWARD_RESIDENT) norm_backward_kernel(const __grid_constant__ Norm p) {
  norm_backward<S>(p);
}
// (104 registers, so that rows of 4096 values are two to an SM)
template <class S>
__global__ void __maxnreg__(104) norm_backward_block_kernel(const __grid_constant__ Norm p) {
  norm_backward<S>(p);
}

// Rows too long for registers: one block a row, which is read three times forward (from L2 after the first).
template <class T, class W>
__device__ __noinline__ void norm_wide_forward_again(const Norm& p, float2 (*box)[32]) {
  for (uint32_t row = blockIdx.x; row < p.rows; row += gridDim.x)
    norm_again<32, true, T, W>(p, row, threadIdx.x == 0, box, [&](auto&& f) {
      for (uint32_t c = threadIdx.x; c < p.width; c += 1024) f(c);
    });
}
template <class T, class W>
__global__ void __launch_bounds__(1024) norm_wide_forward_kernel(const __grid_constant__ Norm p) {
  __shared__ float2 box[2][32];
  int turn = 0;
  const float inverse = 1.0f / float(p.width);
  bool again = false;
  for (uint32_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* from = static_cast<const T*>(p.x) + offset(p.at_x, row, p);
    T* to = static_cast<T*>(p.y) + offset(p.at_y, row, p);
    float2 s = make_float2(0.0f, 0.0f);
    for (uint32_t c = threadIdx.x; c < p.width; c += 1024) s.x += float(from[c]);
    const float mean = row_sum<32, true>(s.x, box, turn) * inverse;
    s = make_float2(0.0f, 0.0f);
    for (uint32_t c = threadIdx.x; c < p.width; c += 1024) {
      const float d = float(from[c]) - mean;
      s.x += d, s.y = fmaf(d, d, s.y);
    }
    float rest;
    const float v = spread(row_sum<32, true>(s, box, turn), inverse, p.eps, rest), rstd = inverse_sqrt(v);
    again |= !in_range(v);
    for (uint32_t c = threadIdx.x; c < p.width; c += 1024) {
      float y[1] = {(float(from[c]) - mean - rest) * rstd};
      if (p.weight) y[0] *= float(static_cast<const W*>(p.weight)[c]);
      if (p.bias) y[0] += float(static_cast<const W*>(p.bias)[c]);
      put(to + c, y);
    }
    if (p.saved && threadIdx.x == 0) p.saved[row] = mean, p.saved[uint64_t(p.rows) + row] = rest, p.saved[2 * uint64_t(p.rows) + row] = rstd;
  }
  if (again) norm_wide_forward_again<T, W>(p, box);
}
// LARGE: the rows in other units (whose dy have been summed) alone; whether there are such.
template <bool LARGE, class T, class W>
__device__ __forceinline__ bool norm_wide_rows(const Norm& p, float2 (*box)[32], int& turn) {
  const float inverse = 1.0f / float(p.width);
  float* line = p.partial ? p.partial + uint64_t(blockIdx.x) * 2 * p.width : nullptr;
  bool again = false;
  for (uint32_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* from = static_cast<const T*>(p.x) + offset(p.at_x, row, p);
    const T* grad = static_cast<const T*>(p.dy) + offset(p.at_dy, row, p);
    const float mean = p.saved[row], rest = p.saved[uint64_t(p.rows) + row], kept = p.saved[2 * uint64_t(p.rows) + row];
    const float rstd = LARGE ? -kept : positive(kept);
    again |= kept < 0.0f;
    if (LARGE && !(kept < 0.0f)) continue;
    auto hat_of = [&](uint32_t c) { return ((LARGE ? float(from[c]) * kDown : float(from[c])) - mean - rest) * rstd; };
    float2 s = make_float2(0.0f, 0.0f);
    for (uint32_t c = threadIdx.x; c < p.width; c += 1024) {  // a thread comes back to its own columns of the line
      const float hat = hat_of(c), dy = float(grad[c]);
      const float dh = p.weight ? dy * float(static_cast<const W*>(p.weight)[c]) : dy;
      s.x += dh, s.y = fmaf(dh, hat, s.y);
      if (line) line[c] = fmaf(dy, hat, line[c]);
      if (line && !LARGE) line[p.width + c] += dy;
    }
    if (!p.dx) continue;
    s = row_sum<32, true>(s, box, turn);
    const float m0 = s.x * inverse, m1 = s.y * inverse;
    T* to = static_cast<T*>(p.dx) + offset(p.at_dx, row, p);
    for (uint32_t c = threadIdx.x; c < p.width; c += 1024) {
      const float hat = hat_of(c), dy = float(grad[c]);
      const float dh = p.weight ? dy * float(static_cast<const W*>(p.weight)[c]) : dy;
      float y[1] = {(dh - fmaf(hat, m1, m0)) * rstd};
      if (LARGE) y[0] *= kDown;
      put(to + c, y);
    }
  }
  return again;
}
template <class T, class W>
__device__ __noinline__ void norm_wide_backward_again(const Norm& p, float2 (*box)[32], int turn) {
  norm_wide_rows<true, T, W>(p, box, turn);
}
template <class T, class W>
__global__ void __launch_bounds__(1024) norm_wide_backward_kernel(const __grid_constant__ Norm p) {
  __shared__ float2 box[2][32];
  int turn = 0;
  if (p.partial) {
    float* line = p.partial + uint64_t(blockIdx.x) * 2 * p.width;
    for (uint32_t c = threadIdx.x; c < p.width; c += 1024) line[c] = 0.0f, line[p.width + c] = 0.0f;
  }
  if (norm_wide_rows<false, T, W>(p, box, turn)) norm_wide_backward_again<T, W>(p, box, turn);
}

// dw and db from the blocks' sums: 32 columns a block, its warps over the lines.
template <class W>
__global__ void __launch_bounds__(1024) norm_reduce_kernel(const float* partial, uint32_t lines, uint32_t width, W* dw, W* db) {
  __shared__ float part[32][33];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t c = blockIdx.x * 32 + lane;
  W* to = blockIdx.y ? db : dw;
  early::wait_for_previous();
  if (!to) return;
  float sum = 0.0f;
  if (c < width)
#pragma unroll 8
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

// Up to 16 values a lane (backward holds x, dy and the two sums of each).
constexpr int kValues = 16;

struct Choice {
  bool vec, block;
  int lanes;    // of a row (a power of two); threads where a block takes one
  int vectors;  // of a lane, as one of the instances
  int width;    // values of a vector
  int values() const { return vectors * width; }
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
    // lanes of one vector, or of two values, each; longer rows take a warp
    const uint32_t least = vec ? 1 : 2;
    c.lanes = vec ? 1 : 4;
    while (uint32_t(c.lanes) * least < pieces && c.lanes < 32) c.lanes *= 2;
    const uint32_t n = (pieces + c.lanes - 1) / c.lanes;
    c.vectors = vec ? (n <= 1 ? 1 : n <= 2 ? 2 : 4) : (n <= 2 ? 2 : n <= 8 ? 8 : 16);
    return c;
  }
  c.block = true;
  c.lanes = int((pieces + 32 * most - 1) / (32 * most) * 32);
  c.vectors = int(most);
  return c;
}

template <class S>
cudaError_t run(const Norm& p, const Choice& c, bool backward, unsigned blocks, cudaStream_t stream) {
  const int threads = S::BLOCK ? c.lanes : 256;
  if (!backward) {
    norm_forward_kernel<S><<<blocks, threads, 0, stream>>>(p);
  } else if constexpr (S::BLOCK) {
    norm_backward_block_kernel<S><<<blocks, threads, 0, stream>>>(p);
  } else {
    norm_backward_kernel<S><<<blocks, threads, p.partial ? size_t(256) * S::N * S::V * 4 : 0, stream>>>(p);
  }
  return cudaGetLastError();
}

template <class T, class W>
cudaError_t by_values(const Norm& p, const Choice& c, bool backward, unsigned blocks, cudaStream_t stream) {
  constexpr int V = 16 / int(sizeof(T)), MOST = kValues / V;
  if (c.block)
    return c.vec ? run<Shape<T, W, V, MOST, 32, true>>(p, c, backward, blocks, stream) : run<Shape<T, W, 1, kValues, 32, true>>(p, c, backward, blocks, stream);
  if (c.vec) {
    if (c.vectors == 1) switch (c.lanes) {
        case 1: return run<Shape<T, W, V, 1, 1, false>>(p, c, backward, blocks, stream);
        case 2: return run<Shape<T, W, V, 1, 2, false>>(p, c, backward, blocks, stream);
        case 4: return run<Shape<T, W, V, 1, 4, false>>(p, c, backward, blocks, stream);
        case 8: return run<Shape<T, W, V, 1, 8, false>>(p, c, backward, blocks, stream);
        case 16: return run<Shape<T, W, V, 1, 16, false>>(p, c, backward, blocks, stream);
        default: return run<Shape<T, W, V, 1, 32, false>>(p, c, backward, blocks, stream);
      }
    if constexpr (V == 4)
      if (c.vectors == 2) return run<Shape<T, W, V, 2, 32, false>>(p, c, backward, blocks, stream);
    return run<Shape<T, W, V, MOST, 32, false>>(p, c, backward, blocks, stream);
  }
  if (c.vectors == 2) switch (c.lanes) {
      case 4: return run<Shape<T, W, 1, 2, 4, false>>(p, c, backward, blocks, stream);
      case 8: return run<Shape<T, W, 1, 2, 8, false>>(p, c, backward, blocks, stream);
      case 16: return run<Shape<T, W, 1, 2, 16, false>>(p, c, backward, blocks, stream);
      default: return run<Shape<T, W, 1, 2, 32, false>>(p, c, backward, blocks, stream);
    }
  if (c.vectors == 8) return run<Shape<T, W, 1, 8, 32, false>>(p, c, backward, blocks, stream);
  return run<Shape<T, W, 1, 16, 32, false>>(p, c, backward, blocks, stream);
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

// Blocks that share the rows: enough to fill the GPU, and backward no more lines of sums than that.
unsigned blocks_of(const ZenoLayerNorm& p, uint32_t rows, bool vec, uint32_t threads_of_sm) {
  if (p.width > kWide) return unsigned(std::min<uint32_t>(rows, kSms));
  const Choice c = choose(p, vec);
  const uint32_t per = c.block ? 1 : 256 / c.lanes, threads = c.block ? c.lanes : 256;
  return unsigned(std::min<uint64_t>((uint64_t(rows) + per - 1) / per, uint64_t(kSms) * std::max<uint32_t>(1, threads_of_sm / threads)));
}
unsigned backward_blocks(const ZenoLayerNorm& p, uint32_t rows, bool vec) { return blocks_of(p, rows, vec, 1024); }

template <class T, class W>
cudaError_t forward(const ZenoLayerNorm& p, cudaStream_t stream) {
  const Norm n = norm_of(p);
  if (p.width > kWide) {
    norm_wide_forward_kernel<T, W><<<std::min(n.rows, 2 * kSms), 1024, 0, stream>>>(n);
    return cudaGetLastError();
  }
  const bool vec = is_vec(p, p.out);
  return by_values<T, W>(n, choose(p, vec), false, blocks_of(p, n.rows, vec, choose(p, vec).values() <= 8 ? 1280 : UINT32_MAX), stream);
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
  return launch_early(norm_reduce_kernel<W>, dim3((p.width + 31) / 32, 2), 1024, 0, stream, static_cast<const float*>(n.partial), uint32_t(blocks), p.width,
                      static_cast<W*>(d.d_weight), static_cast<W*>(d.d_bias));
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
