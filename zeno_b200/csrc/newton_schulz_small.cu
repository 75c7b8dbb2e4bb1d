// Newton-Schulz orthogonalisation of small matrices (64 x 512 at most): one block has one
// matrix in shared memory from the norm to the last step.
//
// The same products as newton_schulz.cu, operands always in two f16 limbs, on mma.sync: at these
// sizes a step's three products are a few hundred instructions a warp and the time is their
// latency and the block's barriers, which launches of a tiled product would multiply.
#include "delta_mma.cuh"
#include "newton_schulz.h"

namespace zb {
namespace ns {
namespace {

using delta::a_rows;
using delta::b_cols;
using delta::b_rows;
using delta::mma;
using delta::store_split;

constexpr int kPitch = kSmallRows + 8;

// The matrix instructions' sums drop what is below 2^-24 of the running sum, always towards zero:
// hi hi goes to the 32-bit sum by an addition that rounds, the small products to a sum of their own.
__device__ __forceinline__ void products(float (&acc)[2][4], float (&low)[2][4], const uint32_t (&ah)[4], const uint32_t (&al)[4],
                                         const uint32_t (&bh)[4], const uint32_t (&bl)[4]) {
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    float t[4] = {};
    mma(t, ah, bh[2 * n], bh[2 * n + 1]);
    mma(low[n], al, bh[2 * n], bh[2 * n + 1]);
    mma(low[n], ah, bl[2 * n], bl[2 * n + 1]);
#pragma unroll
    for (int x = 0; x < 4; ++x) acc[n][x] += t[x];
  }
}
__device__ __forceinline__ void join(float (&acc)[2][4], const float (&low)[2][4]) {
#pragma unroll
  for (int x = 0; x < 8; ++x) acc[x >> 2][x & 3] += low[x >> 2][x & 3];
}

// WARPS warps; np <= 32 WARPS columns.
template <int WARPS, class T>
__global__ void __launch_bounds__(WARPS * 32)
small_kernel(const T* from, Matrix s, T* out, uint32_t steps, bool transposed) {
  extern __shared__ __align__(16) unsigned char raw[];
  __shared__ double sums[WARPS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gi = lane >> 2, qj = (lane & 3) * 2;
  const int m = int(s.m), n = int(s.n), mt = (m + 15) / 16, nt = (n + 15) / 16, pitch = nt * 16 + 8;
  __half* x = reinterpret_cast<__half*>(raw);
  const int xs = mt * 16 * pitch, as = mt * 16 * kPitch;  // a plane
  __half* a = x + 2 * xs;
  __half* b = a + 2 * as;
  const T* at = from + int64_t(blockIdx.x) * s.matrix;
  out += int64_t(blockIdx.x) * m * n;
  const bool by_row = s.col <= s.row;

  double sum = 0.0;
  for (int e = tid; e < m * n; e += WARPS * 32) {
    const int i = by_row ? e / n : e % m, j = by_row ? e % n : e / m;
    const double y = up(at[i * s.row + j * s.col]);
    sum = fma(y, y, sum);
  }
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  if (lane == 0) sums[warp] = sum;
  __syncthreads();
  sum = 0.0;
  for (int w = 0; w < WARPS; ++w) sum += sums[w];
  const double inverse = 1.0 / (sqrt(sum) + kEps);
  if (steps == 0) {
    for (int e = tid; e < m * n; e += WARPS * 32) {
      const int i = transposed ? e % m : e / n, j = transposed ? e / m : e % n;
      const float y = float(inverse * up(at[i * s.row + j * s.col]));
      if constexpr (sizeof(T) == 2) out[e] = __float2bfloat16_rn(y);
      else out[e] = y;
    }
    return;
  }
  const int first = first_extra(inverse);
  const double f = inverse * scalbn(double(kScale), first);
  for (int e = tid; e < mt * nt * 256; e += WARPS * 32) {
    const int i = by_row ? e / (nt * 16) : e % (mt * 16), j = by_row ? e % (nt * 16) : e / (mt * 16);
    const float y = i < m && j < n ? float(f * up(at[i * s.row + j * s.col])) : 0.0f;
    const __half hi = __float2half_rn(y);
    x[i * pitch + j] = hi;
    x[xs + i * pitch + j] = __float2half_rn(y - __half2float(hi));
  }
  __syncthreads();

  for (uint32_t step = 0; step < steps; ++step) {
    const int now = extra_at(first, step), next = extra_at(first, step + 1);
    // A = X X^T
    for (int t = warp; t < mt * mt; t += WARPS) {
      const int r = t / mt * 16, c = t % mt * 16;
      float acc[2][4] = {}, low[2][4] = {};
#pragma unroll 2
      for (int k = 0; k < nt * 16; k += 16) {
        uint32_t ah[4], al[4], bh[4], bl[4];
        a_rows(ah, x + r * pitch + k, pitch, lane), a_rows(al, x + xs + r * pitch + k, pitch, lane);
        b_rows(bh, x + c * pitch + k, pitch, lane), b_rows(bl, x + xs + c * pitch + k, pitch, lane);
        products(acc, low, ah, al, bh, bl);
      }
      join(acc, low);
#pragma unroll
      for (int h = 0; h < 4; ++h)
        store_split(a, a + as, (r + gi + (h & 1) * 8) * kPitch + c + (h >> 1) * 8 + qj, acc[h >> 1][(h & 1) * 2] * kUnscale,
                    acc[h >> 1][(h & 1) * 2 + 1] * kUnscale);
    }
    __syncthreads();
    // B = b A + c A A
    const float fb = kC * exp2f(float(-12 - 2 * now));
    for (int t = warp; t < mt * mt; t += WARPS) {
      const int r = t / mt * 16, c = t % mt * 16;
      float acc[2][4] = {}, low[2][4] = {};
      for (int k = 0; k < mt * 16; k += 16) {
        uint32_t ah[4], al[4], bh[4], bl[4];
        a_rows(ah, a + r * kPitch + k, kPitch, lane), a_rows(al, a + as + r * kPitch + k, kPitch, lane);
        b_rows(bh, a + c * kPitch + k, kPitch, lane), b_rows(bl, a + as + c * kPitch + k, kPitch, lane);
        products(acc, low, ah, al, bh, bl);
      }
      join(acc, low);
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const int to = (r + gi + (h & 1) * 8) * kPitch + c + (h >> 1) * 8 + qj;
        const float2 y = __half22float2(*reinterpret_cast<const __half2*>(a + to)), z = __half22float2(*reinterpret_cast<const __half2*>(a + as + to));
        store_split(b, b + as, to, fmaf(fb, acc[h >> 1][(h & 1) * 2], kB * (y.x + z.x)), fmaf(fb, acc[h >> 1][(h & 1) * 2 + 1], kB * (y.y + z.y)));
      }
    }
    __syncthreads();
    // X <- a X + B X: all of it is read before any of it is written
    const bool last = step + 1 == steps;
    const float fx = exp2f(float(last ? -24 - 3 * now : -12 - 3 * now + next)), fa = kA * exp2f(float(last ? -12 - now : next - now));
    float acc[8][2][4];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int t = warp + u * WARPS;
      if (t < mt * nt) {
        const int r = t % mt * 16, c = t / mt * 16;
        float low[2][4] = {};
#pragma unroll
        for (int h = 0; h < 8; ++h) acc[u][h >> 2][h & 3] = 0.0f;
        for (int k = 0; k < mt * 16; k += 16) {
          uint32_t ah[4], al[4], bh[4], bl[4];
          a_rows(ah, b + r * kPitch + k, kPitch, lane), a_rows(al, b + as + r * kPitch + k, kPitch, lane);
          b_cols(bh, x + k * pitch + c, pitch, lane), b_cols(bl, x + xs + k * pitch + c, pitch, lane);
          products(acc[u], low, ah, al, bh, bl);
        }
        join(acc[u], low);
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const int to = (r + gi + (h & 1) * 8) * pitch + c + (h >> 1) * 8 + qj;
          const float2 y = __half22float2(*reinterpret_cast<const __half2*>(x + to)), z = __half22float2(*reinterpret_cast<const __half2*>(x + xs + to));
          float* v = &acc[u][h >> 1][(h & 1) * 2];
          v[0] = fmaf(fx, v[0], fa * (y.x + z.x)), v[1] = fmaf(fx, v[1], fa * (y.y + z.y));
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int t = warp + u * WARPS;
      if (t < mt * nt) {
        const int r = t % mt * 16, c = t / mt * 16;
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const int i = r + gi + (h & 1) * 8, j = c + (h >> 1) * 8 + qj;
          const float* v = &acc[u][h >> 1][(h & 1) * 2];
          if (!last) {
            store_split(x, x + xs, i * pitch + j, v[0], v[1]);
          } else {
#pragma unroll
            for (int q = 0; q < 2; ++q)
              if (i < m && j + q < n) {
                T* to = out + (transposed ? int64_t(j + q) * m + i : int64_t(i) * n + j + q);
                if constexpr (sizeof(T) == 2) *to = __float2bfloat16_rn(v[q]);
                else *to = v[q];
              }
          }
        }
      }
    }
    __syncthreads();
  }
}

template <int WARPS, class T>
cudaError_t launch(const void* update, const Matrix& s, bool transposed, void* out, uint32_t steps, cudaStream_t stream) {
  const int mp = int(s.m + 15) / 16 * 16, np = int(s.n + 15) / 16 * 16;
  const int smem = 4 * mp * (np + 8 + 2 * kPitch);
  const auto kernel = small_kernel<WARPS, T>;
  static std::atomic<uint64_t> allowed{0};
  const cudaError_t e = allow_smem(kernel, 4 * int(kSmallRows) * int(kSmallCols + 8 + 2 * kPitch), allowed);
  if (e != cudaSuccess) return e;
  kernel<<<s.count, WARPS * 32, smem, stream>>>(static_cast<const T*>(update), s, static_cast<T*>(out), steps, transposed);
  return cudaGetLastError();
}

template <class T>
cudaError_t by_width(const void* update, const Matrix& s, bool transposed, void* out, uint32_t steps, cudaStream_t stream) {
  // 8 tiles of 16 x 16 a warp are held in the registers
  if (s.n <= 256) return launch<8, T>(update, s, transposed, out, steps, stream);
  return launch<16, T>(update, s, transposed, out, steps, stream);
}

}  // namespace

cudaError_t launch_small(const void* update, const Matrix& s, bool transposed, void* out, uint32_t dtype, uint32_t steps,
                         cudaStream_t stream) {
  return dtype == ZENO_DTYPE_BF16 ? by_width<__nv_bfloat16>(update, s, transposed, out, steps, stream)
                                  : by_width<float>(update, s, transposed, out, steps, stream);
}

}  // namespace ns
}  // namespace zb
