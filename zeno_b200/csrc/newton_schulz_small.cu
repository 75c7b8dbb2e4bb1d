// Newton-Schulz orthogonalisation of matrices of at most 64 rows (or columns) by 4096: a cluster
// of blocks has one matrix in shared memory from the norm to the last step, each block a share of
// its columns.
//
// The same products as newton_schulz.cu, operands always in two f16 limbs, on mma.sync: at these
// sizes a step's three products are a few hundred instructions a warp and the time is their
// latency and the blocks' barriers, which launches of a tiled product would multiply (and whose one
// tile would walk over all columns by itself).  A = X X^T is a sum over the blocks, read from
// one another's shared memory; A A and B are the same in all of them; B X needs a block's own columns.
#include <cooperative_groups.h>

#include <algorithm>

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

// 16 warps (with 8: 64 x 256 in 52 us against 43, 200 of them in 146 against 123); a block has `per`
// tiles of 16 columns, 32 at most: a warp holds 8 tiles of 16 x 16 in its registers.
constexpr int WARPS = 16;
template <class T>
__global__ void __launch_bounds__(WARPS * 32)
small_kernel(const T* from, Matrix s, T* out, uint32_t steps, bool transposed, int per) {
  extern __shared__ __align__(16) unsigned char raw[];
  __shared__ double sums[WARPS], total;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gi = lane >> 2, qj = (lane & 3) * 2;
  const auto cluster = cooperative_groups::this_cluster();
  const int ranks = int(cluster.num_blocks()), rank = int(cluster.block_rank());
  const uint32_t matrix = blockIdx.x / ranks;
  const int j0 = rank * per * 16;  // the block's first column
  const int m = int(s.m), n = max(0, min(int(s.n) - j0, per * 16));
  const int mt = (m + 15) / 16, nt = (n + 15) / 16, pitch = per * 16 + 8;
  __half* x = reinterpret_cast<__half*>(raw);
  const int xs = mt * 16 * pitch, as = mt * 16 * kPitch;  // a plane
  __half* a = x + 2 * xs;
  __half* b = a + 2 * as;
  float* part = reinterpret_cast<float*>(b);  // this block's part of A, before B is made
  const T* at = from + int64_t(matrix) * s.matrix + j0 * s.col;
  out += int64_t(matrix) * m * s.n + (transposed ? int64_t(j0) * m : j0);
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
  if (ranks > 1) {
    if (tid == 0) total = sum;
    cluster.sync();
    sum = 0.0;
    for (int r = 0; r < ranks; ++r) sum += *cluster.map_shared_rank(&total, r);
    cluster.sync();
  }
  const double norm = sqrt(sum), inverse = 1.0 / (norm + kEps);
  if (steps == 0) {
    for (int e = tid; e < m * n; e += WARPS * 32) {
      const int i = transposed ? e % m : e / n, j = transposed ? e / m : e % n;
      const float y = float(inverse * up(at[i * s.row + j * s.col]));
      T* to = out + (transposed ? int64_t(j) * m + i : int64_t(i) * s.n + j);
      if constexpr (sizeof(T) == 2) *to = __float2bfloat16_rn(y);
      else *to = y;
    }
    return;
  }
  const int first = first_extra(norm);
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
      if (ranks > 1) {
#pragma unroll
        for (int h = 0; h < 8; ++h)
          part[(r + gi + ((h >> 1) & 1) * 8) * kSmallRows + c + (h >> 2) * 8 + qj + (h & 1)] = acc[h >> 2][h & 3];
        continue;
      }
#pragma unroll
      for (int h = 0; h < 4; ++h)
        store_split(a, a + as, (r + gi + (h & 1) * 8) * kPitch + c + (h >> 1) * 8 + qj, acc[h >> 1][(h & 1) * 2] * kUnscale,
                    acc[h >> 1][(h & 1) * 2 + 1] * kUnscale);
    }
    if (ranks > 1) {
      cluster.sync();
      for (int e = tid; e < mt * 16 * mt * 8; e += WARPS * 32) {
        const int i = e / (mt * 8), j = e % (mt * 8) * 2;
        float2 y = make_float2(0.0f, 0.0f);
#pragma unroll 4
        for (int q = 0; q < ranks; ++q) {
          const float2 z = *reinterpret_cast<const float2*>(cluster.map_shared_rank(part, q) + i * kSmallRows + j);
          y.x += z.x, y.y += z.y;
        }
        store_split(a, a + as, i * kPitch + j, y.x * kUnscale, y.y * kUnscale);
      }
      cluster.sync();  // all have read: B may take the parts' place
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
                T* to = out + (transposed ? int64_t(j + q) * m + i : int64_t(i) * s.n + j + q);
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

template <class T>
cudaError_t launch(const void* update, const Matrix& s, bool transposed, void* out, uint32_t steps, int ranks, int per, cudaStream_t stream) {
  const int mp = int(s.m + 15) / 16 * 16;
  // A and B always have room for 64 rows: the parts of A are kept in B's place
  const int smem = 4 * mp * (per * 16 + 8) + 2 * 4 * int(kSmallRows) * kPitch;
  const auto kernel = small_kernel<T>;
  static std::atomic<uint64_t> allowed{0};
  const cudaError_t e = allow_smem(kernel, 4 * int(kSmallRows) * (32 * WARPS + 8 + 2 * kPitch), allowed);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t c{};
  c.gridDim = dim3(s.count * ranks), c.blockDim = dim3(WARPS * 32), c.dynamicSmemBytes = size_t(smem), c.stream = stream;
  cudaLaunchAttribute a{};
  a.id = cudaLaunchAttributeClusterDimension;
  a.val.clusterDim.x = unsigned(ranks), a.val.clusterDim.y = 1, a.val.clusterDim.z = 1;
  c.attrs = &a, c.numAttrs = 1;
  return cudaLaunchKernelEx(&c, kernel, static_cast<const T*>(update), s, static_cast<T*>(out), steps, transposed, per);
}

template <class T>
cudaError_t by_width(const void* update, const Matrix& s, bool transposed, void* out, uint32_t steps, cudaStream_t stream) {
  // 64 columns a block while all blocks run at once (64 x 256, 8 warps: 52 us against 73 in one block), else 256
  // (200 of them: 146 us against 358); past 2048 columns up to 512.
  const int tiles = int(s.n + 15) / 16, fine = std::min((tiles + 3) / 4, 8), coarse = std::min((tiles + 15) / 16, 8);
  const int ranks = uint64_t(s.count) * fine <= kSms ? fine : coarse, per = (tiles + ranks - 1) / ranks;
  return launch<T>(update, s, transposed, out, steps, ranks, per, stream);
}

}  // namespace

cudaError_t launch_small(const void* update, const Matrix& s, bool transposed, void* out, uint32_t dtype, uint32_t steps,
                         cudaStream_t stream) {
  return dtype == ZENO_DTYPE_BF16 ? by_width<__nv_bfloat16>(update, s, transposed, out, steps, stream)
                                  : by_width<float>(update, s, transposed, out, steps, stream);
}

}  // namespace ns
}  // namespace zb
