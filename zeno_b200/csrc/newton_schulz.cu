// Newton-Schulz orthogonalisation of update matrices.
//
//   X = M / (|M|_F + 1e-7) (transposed so that it is wide, m <= n), then `steps` times
//   A = X X^T,  B = b A + c A A,  X <- a X + B X
//
// Each singular value s of X goes through the odd polynomial a s + b s^3 + c s^5, which takes
// (0, 1] towards 1 and never leaves [0, 1.21]; so no entry of X, A or B exceeds 1.21, 1.47 or 2.81.
//
// The three products of a step are tcgen05 matrix instructions on f16 operands scaled by
// 2^12 (the bounds above keep them in range), with 32-bit accumulators in TMEM.  A matrix
// much smaller than 1e-7 keeps |X| << 1 for many steps; its X carries 2^E more, with E falling
// by 2 a step (a < 4), A and B carry 2^2E.
//
// Precision.  X is kept in two limbs, hi and lo, 22 bits together.  float32 updates: all
// operands are, and a product is hi hi + hi lo + lo hi.  bfloat16 updates of more than 128 rows:
// the products of all steps but the last take the hi limbs alone (11 bits), a third of the
// work; a X always takes both, because a rounding of X in a direction that X does not have
// would be multiplied by 3.4 in each step (a matrix of rank 4 in 200 rows is then 6e-2
// off, and 4e-4 with both limbs).  For Gaussian matrices of 256 to 1024 rows this leaves
// 1.3e-3 of the result's norm, below the 1.7e-3 of rounding the result to bfloat16.
//
// A, B are symmetric: only tiles on and below the diagonal are computed, and stored twice.
// X is kept in both orientations, so that all operands are read along the contracted index.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "newton_schulz.h"

namespace zb {
namespace ns {
namespace {

constexpr int kNormBlocks = 64;
constexpr int kTile = 128;     // rows and columns of a product's tile, and the padding of every matrix
constexpr int kDeep = 64;      // contracted values of a stage: 128 bytes, the swizzle's width
constexpr int kPlane = kTile * kDeep * 2;  // bytes of one operand's stage, one limb
constexpr uint64_t kPatience = 2000000000;  // nanoseconds at a barrier before a block gives up

__host__ __device__ constexpr uint64_t padded(uint64_t x) { return (x + kTile - 1) / kTile * kTile; }

// ---------------------------------------------------------------- norm and first planes

// Sum of squares, in 64 bits (no overflow, no underflow): block y's part of matrix x.
template <class T>
__global__ void __launch_bounds__(256) norm_kernel(const T* from, Matrix s, double* part) {
  __shared__ double sum[8];
  const T* at = from + int64_t(blockIdx.x) * s.matrix;
  const uint64_t n = uint64_t(s.m) * s.n;
  double x = 0.0;
  for (uint64_t i = blockIdx.y * 256ull + threadIdx.x; i < n; i += 256ull * gridDim.y) {
    // neighbouring threads along the axis that is dense in memory
    const uint64_t r = s.col <= s.row ? i / s.n : i % s.m, c = s.col <= s.row ? i % s.n : i / s.m;
    const double y = up(at[int64_t(r) * s.row + int64_t(c) * s.col]);
    x = fma(y, y, x);
  }
  for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
  if ((threadIdx.x & 31) == 0) sum[threadIdx.x >> 5] = x;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; ++i) x += sum[i];
    part[blockIdx.x * gridDim.y + blockIdx.y] = x;
  }
}

__device__ __forceinline__ double inverse_norm(const double* part, uint32_t parts) {
  double sum = 0.0;
  for (uint32_t i = 0; i < parts; ++i) sum += part[i];
  return 1.0 / (sqrt(sum) + kEps);
}

// X's planes in both orientations, zero in the padding: [count][2 limbs][mp][np] and [count][2 limbs][np][mp],
// and the first extra exponent of each matrix.
template <class T>
__global__ void __launch_bounds__(256) planes_kernel(const T* from, Matrix s, const double* part, uint32_t parts, __half* x, __half* xt,
                                                     int* extra) {
  __shared__ float tile[32][33];
  const uint32_t mp = uint32_t(padded(s.m)), np = uint32_t(padded(s.n));
  const double inverse = inverse_norm(part + uint64_t(blockIdx.z) * parts, parts);
  const int more = first_extra(inverse);
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) extra[blockIdx.z] = more;
  const double f = inverse * scalbn(double(kScale), more);
  const T* at = from + int64_t(blockIdx.z) * s.matrix;
  const uint32_t i0 = blockIdx.y * 32, j0 = blockIdx.x * 32;
  const int a = threadIdx.x & 31, b = threadIdx.x >> 5;
  const bool by_row = s.col <= s.row;
  for (int k = b; k < 32; k += 8) {
    const int ti = by_row ? k : a, tj = by_row ? a : k;
    const uint32_t i = i0 + ti, j = j0 + tj;
    tile[ti][tj] = i < s.m && j < s.n ? float(f * up(at[int64_t(i) * s.row + int64_t(j) * s.col])) : 0.0f;
  }
  __syncthreads();
  const uint64_t plane = uint64_t(mp) * np;
  x += uint64_t(blockIdx.z) * 2 * plane, xt += uint64_t(blockIdx.z) * 2 * plane;
  for (int k = b; k < 32; k += 8) {
    const float y = tile[k][a], z = tile[a][k];
    const __half yh = __float2half_rn(y), zh = __float2half_rn(z);
    const uint64_t p = uint64_t(i0 + k) * np + j0 + a, q = uint64_t(j0 + k) * mp + i0 + a;
    x[p] = yh, xt[q] = zh;
    x[plane + p] = __float2half_rn(y - __half2float(yh));
    xt[plane + q] = __float2half_rn(z - __half2float(zh));
  }
}

// No steps: the normalised matrix itself, in the caller's orientation.
template <class T>
__global__ void __launch_bounds__(256) normalise_kernel(const T* from, Matrix s, const double* part, uint32_t parts, T* out, bool transposed) {
  const double f = inverse_norm(part + uint64_t(blockIdx.x) * parts, parts);
  const T* at = from + int64_t(blockIdx.x) * s.matrix;
  const uint64_t n = uint64_t(s.m) * s.n;
  for (uint64_t e = blockIdx.y * 256ull + threadIdx.x; e < n; e += 256ull * gridDim.y) {
    const uint64_t i = transposed ? e % s.m : e / s.n, j = transposed ? e / s.m : e % s.n;
    const float y = float(f * up(at[int64_t(i) * s.row + int64_t(j) * s.col]));
    if constexpr (sizeof(T) == 2) out[blockIdx.x * n + e] = __float2bfloat16_rn(y);
    else out[blockIdx.x * n + e] = y;
  }
}

// ---------------------------------------------------------------- products

__device__ __forceinline__ uint32_t smem_at(const void* p) { return uint32_t(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void barrier_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void barrier_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool barrier_wait(uint32_t bar, uint32_t parity) {
  uint64_t began = 0, now;
  for (;;) {
    uint32_t done;
    asm volatile(
        "{\n.reg .pred p;\n"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n}"
        : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    if (done) return true;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
    if (began == 0) began = now;
    else if (now - began > kPatience) return false;
  }
}
__device__ __forceinline__ void tma_load(uint32_t to, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(to),
      "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// Shared-memory operand of a tcgen05.mma: rows of 128 bytes along the contracted index, 128-byte
// swizzle, groups of 8 rows 1024 bytes apart.
__device__ __forceinline__ uint64_t operand(uint32_t at) {
  return uint64_t((at & 0x3ffff) >> 4) | uint64_t(1) << 16 | uint64_t(1024 >> 4) << 32 | uint64_t(1) << 46 | uint64_t(2) << 61;
}
// f16 operands, 32-bit accumulators, M = N = 128.
constexpr uint32_t kInstruction = 1u << 4 | uint32_t(kTile >> 3) << 17 | uint32_t(kTile >> 4) << 24;

__device__ __forceinline__ void tensor_mma(uint32_t d, uint64_t a, uint64_t b, bool add) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b), "r"(kInstruction), "r"(uint32_t(add))
      : "memory");
}
__device__ __forceinline__ void tensor_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tensor_load(float (&r)[32], uint32_t at) {
  uint32_t* u = reinterpret_cast<uint32_t*>(r);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,"
      "%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]), "=r"(u[9]),
        "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]), "=r"(u[17]), "=r"(u[18]),
        "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]), "=r"(u[25]), "=r"(u[26]), "=r"(u[27]),
        "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
      : "r"(at));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

enum Kind { kGram, kSquare, kApply, kLast };  // A; B; X in both orientations; X to the caller

struct Product {
  uint32_t depth;         // contracted length, a multiple of kDeep
  uint32_t rows, cols;    // padded sizes of the result
  const __half* add;      // planes that the epilogue adds (A for B, X for X)
  __half* out;            // result planes
  __half* out_t;          // kApply: the transposed planes
  void* last;             // kLast: the caller's array
  int add_limbs, out_limbs, out_t_limbs;
  uint32_t step;
  const int* extra;       // first extra exponents
  uint32_t m, n;          // kLast: X's sizes
  uint32_t transposed;    // kLast: the caller's matrices are X^T
  uint32_t* failed;       // set where a barrier was waited for in vain
};

template <int LIMBS>
constexpr int kStages = LIMBS == 2 ? 3 : 6;
template <int LIMBS>
constexpr int kColumns = LIMBS == 2 ? 4 * kTile : kTile;  // of TMEM
template <int LIMBS>
constexpr int kSmem = kStages<LIMBS> * 2 * LIMBS * kPlane + 1024 + 256;

// One block: one 128 x 128 tile of L R^T (rows of both along the contracted index), then the
// step's epilogue.  Warp 0 loads, warp 1 issues the matrix instructions, warps 4 to 7 read
// the accumulators, 32 rows each.
template <int LIMBS, Kind KIND, class T>
__global__ void __launch_bounds__(256, 1)
product_kernel(const __grid_constant__ CUtensorMap left, const __grid_constant__ CUtensorMap right, const __grid_constant__ Product p) {
  constexpr int S = kStages<LIMBS>;
  extern __shared__ unsigned char raw[];
  unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + S * 2 * LIMBS * kPlane);  // full[S], empty[S], done
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * S + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  uint32_t ti, tj;
  if (KIND == kGram || KIND == kSquare) {  // lower triangle, row by row
    const uint32_t t = blockIdx.x;
    ti = uint32_t((sqrtf(8.0f * float(t) + 1.0f) - 1.0f) * 0.5f);
    while ((ti + 1) * (ti + 2) / 2 <= t) ++ti;
    while (ti * (ti + 1) / 2 > t) --ti;
    tj = t - ti * (ti + 1) / 2;
  } else {
    ti = blockIdx.x / (p.cols / kTile), tj = blockIdx.x % (p.cols / kTile);
  }
  const uint32_t z = blockIdx.y;

  if (warp == 0 && lane == 0) {
    for (int s = 0; s < S; ++s) barrier_init(smem_at(bars + s), 1), barrier_init(smem_at(bars + S + s), 1);
    barrier_init(smem_at(bars + 2 * S), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_at(tmem_slot)), "n"(kColumns<LIMBS>) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_slot;
  const int stages = int(p.depth / kDeep);

  if (warp == 0 && lane == 0) {
    int k = 0;
    bool ok = true;
    for (; k < stages && ok; ++k) {
      const int s = k % S;
      if (k >= S) ok = barrier_wait(smem_at(bars + S + s), (k / S - 1) & 1);
      if (!ok) break;
      const uint32_t bar = smem_at(bars + s), at = smem_at(base + s * 2 * LIMBS * kPlane);
      barrier_expect(bar, 2 * LIMBS * kPlane);
#pragma unroll
      for (int l = 0; l < LIMBS; ++l) {
        tma_load(at + l * kPlane, &left, bar, k * kDeep, int(ti * kTile), int(z * 2 + l));
        tma_load(at + (LIMBS + l) * kPlane, &right, bar, k * kDeep, int(tj * kTile), int(z * 2 + l));
      }
    }
    if (!ok) {  // let the copies in flight land before the block ends
      atomicExch(p.failed, 1u);
      for (int j = k > S ? k - S : 0; j < k; ++j) barrier_wait(smem_at(bars + j % S), (j / S) & 1);
    }
  } else if (warp == 1 && lane == 0) {
    bool ok = true;
    for (int k = 0; k < stages && ok; ++k) {
      const int s = k % S;
      ok = barrier_wait(smem_at(bars + s), (k / S) & 1);
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t at = smem_at(base + s * 2 * LIMBS * kPlane);
#pragma unroll
      for (int kk = 0; kk < kDeep; kk += 16) {
        const uint64_t a = operand(at + kk * 2), b = operand(at + LIMBS * kPlane + kk * 2);
        if (LIMBS == 1) {
          tensor_mma(tmem, a, b, k > 0 || kk > 0);
        } else {
          // The tensor cores' sums drop what is below 2^-24 of the running sum, always towards zero;
          // three sums for hi hi in turn and one for the small products keep that below the operands' 2^-23
          // (one sum of 3 x 2048 products: 1.4e-5 of the result, against 1.6e-6).
          const uint64_t al = operand(at + kPlane + kk * 2), bl = operand(at + (LIMBS + 1) * kPlane + kk * 2);
          tensor_mma(tmem + (k % 3) * kTile, a, b, k >= 3 || kk > 0);
          tensor_mma(tmem + 3 * kTile, a, bl, k > 0 || kk > 0);
          tensor_mma(tmem + 3 * kTile, al, b, true);
        }
      }
      tensor_commit(smem_at(bars + S + s));
    }
    if (ok) tensor_commit(smem_at(bars + 2 * S));
    else atomicExch(p.failed, 1u);
  } else if (warp >= 4) {
    bool ok = barrier_wait(smem_at(bars + 2 * S), 0);
    ok = __all_sync(0xffffffffu, ok);
    if (ok) {
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const int quarter = warp & 3;
      const uint32_t i = ti * kTile + quarter * 32 + lane;
      const uint64_t plane = uint64_t(p.rows) * p.cols;
      const __half* add = p.add + uint64_t(z) * 2 * plane + uint64_t(i) * p.cols;
      __half* out = p.out + uint64_t(z) * 2 * plane + uint64_t(i) * p.cols;
      // Scales: X 2^(12 + E), A and B 2^(12 + 2 E), their products the sums of the two.
      const int now = extra_at(p.extra[z], p.step), next = extra_at(p.extra[z], p.step + 1);
      const float f = KIND == kGram     ? kUnscale
                      : KIND == kSquare ? kC * exp2f(float(-12 - 2 * now))
                      : KIND == kApply  ? exp2f(float(-12 - 3 * now + next))
                                        : exp2f(float(-24 - 3 * now));
      const float g = KIND == kSquare ? kB : KIND == kApply ? kA * exp2f(float(next - now)) : kA * exp2f(float(-12 - now));
#pragma unroll 1
      for (int c = 0; c < kTile; c += 32) {
        const uint32_t j0 = tj * kTile + c;
        float v[32];
        tensor_load(v, tmem + (uint32_t(quarter * 32) << 16) + c);
        if (LIMBS == 2) {
          float w[32];
#pragma unroll 1
          for (int u = 1; u < 4; ++u) {
            if (u < 3 && u >= stages) continue;
            tensor_load(w, tmem + (uint32_t(quarter * 32) << 16) + u * kTile + c);
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] += w[e];
          }
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float y[8] = {};
          if (KIND != kGram) {
            for (int l = 0; l < p.add_limbs; ++l) {
              const uint4 w = *reinterpret_cast<const uint4*>(add + l * plane + j0 + q * 8);
              const __half2* h = reinterpret_cast<const __half2*>(&w);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 t = __half22float2(h[e]);
                y[2 * e] += t.x, y[2 * e + 1] += t.y;
              }
            }
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) v[q * 8 + e] = KIND == kGram ? v[q * 8 + e] * f : fmaf(v[q * 8 + e], f, g * y[e]);
        }
        if constexpr (KIND == kLast) {
          T* to = static_cast<T*>(p.last) + uint64_t(z) * p.m * p.n;
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const uint32_t j = j0 + e;
            if (i < p.m && j < p.n) {
              T* at = to + (p.transposed ? uint64_t(j) * p.m + i : uint64_t(i) * p.n + j);
              const float y = v[e];
              if constexpr (sizeof(T) == 2) *at = __float2bfloat16_rn(y);
              else *at = y;
            }
          }
        } else {
          const bool mirror = (KIND == kGram || KIND == kSquare) && ti != tj;
          __half* out_t = KIND == kApply ? p.out_t : p.out;
          const uint64_t pitch = KIND == kApply ? p.rows : p.cols;
          const int limbs_t = KIND == kApply ? p.out_t_limbs : p.out_limbs;
          out_t += uint64_t(z) * 2 * plane + i;
#pragma unroll
          for (int l = 0; l < 2; ++l) {
            if (l >= p.out_limbs) break;
            __half2 h[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              h[e] = __floats2half2_rn(v[2 * e], v[2 * e + 1]);
              const float2 t = __half22float2(h[e]);
              v[2 * e] -= t.x, v[2 * e + 1] -= t.y;
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) *reinterpret_cast<uint4*>(out + l * plane + j0 + q * 8) = *reinterpret_cast<const uint4*>(&h[4 * q]);
            if ((KIND == kApply || mirror) && l < limbs_t) {
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                out_t[l * plane + uint64_t(j0 + 2 * e) * pitch] = __low2half(h[e]);
                out_t[l * plane + uint64_t(j0 + 2 * e + 1) * pitch] = __high2half(h[e]);
              }
            }
          }
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    } else if (lane == 0) {
      atomicExch(p.failed, 1u);
    }
  }
  __syncthreads();
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(kColumns<LIMBS>));
  }
}

// ---------------------------------------------------------------- host

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                 CUtensorMapFloatOOBfill);

EncodeTiled encoder() {
  static const EncodeTiled fn = [] {
    void* at = nullptr;
    cudaDriverEntryPointQueryResult found;
    const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &at, 12000, cudaEnableDefault, &found);
    return e == cudaSuccess && found == cudaDriverEntryPointSuccess ? reinterpret_cast<EncodeTiled>(at) : nullptr;
  }();
  return fn;
}

// Planes [layers][rows][cols] in boxes of 128 rows and 64 columns.
cudaError_t make_map(CUtensorMap* map, __half* at, uint64_t cols, uint64_t rows, uint64_t layers) {
  const EncodeTiled encode = encoder();
  if (!encode) return cudaErrorNotSupported;
  const cuuint64_t size[3] = {cols, rows, layers}, stride[2] = {cols * 2, cols * rows * 2};
  const cuuint32_t box[3] = {kDeep, kTile, 1}, step[3] = {1, 1, 1};
  const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, at, size, stride, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

uint64_t align(uint64_t x) { return (x + 1023) / 1024 * 1024; }

struct Layout {
  uint64_t x, a, part, total;  // bytes of one X (one orientation), of A, of the norms' parts
  Layout(uint64_t count, uint64_t m, uint64_t n)
      : x(align(count * 2 * padded(m) * padded(n) * 2)), a(align(count * 2 * padded(m) * padded(m) * 2)),
        part(align(count * kNormBlocks * 8)) {
    total = 4 * x + 2 * a + part + align(count * 4 + 4);
  }
};

template <int LIMBS, Kind KIND, class T>
cudaError_t launch(const CUtensorMap& l, const CUtensorMap& r, const Product& p, uint32_t tiles, uint32_t count, cudaStream_t stream) {
  const auto kernel = product_kernel<LIMBS, KIND, T>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem<LIMBS>);
  if (e != cudaSuccess) return e;
  kernel<<<dim3(tiles, count), 256, kSmem<LIMBS>, stream>>>(l, r, p);
  return cudaGetLastError();
}

template <Kind KIND, class T>
cudaError_t launch(int limbs, const CUtensorMap& l, const CUtensorMap& r, const Product& p, uint32_t tiles, uint32_t count,
                   cudaStream_t stream) {
  return limbs == 2 ? launch<2, KIND, T>(l, r, p, tiles, count, stream) : launch<1, KIND, T>(l, r, p, tiles, count, stream);
}

template <class T>
cudaError_t run(const void* update, const Matrix& s, bool transposed, void* out, uint32_t steps, void* workspace, cudaStream_t stream) {
  const Layout lay(s.count, s.m, s.n);
  char* at = static_cast<char*>(workspace);
  __half *x[2], *xt[2];
  for (int i = 0; i < 2; ++i) x[i] = reinterpret_cast<__half*>(at + 2 * i * lay.x), xt[i] = reinterpret_cast<__half*>(at + (2 * i + 1) * lay.x);
  __half* a = reinterpret_cast<__half*>(at + 4 * lay.x);
  __half* b = reinterpret_cast<__half*>(at + 4 * lay.x + lay.a);
  double* part = reinterpret_cast<double*>(at + 4 * lay.x + 2 * lay.a);
  uint32_t* failed = reinterpret_cast<uint32_t*>(at + 4 * lay.x + 2 * lay.a + lay.part);
  int* extra = reinterpret_cast<int*>(failed + 1);
  const T* from = static_cast<const T*>(update);
  const uint32_t mp = uint32_t(padded(s.m)), np = uint32_t(padded(s.n));

  norm_kernel<T><<<dim3(s.count, kNormBlocks), 256, 0, stream>>>(from, s, part);
  if (steps == 0) {
    normalise_kernel<T><<<dim3(s.count, kNormBlocks), 256, 0, stream>>>(from, s, part, kNormBlocks, static_cast<T*>(out), transposed);
    return cudaGetLastError();
  }
  planes_kernel<T><<<dim3(np / 32, mp / 32, s.count), 256, 0, stream>>>(from, s, part, kNormBlocks, x[0], xt[0], extra);
  CUtensorMap mx[2], mxt[2], ma, mb;
  cudaError_t e = cudaGetLastError();
  const uint64_t layers = uint64_t(s.count) * 2;
  for (int i = 0; i < 2 && e == cudaSuccess; ++i) {
    e = make_map(&mx[i], x[i], np, mp, layers);
    if (e == cudaSuccess) e = make_map(&mxt[i], xt[i], mp, np, layers);
  }
  if (e == cudaSuccess) e = make_map(&ma, a, mp, mp, layers);
  if (e == cudaSuccess) e = make_map(&mb, b, mp, mp, layers);
  const uint32_t mt = mp / kTile, nt = np / kTile;
  // limbs of a step's products
  const auto limbs_of = [&](uint32_t i) { return sizeof(T) == 4 || mt == 1 || i + 1 >= steps ? 2 : 1; };
  for (uint32_t i = 0; i < steps && e == cudaSuccess; ++i) {
    const int now = i & 1, next = now ^ 1, limbs = limbs_of(i);
    Product p{};
    p.m = s.m, p.n = s.n, p.transposed = transposed, p.failed = failed, p.extra = extra, p.step = i;
    p.depth = np, p.rows = mp, p.cols = mp, p.add = a, p.out = a;
    p.add_limbs = p.out_limbs = limbs;
    e = launch<kGram, T>(limbs, mx[now], mx[now], p, mt * (mt + 1) / 2, s.count, stream);
    p.depth = mp, p.out = b;
    if (e == cudaSuccess) e = launch<kSquare, T>(limbs, ma, ma, p, mt * (mt + 1) / 2, s.count, stream);
    p.cols = np, p.add = x[now], p.out = x[next], p.out_t = xt[next], p.last = out;
    p.add_limbs = p.out_limbs = 2, p.out_t_limbs = limbs_of(i + 1);
    if (e == cudaSuccess)
      e = i + 1 < steps ? launch<kApply, T>(limbs, mb, mxt[now], p, mt * nt, s.count, stream)
                        : launch<kLast, T>(limbs, mb, mxt[now], p, mt * nt, s.count, stream);
  }
  return e;
}

}  // namespace
}  // namespace ns

uint64_t orthogonalize_workspace(uint32_t count, uint32_t rows, uint32_t cols, uint32_t) {
  const uint64_t m = rows < cols ? rows : cols, n = rows < cols ? cols : rows;
  if (m <= ns::kSmallRows && n <= ns::kSmallCols) return 0;
  return ns::Layout(count, m, n).total;
}

cudaError_t launch_orthogonalize(const void* update, const int64_t* strides, void* out, uint32_t count, uint32_t rows, uint32_t cols,
                                 uint32_t dtype, uint32_t steps, void* workspace, cudaStream_t stream) {
  const bool t = rows > cols;
  const ns::Matrix s{count, t ? cols : rows, t ? rows : cols, strides[0], t ? strides[2] : strides[1], t ? strides[1] : strides[2]};
  if (s.m <= ns::kSmallRows && s.n <= ns::kSmallCols) return ns::launch_small(update, s, t, out, dtype, steps, stream);
  return dtype == ZENO_DTYPE_BF16 ? ns::run<__nv_bfloat16>(update, s, t, out, steps, workspace, stream)
                                  : ns::run<float>(update, s, t, out, steps, workspace, stream);
}

}  // namespace zb
