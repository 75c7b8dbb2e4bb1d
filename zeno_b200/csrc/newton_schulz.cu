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
// Precision.  All operands are kept in two limbs, hi and lo, 22 bits together, and a product is
// hi hi + hi lo + lo hi, for bfloat16 updates too: the result is rounded to 16 bits once, at the end.
// (A rounding of X in a direction that X does not have would be multiplied by 3.4 in each step.)
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

constexpr uint32_t kNormBlocks = 256;  // of a matrix, at most
constexpr int kTile = 128;     // rows and columns of a product's tile, and the padding of every matrix
constexpr int kDeep = 64;      // contracted values of a stage: 128 bytes, the swizzle's width
constexpr int kPlane = kTile * kDeep * 2;  // bytes of one operand's stage, one limb
// Contracted values of one launch at most: the tensor cores' truncating sums lose in proportion to their length, rounded
// sums of such parts do not (130 x 262144 in one sum: 9.3e-4 of the result, 16.2 ms; in parts 1.0e-5, 18.5 ms; 2048 x 8192:
// 1.7e-5, 1776 us and 6.9e-6, 1804 us).
constexpr uint32_t kLongest = 4096;
constexpr uint64_t kPatience = 2000000000;  // nanoseconds at a barrier before a block gives up
std::atomic<uint64_t> wait_limit{kPatience};

__host__ __device__ constexpr uint64_t padded(uint64_t x) { return (x + kTile - 1) / kTile * kTile; }

// ---------------------------------------------------------------- norm and first planes

// Sums over a block of 256 threads, in every thread.
__device__ __forceinline__ double block_sum(double x) {
  __shared__ double sum[8];
  for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
  if ((threadIdx.x & 31) == 0) sum[threadIdx.x >> 5] = x;
  __syncthreads();
  x = 0.0;
  for (int i = 0; i < 8; ++i) x += sum[i];
  return x;
}

// The next kernel's blocks may start (they wait for this kernel's end before they read) ...
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
// ... and this one's for the kernel in front of it.
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Sum of squares, in 64 bits (no overflow, no underflow): block y's rows of matrix x, a warp a row
// along the axis that is dense in memory.
template <class T>
__global__ void __launch_bounds__(256) norm_kernel(const T* from, Matrix s, double* part) {
  wait_for_previous();
  let_next_start();
  const T* at = from + int64_t(blockIdx.x) * s.matrix;
  const bool by_row = s.col <= s.row;
  const uint32_t rows = by_row ? s.m : s.n, cols = by_row ? s.n : s.m;
  const int64_t row = by_row ? s.row : s.col, col = by_row ? s.col : s.row;
  double x = 0.0;
  for (uint32_t r = blockIdx.y * 8 + (threadIdx.x >> 5); r < rows; r += gridDim.y * 8) {
    const T* line = at + int64_t(r) * row;
#pragma unroll 4
    for (uint32_t c = threadIdx.x & 31; c < cols; c += 32) {
      const double y = up(line[int64_t(c) * col]);
      x = fma(y, y, x);
    }
  }
  x = block_sum(x);
  if (threadIdx.x == 0) part[blockIdx.x * gridDim.y + blockIdx.y] = x;
}

// By a whole block of 256 threads; parts <= 256.
__device__ __forceinline__ double norm_of(const double* part, uint32_t parts) {
  return sqrt(block_sum(threadIdx.x < parts ? part[threadIdx.x] : 0.0));
}

// X's planes in both orientations, zero in the padding: [count][2 limbs][mp][np] and [count][2 limbs][np][mp];
// the first extra exponent of each matrix, and no failure yet.  A block has 64 x 64 elements.
template <class T>
__global__ void __launch_bounds__(256) planes_kernel(const T* from, Matrix s, const double* part, uint32_t parts, __half* x, __half* xt,
                                                     uint32_t* failed, int* extra) {
  __shared__ float tile[64][65];
  wait_for_previous();
  let_next_start();
  const uint32_t mp = uint32_t(padded(s.m)), np = uint32_t(padded(s.n));
  const double norm = norm_of(part + uint64_t(blockIdx.z) * parts, parts);
  const int more = first_extra(norm);
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) {
    extra[blockIdx.z] = more;
    if (blockIdx.z == 0) *failed = 0;
  }
  const double f = scalbn(double(kScale), more) / (norm + kEps);
  const T* at = from + int64_t(blockIdx.z) * s.matrix;
  const uint32_t i0 = blockIdx.y * 64, j0 = blockIdx.x * 64;
  const bool by_row = s.col <= s.row;
#pragma unroll 4
  for (int e = threadIdx.x; e < 4096; e += 256) {
    const int ti = by_row ? e >> 6 : e & 63, tj = by_row ? e & 63 : e >> 6;
    const uint32_t i = i0 + ti, j = j0 + tj;
    tile[ti][tj] = i < s.m && j < s.n ? float(f * up(at[int64_t(i) * s.row + int64_t(j) * s.col])) : 0.0f;
  }
  __syncthreads();
  const uint64_t plane = uint64_t(mp) * np;
  x += uint64_t(blockIdx.z) * 2 * plane, xt += uint64_t(blockIdx.z) * 2 * plane;
  const int a = (threadIdx.x & 31) * 2;
#pragma unroll 4
  for (int k = threadIdx.x >> 5; k < 64; k += 8) {
    const uint64_t p = uint64_t(i0 + k) * np + j0 + a, q = uint64_t(j0 + k) * mp + i0 + a;
    const __half2 y = __floats2half2_rn(tile[k][a], tile[k][a + 1]), z = __floats2half2_rn(tile[a][k], tile[a + 1][k]);
    const float2 fy = __half22float2(y), fz = __half22float2(z);
    *reinterpret_cast<__half2*>(x + p) = y;
    *reinterpret_cast<__half2*>(xt + q) = z;
    *reinterpret_cast<__half2*>(x + plane + p) = __floats2half2_rn(tile[k][a] - fy.x, tile[k][a + 1] - fy.y);
    *reinterpret_cast<__half2*>(xt + plane + q) = __floats2half2_rn(tile[a][k] - fz.x, tile[a + 1][k] - fz.y);
  }
}

// No steps: the normalised matrix itself, in the caller's orientation.
template <class T>
__global__ void __launch_bounds__(256) normalise_kernel(const T* from, Matrix s, const double* part, uint32_t parts, T* out, bool transposed) {
  wait_for_previous();
  const double f = 1.0 / (norm_of(part + uint64_t(blockIdx.x) * parts, parts) + kEps);
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
// Whether the phase ended within `patience` nanoseconds (0: not waited for at all).
__device__ __forceinline__ bool barrier_wait(uint32_t bar, uint32_t parity, uint64_t patience) {
  uint64_t began = 0, now;
  if (patience == 0) return false;
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
    else if (now - began > patience) return false;
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
// 16 rows and 64 columns of accumulators: v[4 c + x] is column 8 c + 2 (lane % 4) + (x & 1) of row
// lane / 4 + 8 (x >> 1), as the tiles of mma.sync have it.
__device__ __forceinline__ void tensor_load(float (&r)[32], uint32_t at) {
  uint32_t* u = reinterpret_cast<uint32_t*>(r);
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,"
      "%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]), "=r"(u[9]),
        "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]), "=r"(u[17]), "=r"(u[18]),
        "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]), "=r"(u[25]), "=r"(u[26]), "=r"(u[27]),
        "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
      : "r"(at));
}
// The loads in front of it have their values.  They pass through here, so that no use of them moves up.
__device__ __forceinline__ void tensor_wait(float (&a)[32], float (&b)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) asm volatile("" : "+f"(a[i]), "+f"(b[i]));
}

// Four 8 x 8 tiles of 16-bit values to shared memory, lane l giving the address of row l % 8 of tile l / 8.
__device__ __forceinline__ void store_tiles(uint32_t at, const uint32_t (&r)[4]) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3])
               : "memory");
}
__device__ __forceinline__ void store_tiles_transposed(uint32_t at, const uint32_t (&r)[4]) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3])
               : "memory");
}
__device__ __forceinline__ void tma_store(const CUtensorMap* map, uint32_t from, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map), "r"(from), "r"(x),
               "r"(y), "r"(z)
               : "memory");
}

// Barrier of the 256 threads of the epilogue: whether all of them say yes.
__device__ __forceinline__ bool all_of_256(bool yes) {
  uint32_t all;
  asm volatile(
      "{\n.reg .pred p, q;\nsetp.ne.u32 p, %1, 0;\n"
      "barrier.cta.red.and.pred q, 1, 256, p;\nselp.u32 %0, 1, 0, q;\n}"
      : "=r"(all) : "r"(uint32_t(yes)) : "memory");
  return all != 0;
}

enum Kind { kGram, kSquare, kApply, kLast };  // A; B; X in both orientations; X to the caller

struct Product {
  uint32_t depth;         // contracted length, a multiple of kDeep,
  uint32_t from;          // from this index on
  uint32_t more;          // further part of a long sum: the result so far is what is added to
  uint32_t cols;          // padded columns of the result
  uint32_t step;
  const int* extra;       // first extra exponents
  void* last;             // kLast: the caller's array
  uint32_t m, n;          // kLast: X's sizes
  uint32_t transposed;    // kLast: the caller's matrices are X^T
  uint32_t* failed;       // set where a barrier was waited for in vain; kLast writes NaN then
  uint64_t patience;
};

// Shared memory: a ring of 6 units of 32 KB; a stage is two units, both operands' hi and lo limbs.
// Behind the last stage come two units with the tile that the epilogue adds, and the
// other four, once the products are done, hold the result's limb planes in both orientations.
constexpr int kLimbs = 2, kUnits = 6, kUnit = 2 * kPlane;
constexpr int kSmem = kUnits * kUnit + 1024 + 256;
constexpr int kColumns = 4 * kTile;  // of TMEM

// Byte of element (row, col) in a unit that holds a 128 x 128 tile as two swizzled boxes of 64 columns.
__device__ __forceinline__ uint32_t in_unit(uint32_t row, uint32_t col) {
  return (col >> 6) * kPlane + row * 128 + ((((col >> 3) & 7) ^ (row & 7)) << 4) + (col & 7) * 2;
}

// One block: one 128 x 128 tile of L R^T (rows of both along the contracted index), then the
// step's epilogue.  Warp 0 loads, warp 1 issues the matrix instructions, warps 4 to 11 read
// the accumulators, 32 rows and 64 columns each.
template <Kind KIND, class T>
__global__ void __launch_bounds__(384, 1)
product_kernel(const __grid_constant__ CUtensorMap left, const __grid_constant__ CUtensorMap right, const __grid_constant__ CUtensorMap add,
               const __grid_constant__ CUtensorMap out, const __grid_constant__ CUtensorMap out_t, const __grid_constant__ Product p) {
  constexpr int S = kUnits / kLimbs;
  extern __shared__ unsigned char raw[];
  unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + kUnits * kUnit);  // full[S], empty[S], done, added, drained
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * S + 3);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr bool kSymmetric = KIND == kGram || KIND == kSquare;

  uint32_t ti, tj;
  if (kSymmetric) {  // lower triangle, row by row
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
    for (int s = 0; s < 2 * S + 3; ++s) barrier_init(smem_at(bars + s), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_at(tmem_slot)), "n"(kColumns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_slot;
  const int stages = int(p.depth / kDeep);
  const bool adds = KIND != kGram || p.more;
  const uint32_t unit0 = smem_at(base);
  const int first_add = stages * kLimbs % kUnits;
  const uint32_t done = smem_at(bars + 2 * S), added = smem_at(bars + 2 * S + 1), drained = smem_at(bars + 2 * S + 2);
  wait_for_previous();
  let_next_start();
  asm volatile("fence.proxy.async;" ::: "memory");  // the planes may come from ordinary stores

  if (warp == 0 && lane == 0) {
    int k = 0;
    bool ok = true;
    for (; k < stages; ++k) {
      const int s = k % S;
      if (k >= S) ok = barrier_wait(smem_at(bars + S + s), (k / S - 1) & 1, p.patience);
      if (!ok) break;
      const uint32_t bar = smem_at(bars + s), at = unit0 + s * kLimbs * kUnit;
      barrier_expect(bar, kLimbs * kUnit);
#pragma unroll
      for (int l = 0; l < kLimbs; ++l) {
        tma_load(at + l * kPlane, &left, bar, int(p.from) + k * kDeep, int(ti * kTile), int(z * 2 + l));
        tma_load(at + (kLimbs + l) * kPlane, &right, bar, int(p.from) + k * kDeep, int(tj * kTile), int(z * 2 + l));
      }
    }
    if (adds && ok) {
      if (stages >= S) ok = barrier_wait(smem_at(bars + S + stages % S), (stages / S - 1) & 1, p.patience);
      if (ok) {
        barrier_expect(added, kLimbs * kUnit);
        for (int l = 0; l < kLimbs; ++l)
          for (int half = 0; half < 2; ++half)
            tma_load(unit0 + (first_add + l) % kUnits * kUnit + half * kPlane, &add, added, int(tj * kTile) + half * kDeep, int(ti * kTile),
                     int(z * 2 + l));
      }
    }
    if (!ok) atomicExch(p.failed, 1u);
    // the copies in flight land before the block ends, whoever gave up
    for (int j = k > S ? k - S : 0; j < k; ++j) barrier_wait(smem_at(bars + j % S), (j / S) & 1, kPatience);
    if (adds && ok) barrier_wait(added, 0, kPatience);
  } else if (warp == 1 && lane == 0) {
    bool ok = true;
    for (int k = 0; k < stages; ++k) {
      const int s = k % S;
      ok = barrier_wait(smem_at(bars + s), (k / S) & 1, p.patience);
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t at = unit0 + s * kLimbs * kUnit;
#pragma unroll
      for (int kk = 0; kk < kDeep; kk += 16) {
        // The tensor cores' sums drop what is below 2^-24 of the running sum, always towards zero;
        // three sums for hi hi in turn and one for the small products keep that below the operands' 2^-23
        // (2048 x 2048: one sum of 3 x 2048 products leaves 1.4e-5 of the result, these 4.5e-6, 32-bit torch 3.7e-6).
        const uint64_t a = operand(at + kk * 2), b = operand(at + kLimbs * kPlane + kk * 2);
        const uint64_t al = operand(at + kPlane + kk * 2), bl = operand(at + (kLimbs + 1) * kPlane + kk * 2);
        tensor_mma(tmem + (k % 3) * kTile, a, b, k >= 3 || kk > 0);
        tensor_mma(tmem + 3 * kTile, a, bl, k > 0 || kk > 0);
        tensor_mma(tmem + 3 * kTile, al, b, true);
      }
      tensor_commit(smem_at(bars + S + s));
    }
    if (!ok) atomicExch(p.failed, 1u);
    // ... and the products under way end before the accumulators are given back
    const uint32_t end = ok ? done : drained;
    tensor_commit(end);
    barrier_wait(end, 0, kPatience);
  } else if (warp >= 4) {
    // Scales: X 2^(12 + E), A and B 2^(12 + 2 E), their products the sums of the two.
    const int first = p.extra[z], now = extra_at(first, p.step), next = extra_at(first, p.step + 1);
    const float f = KIND == kGram     ? kUnscale
                    : KIND == kSquare ? kC * exp2f(float(-12 - 2 * now))
                    : KIND == kApply  ? exp2f(float(-12 - 3 * now + next))
                                      : exp2f(float(-24 - 3 * now));
    const float g = KIND == kLast ? (p.more ? exp2f(float(-12 - next)) : kA * exp2f(float(-12 - now)))
                    : p.more      ? 1.0f
                    : KIND == kSquare ? kB
                                      : kA * exp2f(float(next - now));
    const bool earlier = KIND == kLast && *p.failed != 0;  // a product that this one builds on gave up
    bool ok = barrier_wait(done, 0, p.patience);
    if (adds && ok) ok = barrier_wait(added, 0, p.patience);
    ok = __all_sync(0xffffffffu, ok && !earlier);
    if (ok) {
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const int quarter = warp & 3, gi = lane >> 2, qj = (lane & 3) * 2;
      const bool mirror = KIND == kApply || (kSymmetric && ti != tj);
      const unsigned char* add0 = base + first_add * kUnit;
      const unsigned char* add1 = base + (first_add + 1) % kUnits * kUnit;
#pragma unroll 1
      for (int part = 0; part < 2; ++part) {
        const uint32_t r0 = quarter * 32 + part * 16, c0 = ((warp >> 2) - 1) * 64;
        float v[32], w[32];
        const uint32_t at = tmem + (r0 << 16) + c0;
        tensor_load(v, at);
        tensor_load(w, at + 3 * kTile);
        tensor_wait(v, w);
        float x[32];
        const bool third = stages > 2;
        tensor_load(x, at + kTile);
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] += w[e];
        if (third) tensor_load(w, at + 2 * kTile);
        tensor_wait(x, w);
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] += third ? x[e] + w[e] : x[e];
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const uint32_t row = r0 + gi + ((e >> 1) & 1) * 8, col = c0 + (e >> 2) * 8 + qj;
          if (!adds) {
            v[e] *= f, v[e + 1] *= f;
          } else {
            const float2 y = __half22float2(*reinterpret_cast<const __half2*>(add0 + in_unit(row, col)));
            const float2 z = __half22float2(*reinterpret_cast<const __half2*>(add1 + in_unit(row, col)));
            v[e] = fmaf(v[e], f, g * (y.x + z.x)), v[e + 1] = fmaf(v[e + 1], f, g * (y.y + z.y));
          }
          if constexpr (KIND == kLast) {
            const uint32_t i = ti * kTile + row, j = tj * kTile + col;
            T* to = static_cast<T*>(p.last) + uint64_t(z) * p.m * p.n;
#pragma unroll
            for (int q = 0; q < 2; ++q)
              if (i < p.m && j + q < p.n) {
                T* at_out = to + (p.transposed ? uint64_t(j + q) * p.m + i : uint64_t(i) * p.n + j + q);
                if constexpr (sizeof(T) == 2) *at_out = __float2bfloat16_rn(v[e + q]);
                else *at_out = v[e + q];
              }
          }
        }
        if constexpr (KIND != kLast) {
          const uint32_t tile_row = lane & 7, right_tile = (lane >> 4) * 8, low_tile = ((lane >> 3) & 1) * 8;
#pragma unroll
          for (int l = 0; l < kLimbs; ++l) {
            const uint32_t u_row = unit0 + (first_add + 2 + l) % kUnits * kUnit, u_col = unit0 + (first_add + 4 + l) % kUnits * kUnit;
#pragma unroll
            for (int c = 0; c < 64; c += 16) {
              uint32_t h[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                float* x = &v[c / 2 + e * 2];
                const __half2 y = __floats2half2_rn(x[0], x[1]);
                const float2 b = __half22float2(y);
                x[0] -= b.x, x[1] -= b.y;
                h[e] = *reinterpret_cast<const uint32_t*>(&y);
              }
              store_tiles(u_row + in_unit(r0 + low_tile + tile_row, c0 + c + right_tile), h);
              if (mirror) store_tiles_transposed(u_col + in_unit(c0 + c + right_tile + tile_row, r0 + low_tile), h);
            }
          }
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    } else {
      if (lane == 0) atomicExch(p.failed, 1u);
      if constexpr (KIND == kLast) {  // what cannot be computed is not a number
        T* to = static_cast<T*>(p.last) + uint64_t(z) * p.m * p.n;
        const uint32_t i = ti * kTile + (warp & 3) * 32 + lane, j0 = tj * kTile + ((warp >> 2) - 1) * 64;
        if (i < p.m)
          for (uint32_t j = j0; j < min(j0 + 64, p.n); ++j)
            to[p.transposed ? uint64_t(j) * p.m + i : uint64_t(i) * p.n + j] = T(__int_as_float(0x7fffffff));
      }
    }
    if (KIND != kLast) {
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      if (all_of_256(ok) && warp == 4 && lane == 0) {
        const bool mirror = KIND == kApply || ti != tj;
        for (int l = 0; l < kLimbs; ++l)
          for (int half = 0; half < 2; ++half) {
            tma_store(&out, unit0 + (first_add + 2 + l) % kUnits * kUnit + half * kPlane, int(tj * kTile) + half * kDeep, int(ti * kTile),
                      int(z * 2 + l));
            if (mirror)
              tma_store(&out_t, unit0 + (first_add + 4 + l) % kUnits * kUnit + half * kPlane, int(ti * kTile) + half * kDeep,
                        int(tj * kTile), int(z * 2 + l));
          }
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
      }
    }
  }
  __syncthreads();
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(kColumns));
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

// A launch whose blocks may start while the kernel in front of it ends.
template <class... Params, class... Args>
cudaError_t launch_after(void (*kernel)(Params...), dim3 grid, int threads, int smem, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t c{};
  c.gridDim = grid, c.blockDim = dim3(threads), c.dynamicSmemBytes = size_t(smem), c.stream = stream;
  cudaLaunchAttribute a{};
  a.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  a.val.programmaticStreamSerializationAllowed = 1;
  c.attrs = &a, c.numAttrs = 1;
  return cudaLaunchKernelEx(&c, kernel, args...);
}

struct Maps {
  CUtensorMap left, right, add, out, out_t;
};

template <Kind KIND, class T = float>  // T: the caller's type, of kLast
cudaError_t launch(const Maps& m, const Product& p, uint32_t tiles, uint32_t count, cudaStream_t stream) {
  const auto kernel = product_kernel<KIND, T>;
  static std::atomic<uint64_t> allowed{0};
  const cudaError_t e = allow_smem(kernel, kSmem, allowed);
  if (e != cudaSuccess) return e;
  return launch_after(kernel, dim3(tiles, count), 384, kSmem, stream, m.left, m.right, m.add, m.out, m.out_t, p);
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

  const uint32_t dense_rows = s.col <= s.row ? s.m : s.n;
  const uint32_t parts = dense_rows >= 8 * kNormBlocks ? kNormBlocks : (dense_rows + 7) / 8;
  cudaError_t e = launch_after(norm_kernel<T>, dim3(s.count, parts), 256, 0, stream, from, s, part);
  if (e != cudaSuccess) return e;
  if (steps == 0)
    return launch_after(normalise_kernel<T>, dim3(s.count, 64), 256, 0, stream, from, s, static_cast<const double*>(part), parts,
                        static_cast<T*>(out), transposed);
  e = launch_after(planes_kernel<T>, dim3(np / 64, mp / 64, s.count), 256, 0, stream, from, s, static_cast<const double*>(part), parts, x[0],
                   xt[0], failed, extra);
  CUtensorMap mx[2], mxt[2], ma, mb;
  const uint64_t layers = uint64_t(s.count) * 2;
  for (int i = 0; i < 2 && e == cudaSuccess; ++i) {
    e = make_map(&mx[i], x[i], np, mp, layers);
    if (e == cudaSuccess) e = make_map(&mxt[i], xt[i], mp, np, layers);
  }
  if (e == cudaSuccess) e = make_map(&ma, a, mp, mp, layers);
  if (e == cudaSuccess) e = make_map(&mb, b, mp, mp, layers);
  const uint32_t mt = mp / kTile, nt = np / kTile, lower = mt * (mt + 1) / 2;
  for (uint32_t i = 0; i < steps && e == cudaSuccess; ++i) {
    const int now = i & 1, next = now ^ 1;
    Product p{};
    p.m = s.m, p.n = s.n, p.transposed = transposed, p.failed = failed, p.extra = extra, p.step = i, p.last = out;
    p.patience = wait_limit.load(std::memory_order_relaxed);
    // The parts of a product, each added to what the ones in front of it left in `sum`.
    const auto in_parts = [&](uint32_t depth, const CUtensorMap& sum, Maps m, const auto& launch_part) {
      const uint32_t parts = (depth + kLongest - 1) / kLongest, each = (depth / kTile + parts - 1) / parts * kTile;
      for (p.from = p.more = 0; p.from < depth && e == cudaSuccess; p.from += each, p.more = 1, m.add = sum) {
        p.depth = depth - p.from < each ? depth - p.from : each;
        e = launch_part(m, p.from + each >= depth);
      }
    };
    p.cols = mp;
    in_parts(np, ma, Maps{mx[now], mx[now], ma, ma, ma},
             [&](const Maps& m, bool) { return launch<kGram>(m, p, lower, s.count, stream); });
    in_parts(mp, mb, Maps{ma, ma, ma, mb, mb}, [&](const Maps& m, bool) { return launch<kSquare>(m, p, lower, s.count, stream); });
    p.cols = np;
    in_parts(mp, mx[next], Maps{mb, mxt[now], mx[now], mx[next], mxt[next]}, [&](const Maps& m, bool end) {
      return end && i + 1 == steps ? launch<kLast, T>(m, p, mt * nt, s.count, stream) : launch<kApply>(m, p, mt * nt, s.count, stream);
    });
  }
  return e;
}

}  // namespace
}  // namespace ns

uint64_t orthogonalize_wait_limit(uint64_t nanoseconds) { return ns::wait_limit.exchange(nanoseconds); }

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
