// Long rollouts of wide heads (more than 64 channels, bfloat16): the chunked linear attention of linear_forward.cuh with its products on
// tcgen05.
//
// A chunk of 64 tokens is products of 64 and 128 rows, too few instructions apart for mma.sync to be fed: loading and holding its operands
// was two thirds of the instructions that the general kernels issue for such a head (1800 a warp and chunk forward).  Here operands are
// tiles of 64 columns in shared memory with the 128-byte swizzle, read along either axis, one thread issues the products,
// and the warps do what is left: decays, limbs, the state's sum.  The accumulators come back in the same fragments as those of mma.sync, so that
// the formulas are written as there.  Sums of a chunk are taken in TMEM, the state itself is summed in registers (the tensor cores truncate).
//
// 2 x 4096 tokens, 8 heads of 128 x 128: 27 us for the segments' sums and 61 us for the results (8 segments of 8 chunks for each head, 128 blocks on 148 SMs:
// a chain that is walked twice); 8 x 1000 tokens backward: 150 us.  The tensor pipe is 16 % and 21 % busy; a chunk's loads, limbs and products wait for one another.
//
// Waits end after a limit; a block whose products do not finish writes NaN.
#pragma once
#include "linear_backward.cuh"

namespace zb {
namespace linear {
namespace tensor {

constexpr int C = 64, D = 128;
constexpr int kTok = C * D;          // elements of a tile of token rows: two blocks [64 rows][64 columns]
constexpr int kPair = C * C;         // of a token-by-token tile: one block
constexpr int kState = D * D;        // of a state: two blocks [128 rows][64 columns]
constexpr uint64_t kPatience = 2000000000;  // nanoseconds at a barrier before a block gives up

// Where an element is: blocks of 64 columns, rows of 128 bytes whose 16-byte pieces are swapped within groups of 8 rows.
template <int ROWS>
__device__ __forceinline__ int spot(int row, int col) {
  return (col >> 6) * (ROWS * 64) + row * 64 + ((((col >> 3) & 7) ^ (row & 7)) << 3) + (col & 7);
}

// Operands of tcgen05.mma.  ALONG: rows hold the contracted index (step k: 16 columns of a block).  ACROSS: rows are the contracted index, the
// operand's own index lies along them (step k: 16 rows), its blocks of 64 are ROWS * 128 bytes apart.
__device__ __forceinline__ uint64_t descriptor(uint32_t at, uint32_t leading) {
  return uint64_t((at & 0x3ffff) >> 4) | uint64_t(leading >> 4) << 16 | uint64_t(1024 >> 4) << 32 | uint64_t(1) << 46 | uint64_t(2) << 61;
}
template <int ROWS>
__device__ __forceinline__ uint64_t along(uint32_t at, int k) {
  return descriptor(at + (k >> 2) * (ROWS * 128) + (k & 3) * 32, 16);
}
template <int ROWS>
__device__ __forceinline__ uint64_t across(uint32_t at, int k) {
  return descriptor(at + k * 2048, ROWS * 128);
}
// bfloat16 operands, 32-bit sums, M x N; TA, TB: A, B are read across.
template <int M, int N, bool TA, bool TB>
constexpr uint32_t kInstruction = 1u << 4 | 1u << 7 | 1u << 10 | uint32_t(TA) << 15 | uint32_t(TB) << 16 | uint32_t(N >> 3) << 17 |
                                  uint32_t(M >> 4) << 24;
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t instruction, bool add) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b), "r"(instruction), "r"(uint32_t(add))
      : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Whether the phase ended within `patience` nanoseconds (0: not waited for at all).
__device__ __forceinline__ bool ended(uint32_t bar, uint32_t parity, uint64_t patience) {
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

// 16 rows and 8 X columns of accumulators: r[4 c + x] is column 8 c + 2 (lane % 4) + (x & 1) of row lane / 4 + 8 (x >> 1), as the tiles of
// mma.sync have it.
__device__ __forceinline__ void fetch2(float* r, uint32_t at) {
  uint32_t* u = reinterpret_cast<uint32_t*>(r);
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]) : "r"(at));
}
__device__ __forceinline__ void fetch4(float* r, uint32_t at) {
  uint32_t* u = reinterpret_cast<uint32_t*>(r);
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
                 "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
               : "r"(at));
}
// The loads in front of it have their values; these pass through here, so that no use of them moves up.
template <int N>
__device__ __forceinline__ void fetched(float (&r)[N][2][4]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) asm volatile("" : "+f"(r[j][e >> 2][e & 3]));
}

// The value that N planes hold; the first alone where it is not finite.
template <int N, int ROWS>
__device__ __forceinline__ float value_at(const plane_t* at, int plane, int row, int col) { return value<N>(at + spot<ROWS>(row, col), plane); }

// Which 8 columns of which rows of a chunk a thread moves.
template <int THREADS>
struct Mover {
  static constexpr int STEP = THREADS / 16, TURNS = C / STEP;
  int row, c;
  __device__ __forceinline__ explicit Mover(int tid) : row(tid >> 4), c((tid & 15) * 8) {}
};

// All threads: a chunk's rows as a tile, zero for absent tokens and past the width.
template <int THREADS>
__device__ __forceinline__ void load_tile(plane_t* to, const bf16* from, int64_t stride, int width, bool vec, int n, const Mover<THREADS>& mv) {
  using M = Mover<THREADS>;
  const bf16* at = from + mv.row * stride + mv.c;
#pragma unroll
  for (int u = 0; u < M::TURNS; ++u) {
    const int row = mv.row + u * M::STEP;
    const bool there = row < n && mv.c < width;
    plane_t* spot_at = to + spot<C>(row, mv.c);
    if (vec) {
      copy16(spot_at, there ? at : from, there);
    } else {
      delta::Eight raw{};
      if (there) raw = delta::fetch8_slow(at, width - mv.c);
      *reinterpret_cast<uint4*>(spot_at) = raw.a;
    }
    at += M::STEP * stride;
  }
}
template <int THREADS>
__device__ __forceinline__ void store_tile(bf16* to, int64_t stride, const plane_t* from, int width, bool vec, int n, const Mover<THREADS>& mv) {
  using M = Mover<THREADS>;
  if (mv.c >= width) return;
  plane_t* at = reinterpret_cast<plane_t*>(to) + mv.row * stride + mv.c;
#pragma unroll
  for (int u = 0; u < M::TURNS; ++u) {
    const int row = mv.row + u * M::STEP;
    if (row >= n) break;
    const plane_t* x = from + spot<C>(row, mv.c);
    if (vec) {
      *reinterpret_cast<uint4*>(at) = *reinterpret_cast<const uint4*>(x);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (mv.c + i < width) at[i] = x[i];
    }
    at += M::STEP * stride;
  }
}
// Whether something that this thread brought is not finite.
template <int THREADS>
__device__ __forceinline__ bool tile_odd(const plane_t* at, const Mover<THREADS>& mv) {
  __nv_bfloat162 z = __floats2bfloat162_rn(0.0f, 0.0f);
  const __nv_bfloat162 nothing = z;
#pragma unroll
  for (int u = 0; u < Mover<THREADS>::TURNS; ++u) {
    const uint4 w = *reinterpret_cast<const uint4*>(at + spot<C>(mv.row + u * Mover<THREADS>::STEP, mv.c));
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) z = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&x[e]), nothing, z);
  }
  const float sum = __low2float(z) + __high2float(z);
  return sum != sum;
}

// The pieces that this thread brought, each row times factor weight[row], as three tiles of limbs.
template <int THREADS>
__device__ __forceinline__ void weigh(plane_t* to, const plane_t* from, const float* weight, float factor, const Mover<THREADS>& mv) {
#pragma unroll
  for (int u = 0; u < Mover<THREADS>::TURNS; ++u) {
    const int row = mv.row + u * Mover<THREADS>::STEP, at = spot<C>(row, mv.c);
    const float f = weight[row] * factor;
    const uint4 w = *reinterpret_cast<const uint4*>(from + at);
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
    uint32_t r[4][3];
#pragma unroll
    for (int i = 0; i < 4; ++i) split<3>(lower(x[i]) * f, upper(x[i]) * f, r[i]);
#pragma unroll
    for (int l = 0; l < 3; ++l) *reinterpret_cast<uint4*>(to + l * kTok + at) = make_uint4(r[0][l], r[1][l], r[2][l], r[3][l]);
  }
}

// A part of a state in planes, N limbs.
template <class S, int N>
__device__ __forceinline__ void dump(const float (&m)[S::NM][2][4], plane_t* to, const Part<S>& part, int lane) {
#pragma unroll
  for (int j = 0; j < S::NM; ++j)
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        uint32_t w[N];
        split<N>(m[j][h][2 * r], m[j][h][2 * r + 1], w);
        const int at = spot<D>(part.row + (lane >> 2) + r * 8, part.col + j * 16 + h * 8 + (lane & 3) * 2);
#pragma unroll
        for (int l = 0; l < N; ++l) *reinterpret_cast<uint32_t*>(to + l * kState + at) = w[l];
      }
}

// The part of a state that a warp has: 16 rows of its quarter of TMEM's lanes, and every column or half of them.
template <class S>
__device__ __forceinline__ Part<S> part_of(int warp) {
  Part<S> part(0, D, D);
  part.row = (warp & 3) * 32 + ((warp >> 2) & 1) * 16;
  part.col = (warp >> 3) * S::NM * 16;
  part.pairs = S::NM;
  return part;
}

// A state that is kept for the backward pass: as the threads hold it, whole vectors of a warp side by side, where it has the full width (and
// then the same number of bytes), in rows otherwise.
template <class S>
__device__ __forceinline__ void write_saved(const float (&m)[S::NM][2][4], float* to, const Part<S>& part, int dk, int dv, int lane, int tid) {
  if constexpr (S::FULL) {
#pragma unroll
    for (int i = 0; i < S::NM * 2; ++i)
      reinterpret_cast<float4*>(to)[i * S::THREADS + tid] = make_float4(m[i >> 1][i & 1][0], m[i >> 1][i & 1][1], m[i >> 1][i & 1][2], m[i >> 1][i & 1][3]);
  } else {
    write_state<S>(m, to, part, dk, dv, lane);
  }
}
template <class S>
__device__ __forceinline__ void read_saved(float (&m)[S::NM][2][4], const float* from, const Part<S>& part, int dk, int dv, int lane, int tid) {
  if constexpr (S::FULL) {
#pragma unroll
    for (int i = 0; i < S::NM * 2; ++i) {
      const float4 x = reinterpret_cast<const float4*>(from)[i * S::THREADS + tid];
      m[i >> 1][i & 1][0] = x.x, m[i >> 1][i & 1][1] = x.y, m[i >> 1][i & 1][2] = x.z, m[i >> 1][i & 1][3] = x.w;
    }
  } else {
    read_state<S>(m, from, part, dk, dv, lane);
  }
}
// One value of it.
template <class S>
__device__ __forceinline__ float saved_value(const float* from, bool saved, int row, int col, int dv) {
  if (!S::FULL || !saved) return from[row * dv + col];
  const int warp = (row >> 5) | ((row >> 4) & 1) << 2 | (col / (S::NM * 16)) << 3;
  const int j = col % (S::NM * 16) / 16, h = (col >> 3) & 1, lane = (row & 7) * 4 + ((col & 7) >> 1);
  return from[((j * 2 + h) * S::THREADS + warp * 32 + lane) * 4 + ((row >> 3) & 1) * 2 + (col & 1)];
}

// m = keep m + the accumulators at `at`.
template <class S>
__device__ __forceinline__ void merge(float (&m)[S::NM][2][4], uint32_t at, float keep, const Part<S>& part) {
#pragma unroll
  for (int j = 0; j < S::NM; j += 2) {
    float add[2][2][4];
    fetch4(&add[0][0][0], at + (uint32_t(part.row) << 16) + part.col + j * 16);
    fetched(add);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      float& z = m[j + (e >> 3)][(e >> 2) & 1][e & 3];
      const float y = add[e >> 3][(e >> 2) & 1][e & 3];
      z = keep == 0.0f ? y : fmaf(keep, z, y);
    }
  }
}
// The same element by element, leaving out tokens of no weight.
template <class S>
__device__ __noinline__ void merge_slow(float* m, const plane_t* x, const plane_t* y, const float* weight, float factor, float keep, int n, int row, int col) {
  float sum = 0.0f;
  for (int j = 0; j < n; ++j)
    if (weight[j] != 0.0f) sum = fmaf(weight[j] * factor * value_at<1, C>(x, 0, j, row), value_at<1, C>(y, 0, j, col), sum);
  *m = keep == 0.0f ? sum : fmaf(keep, *m, sum);
}
template <class S>
__device__ __forceinline__ void merge_masked(float (&m)[S::NM][2][4], const plane_t* x, const plane_t* y, const float* weight, float factor, float keep,
                                             int n, const Part<S>& part, int lane) {
#pragma unroll
  for (int j = 0; j < S::NM; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float z = m[j][e >> 2][e & 3];
      merge_slow<S>(&z, x, y, weight, factor, keep, n, part.row + (lane >> 2) + ((e >> 1) & 1) * 8,
                    part.col + j * 16 + (e >> 2) * 8 + (lane & 3) * 2 + (e & 1));
      m[j][e >> 2][e & 3] = z;
    }
}

// What a block holds besides its tiles.
struct Control {
  uint64_t bar;
  uint32_t tmem, pad;
};
template <int COLUMNS>
__device__ __forceinline__ void begin(Control& c, int warp, int tid) {
  if (tid == 0) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(delta::smem_at(&c.bar)) : "memory");
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(delta::smem_at(&c.tmem)), "n"(COLUMNS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  fence_after();
}
template <int COLUMNS>
__device__ __forceinline__ void end(uint32_t tmem, int warp) {
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(COLUMNS));
}

// The products issued since the last wait: whether they ended, the same answer in every thread.  Where they did not, another wait
// lets them end before anything is given back.
struct Products {
  uint32_t bar, parity;
  uint64_t patience;
  __device__ __forceinline__ void issued(bool mine) {
    if (mine) commit(bar);
  }
  __device__ __forceinline__ bool done() {
    bool ok = ended(bar, parity, patience);
    ok = __syncthreads_and(ok);
    if (!ok) ended(bar, parity, kPatience);
    parity ^= 1;
    fence_after();
    return ok;
  }
};

template <bool FULL>
using WideShape = Shape<bf16, D, C, 16, FULL>;     // main kernels
template <bool FULL>
using SegmentShape = Shape<bf16, D, C, 8, FULL>;   // segments

// Not a number, where a block gave up.
__device__ __forceinline__ float lost() { return __uint_as_float(0x7fffffffu); }

constexpr int kForwardBytes = 1024 + 2 * (5 * kTok + 2 * kPair + 2 * kState + 3 * kTok) + 2 * int(sizeof(Gates<C>)) + int(sizeof(Control));
constexpr int kSegmentBytes = 1024 + 2 * (3 * kTok + 3 * kTok) + 2 * int(sizeof(Gates<C>)) + int(sizeof(Control));

// The next chunk's rows and gates are fetched while a chunk's products run: Q and V into a second tile each, K, once it is not needed
// any more, into its own.  The outputs leave by way of P's tiles.
template <class S>
__global__ void __launch_bounds__(S::THREADS, 1)
linear_tensor_forward_kernel(const __grid_constant__ ZenoLinearAttention p, const Segments sg, const uint64_t patience) {
  extern __shared__ char smem[];
  plane_t* const q0 = reinterpret_cast<plane_t*>((reinterpret_cast<uintptr_t>(smem) + 1023) / 1024 * 1024);
  plane_t *const v0 = q0 + 2 * kTok, *const k = v0 + 2 * kTok, *const pr = k + kTok, *const st = pr + 2 * kPair, *const wk = st + 2 * kState;
  Gates<C>* const gates = reinterpret_cast<Gates<C>*>(wk + 3 * kTok);
  Control& control = *reinterpret_cast<Control*>(gates + 2);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rt = warp & 3, ct = warp >> 2;  // 16 tokens, and a quarter of a product's columns
  const int dk = S::FULL ? D : int(p.key_dim), dv = S::FULL ? D : int(p.value_dim);
  const At a = block_at(p, sg, 0, C);
  if (a.b >= p.batch) return;
  const Mover<S::THREADS> mv(tid);
  const int64_t state_size = int64_t(dk) * dv;
  const bf16 *gq = place<bf16>(p.q, a.b, a.kh), *gk = place<bf16>(p.k, a.b, a.kh), *gv = place<bf16>(p.v, a.b, a.h);
  const float* gg = place<float>(p.g, a.b, a.h);
  const uint8_t* gr = p.reset.data ? static_cast<const uint8_t*>(p.reset.data) + int64_t(a.b) * p.reset.stride[0] : nullptr;
  bf16* go = place<bf16>(p.out, a.b, a.h);
  auto tokens_of = [&](int c) { return int(min(int64_t(C), int64_t(p.tokens) - int64_t(c) * C)); };
  auto fetch_k = [&](int c) { load_tile(k, gk + int64_t(c) * C * p.k.stride[1], p.k.stride[1], dk, sg.vec & kVecK, tokens_of(c), mv); };
  auto fetch = [&](int c) {
    const int n = tokens_of(c), turn = (c - a.c0) & 1;
    GateIn<C> in{};
    if (warp == S::NW - 1) in = fetch_gates<C>(gg, p.g.stride[1], gr, p.reset.stride[1], int64_t(c) * C, n, lane);
    load_tile(q0 + turn * kTok, gq + int64_t(c) * C * p.q.stride[1], p.q.stride[1], dk, sg.vec & kVecQ, n, mv);
    load_tile(v0 + turn * kTok, gv + int64_t(c) * C * p.v.stride[1], p.v.stride[1], dv, sg.vec & kVecV, n, mv);
    if (warp == S::NW - 1) scan_gates<C>(gates[turn], in, p.g.stride[1] == 0, n, lane);
  };
  if (a.c0 < a.c1) fetch_k(a.c0), fetch(a.c0);
  begin<512>(control, warp, tid);
  const uint32_t tmem = control.tmem;
  // columns of TMEM: S^T q's and P's part of the outputs, the update, the scores
  const uint32_t t_state = tmem, t_pairs = tmem + 128, t_update = tmem + 256, t_scores = tmem + 384;
  Products products{delta::smem_at(&control.bar), 0, patience};

  const Part<S> part = part_of<S>(warp);
  float m[S::NM][2][4];
  // (of several segments the first one's is a copy too: the last one may be writing over the initial state by now)
  const float* first = a.seg || (sg.count > 1 && p.initial_state) ? sg.state + (int64_t(a.row) * sg.count + a.seg) * state_size
                       : p.initial_state                          ? p.initial_state + int64_t(a.row) * state_size
                                                                  : nullptr;
  early::wait_for_previous();
  if (first) read_state<S>(m, first, part, dk, dv, lane);
  else clear<S>(m);
  bool ok = true;

  for (int c = a.c0; c < a.c1; ++c) {
    const int64_t t0 = int64_t(c) * C;
    const int n = tokens_of(c), turn = (c - a.c0) & 1;
    plane_t *const q = q0 + turn * kTok, *const v = v0 + turn * kTok;
    const Gates<C>& s = gates[turn];
    const bool have = c > a.c0 || first, goes_on = c + 1 < a.c1 || (c + 1 == a.chunks && p.final_state);
    if (have) dump<S, 2>(m, st, part, lane);
    if (p.saved && c > 0) write_saved<S>(m, p.saved + (int64_t(a.row) * (a.chunks - 1) + c - 1) * state_size, part, dk, dv, lane, tid);
    copies_landed();
    const bool odd = tile_odd(q, mv) || tile_odd(k, mv) || tile_odd(v, mv);
    fence_shared();
    fence_before();
    const bool bad_rows = __syncthreads_or(odd);
    if (tid == 0) {
      fence_after();
      const uint32_t aq = delta::smem_at(q), ak = delta::smem_at(k);
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) mma(t_scores, along<C>(aq, kk), along<C>(ak, kk), kInstruction<64, 64, false, false>, kk > 0);
    }
    products.issued(tid == 0);
    if (c + 1 < a.c1) fetch(c + 1);
    if (goes_on) weigh(wk, k, s.to_end, 1.0f, mv);
    ok = products.done();
    if (!ok) break;

    {  // P, the masked pairs as zeros
      float acc[1][2][4];
      fetch2(&acc[0][0][0], t_scores + (uint32_t(rt * 32) << 16) + ct * 16);
      fetched(acc);
      const int i0 = rt * 16 + (lane >> 2);
      const Token ti[2] = {s.token[i0], s.token[i0 + 8]};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int col = ct * 16 + h * 8 + (lane & 3) * 2;
        const Token u0 = s.token[col], u1 = s.token[col + 1];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int i = i0 + r * 8;
          const bool m0 = meets(ti[r], u0, i, col), m1 = meets(ti[r], u1, i, col + 1);
          const float f0 = pair_decay(ti[r], u0, m0) * p.scale, f1 = pair_decay(ti[r], u1, m1) * p.scale;
          uint32_t w[2];
          split<2>(m0 ? acc[0][h][2 * r] * f0 : 0.0f, m1 ? acc[0][h][2 * r + 1] * f1 : 0.0f, w);
          const int at = spot<C>(i, col);
          *reinterpret_cast<uint32_t*>(pr + at) = w[0];
          *reinterpret_cast<uint32_t*>(pr + kPair + at) = w[1];
        }
      }
    }
    fence_shared();
    fence_before();
    __syncthreads();
    if (tid == 0) {
      fence_after();
      const uint32_t aq = delta::smem_at(q), av = delta::smem_at(v), ap = delta::smem_at(pr), as = delta::smem_at(st), aw = delta::smem_at(wk);
#pragma unroll
      for (int l = 1; l >= 0; --l)
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          mma(t_pairs, along<C>(ap + l * kPair * 2, kk), across<C>(av, kk), kInstruction<64, 128, false, true>, l == 0 || kk > 0);
      if (have) {
#pragma unroll
        for (int l = 1; l >= 0; --l)
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            mma(t_state, along<C>(aq, kk), across<D>(as + l * kState * 2, kk), kInstruction<64, 128, false, true>, l == 0 || kk > 0);
      }
      if (goes_on) {
#pragma unroll
        for (int l = 2; l >= 0; --l)
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma(t_update, across<C>(aw + l * kTok * 2, kk), across<C>(av, kk), kInstruction<128, 128, true, true>, l < 2 || kk > 0);
      }
    }
    products.issued(tid == 0);
    if (c + 1 < a.c1 && !bad_rows) fetch_k(c + 1);
    ok = products.done();
    if (!ok) break;

    const int col = ct * 32;
    float acc[2][2][4];
    fetch4(&acc[0][0][0], t_pairs + (uint32_t(rt * 32) << 16) + col);
    fetched(acc);
    if (have) {
      float more[2][2][4];
      fetch4(&more[0][0][0], t_state + (uint32_t(rt * 32) << 16) + col);
      fetched(more);
      const float f0 = s.carried[rt * 16 + (lane >> 2)], f1 = s.carried[rt * 16 + (lane >> 2) + 8];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float f = e & 2 ? f1 : f0;
          float& y = acc[j][e >> 2][e & 3];
          y = f == 0.0f ? y : fmaf(f * p.scale, more[j][e >> 2][e & 3], y);
        }
    }
    if (__syncthreads_or(not_finite(acc))) {  // (products have overflowed, where the rows are finite)
#pragma unroll 1
      for (int x = 0; x < 16; ++x) {
        const int i = rt * 16 + (lane >> 2) + ((x >> 1) & 1) * 8, cc = col + (x >> 3) * 16 + ((x >> 2) & 1) * 8 + (lane & 3) * 2 + (x & 1);
        if (i >= n || cc >= dv) continue;
        float y = 0.0f;
        if (have && s.carried[i] != 0.0f) {
          for (int d = 0; d < dk; ++d) y = fmaf(value_at<1, C>(q, 0, i, d), value_at<2, D>(st, kState, d, cc), y);
          y *= s.carried[i] * p.scale;
        }
        for (int j = 0; j <= i; ++j)
          if (pair_decay(s.token[i], s.token[j], meets(s.token[i], s.token[j], i, j)) != 0.0f)
            y = fmaf(value_at<2, C>(pr, kPair, i, j), value_at<1, C>(v, 0, j, cc), y);
#pragma unroll
        for (int z = 0; z < 16; ++z)
          if (z == x) acc[z >> 3][(z >> 2) & 1][z & 3] = y;
      }
      __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 2; ++r)
          *reinterpret_cast<uint32_t*>(pr + spot<C>(rt * 16 + (lane >> 2) + r * 8, col + j * 16 + h * 8 + (lane & 3) * 2)) =
              pack_round(acc[j][h][2 * r], acc[j][h][2 * r + 1]);
    if (goes_on) {
      if (bad_rows) merge_masked<S>(m, k, v, s.to_end, 1.0f, s.keep, n, part, lane);
      else merge<S>(m, t_update, s.keep, part);
    }
    fence_before();
    __syncthreads();
    if (bad_rows && c + 1 < a.c1) fetch_k(c + 1);
    store_tile(go + t0 * p.out.stride[1], p.out.stride[1], pr, dv, sg.vec & kVecOut, n, mv);
  }
  copies_landed();
  if (!ok) {  // what this block would have written
    for (int64_t t = int64_t(a.c0) * C + warp; t < min(int64_t(a.c1) * C, int64_t(p.tokens)); t += S::NW)
      for (int x = lane; x < dv; x += 32) go[t * p.out.stride[1] + x] = __float2bfloat16_rn(lost());
#pragma unroll
    for (int j = 0; j < S::NM; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) m[j][e >> 2][e & 3] = lost();
    if (p.saved)
      for (int c = max(a.c0, 1); c < a.c1; ++c)
        write_state<S>(m, p.saved + (int64_t(a.row) * (a.chunks - 1) + c - 1) * state_size, part, dk, dv, lane);
  }
  if (a.c1 == a.chunks && p.final_state) write_state<S>(m, p.final_state + int64_t(a.row) * state_size, part, dk, dv, lane);
  end<512>(tmem, warp);
}

// What each segment adds to the state behind it, as linear_segment_kernel.  The next chunk is fetched while a chunk's products run (X, whose limbs
// they read, into its own tile).
template <class S>
__global__ void __launch_bounds__(S::THREADS, 2)
linear_tensor_segment_kernel(const __grid_constant__ ZenoLinearAttention p, const ZenoTensor tx, const ZenoTensor ty, const Segments sg, const bool reverse,
                             const uint64_t patience) {
  extern __shared__ char smem[];
  plane_t* const x = reinterpret_cast<plane_t*>((reinterpret_cast<uintptr_t>(smem) + 1023) / 1024 * 1024);
  plane_t *const y0 = x + kTok, *const wx = y0 + 2 * kTok;
  Gates<C>* const gates = reinterpret_cast<Gates<C>*>(wx + 3 * kTok);
  Control& control = *reinterpret_cast<Control*>(gates + 2);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int dk = S::FULL ? D : int(p.key_dim), dv = S::FULL ? D : int(p.value_dim);
  const At a = block_at(p, sg, reverse ? 1 : 0, C);
  const Mover<S::THREADS> mv(tid);
  const bf16 *gx = place<bf16>(tx, a.b, a.kh), *gy = place<bf16>(ty, a.b, a.h);
  const float* gg = place<float>(p.g, a.b, a.h);
  const uint8_t* gr = p.reset.data ? static_cast<const uint8_t*>(p.reset.data) + int64_t(a.b) * p.reset.stride[0] : nullptr;
  const bool vx = sg.vec & (reverse ? kVecQ : kVecK), vy = sg.vec & (reverse ? kVecOut : kVecV);
  const int steps = a.c1 - a.c0;
  auto fetch = [&](int step) {
    const int64_t t0 = int64_t(reverse ? a.c1 - 1 - step : a.c0 + step) * C;
    const int n = int(min(int64_t(C), int64_t(p.tokens) - t0));
    GateIn<C> in{};
    if (warp == S::NW - 1) in = fetch_gates<C>(gg, p.g.stride[1], gr, p.reset.stride[1], t0, n, lane);
    load_tile(x, gx + t0 * tx.stride[1], tx.stride[1], dk, vx, n, mv);
    load_tile(y0 + (step & 1) * kTok, gy + t0 * ty.stride[1], ty.stride[1], dv, vy, n, mv);
    if (warp == S::NW - 1) scan_gates<C>(gates[step & 1], in, p.g.stride[1] == 0, n, lane);
  };
  fetch(0);
  begin<128>(control, warp, tid);
  const uint32_t tmem = control.tmem;
  Products products{delta::smem_at(&control.bar), 0, patience};
  const Part<S> part = part_of<S>(warp);
  float m[S::NM][2][4];
  clear<S>(m);
  float kept = 1.0f;
  early::let_next_start();
  bool ok = true;
  for (int step = 0; step < steps; ++step) {
    const Gates<C>& s = gates[step & 1];
    const plane_t* y = y0 + (step & 1) * kTok;
    const float* weight = reverse ? s.carried : s.to_end;
    const float factor = reverse ? p.scale : 1.0f;
    copies_landed();
    const bool bad = __syncthreads_or(tile_odd(x, mv) || tile_odd(y, mv));
    const float keep = step ? s.keep : 0.0f;
    kept = both_keep(kept, s.keep);
    if (bad) {
      const int64_t t0 = int64_t(reverse ? a.c1 - 1 - step : a.c0 + step) * C;
      merge_masked<S>(m, x, y, weight, factor, keep, int(min(int64_t(C), int64_t(p.tokens) - t0)), part, lane);
      __syncthreads();
      if (step + 1 < steps) fetch(step + 1);
      continue;
    }
    weigh(wx, x, weight, factor, mv);
    fence_shared();
    fence_before();
    __syncthreads();
    if (tid == 0) {
      fence_after();
      const uint32_t aw = delta::smem_at(wx), ay = delta::smem_at(y);
#pragma unroll
      for (int l = 2; l >= 0; --l)
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          mma(tmem, across<C>(aw + l * kTok * 2, kk), across<C>(ay, kk), kInstruction<128, 128, true, true>, l < 2 || kk > 0);
    }
    products.issued(tid == 0);
    if (step + 1 < steps) fetch(step + 1);
    ok = products.done();
    if (!ok) break;
    merge<S>(m, tmem, keep, part);
    fence_before();
  }
  copies_landed();
  if (!ok) {
#pragma unroll
    for (int j = 0; j < S::NM; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) m[j][e >> 2][e & 3] = lost();
  }
  const int64_t at = int64_t(a.row) * sg.count + a.seg;
  write_state<S>(m, sg.state + at * dk * dv, part, dk, dv, lane);
  if (tid == 0) sg.keep[at] = ok ? kept : lost();
  end<128>(tmem, warp);
}

// ---------------------------------------------------------------- gradients
struct BackwardSums {
  float x[4][C], y[4][C];  // x_i and y_j over each quarter of the columns
  float pairs[4][C];       // sum over the rows of a tile i >= t of the A_ij in front of t in t's quarter
  float row[4][C];         // sum of A_ij over each quarter
  float state[16];         // <S, R> over each warp's part
};
constexpr int kBackwardBytes =
    1024 + 2 * (4 * kTok + 4 * kPair + 3 * kState) + int(sizeof(Gates<C>)) + int(sizeof(BackwardSums)) + int(sizeof(Control));

// acc = acc + f[i] scale more (what f is zero for is left out).  Returns the products of that with the lane's two rows of X over its columns.
__device__ __forceinline__ float2 add_and_dot(float (&acc)[2][2][4], const float (&more)[2][2][4], const float* f, float scale, const plane_t* x, int rt,
                                              int col, int lane) {
  const int i0 = rt * 16 + (lane >> 2);
  const float f0 = f[i0], f1 = f[i0 + 8], s0 = f0 * scale, s1 = f1 * scale;
  float d0 = 0.0f, d1 = 0.0f;
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int at = col + j * 16 + h * 8 + (lane & 3) * 2;
      const uint32_t w0 = *reinterpret_cast<const uint32_t*>(x + spot<C>(i0, at)), w1 = *reinterpret_cast<const uint32_t*>(x + spot<C>(i0 + 8, at));
      float y[4];
      y[0] = f0 == 0.0f ? 0.0f : more[j][h][0] * s0, y[1] = f0 == 0.0f ? 0.0f : more[j][h][1] * s0;
      y[2] = f1 == 0.0f ? 0.0f : more[j][h][2] * s1, y[3] = f1 == 0.0f ? 0.0f : more[j][h][3] * s1;
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][h][e] += y[e];
      d0 = fmaf(lower(w0), y[0], fmaf(upper(w0), y[1], d0)), d1 = fmaf(lower(w1), y[2], fmaf(upper(w1), y[3], d1));
    }
  return make_float2(f0 == 0.0f ? 0.0f : d0, f1 == 0.0f ? 0.0f : d1);
}

// One element of a gradient over the pairs that the mask leaves (ROWS: of a query's): pairs with y's column, after `sum` from the state.
template <bool ROWS>
__device__ __noinline__ float over_pairs(const Gates<C>& s, float sum, const plane_t* pairs, const plane_t* y, int at, int col, int n) {
  for (int o = ROWS ? 0 : at; o < (ROWS ? at + 1 : n); ++o) {
    const int i = ROWS ? at : o, j = ROWS ? o : at;
    if (pair_decay(s.token[i], s.token[j], meets(s.token[i], s.token[j], i, j)) != 0.0f)
      sum = fmaf(value_at<2, C>(pairs, kPair, i, j), value_at<1, C>(y, 0, o, col), sum);
  }
  return sum;
}
template <class F>
__device__ __forceinline__ void again(float (&acc)[2][2][4], int rt, int col, int n, int width, int lane, F&& element) {
#pragma unroll 1
  for (int x = 0; x < 16; ++x) {
    const int i = rt * 16 + (lane >> 2) + ((x >> 1) & 1) * 8, c = col + (x >> 3) * 16 + ((x >> 2) & 1) * 8 + (lane & 3) * 2 + (x & 1);
    if (i >= n || c >= width) continue;
    const float y = element(i, c);
#pragma unroll
    for (int z = 0; z < 16; ++z)
      if (z == x) acc[z >> 3][(z >> 2) & 1][z & 3] = y;
  }
}
__device__ __forceinline__ void stage_tile(plane_t* to, const float (&acc)[2][2][4], int rt, int col, int lane) {
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int r = 0; r < 2; ++r)
        *reinterpret_cast<uint32_t*>(to + spot<C>(rt * 16 + (lane >> 2) + r * 8, col + j * 16 + h * 8 + (lane & 3) * 2)) =
            pack_round(acc[j][h][2 * r], acc[j][h][2 * r + 1]);
}

// 32-bit rows of 128 values in shared memory, their 16-byte pieces swapped within groups of 8 rows; to rows in memory.
__device__ __forceinline__ int float_spot(int row, int col) { return row * D + (((col >> 2) ^ (row & 7)) << 2) + (col & 3); }
__device__ __forceinline__ void stage_float(float* to, const float (&acc)[2][2][4], int rt, int col, int lane) {
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int r = 0; r < 2; ++r)
        *reinterpret_cast<float2*>(to + float_spot(rt * 16 + (lane >> 2) + r * 8, col + j * 16 + h * 8 + (lane & 3) * 2)) =
            make_float2(acc[j][h][2 * r], acc[j][h][2 * r + 1]);
}
__device__ __forceinline__ void store_staged(float* to, int64_t stride, const float* from, int width, int n, int tid) {
  const int c = (tid & 31) * 4;
  if (c >= width) return;
  const bool four = width % 4 == 0;  // (and then the workspace's rows are whole vectors)
  for (int row = tid >> 5; row < n; row += 16) {
    const float4 x = *reinterpret_cast<const float4*>(from + float_spot(row, c));
    float* at = to + row * stride + c;
    if (four) {
      *reinterpret_cast<float4*>(at) = x;
    } else {
      at[0] = x.x;
      if (c + 1 < width) at[1] = x.y;
      if (c + 2 < width) at[2] = x.z;
      if (c + 3 < width) at[3] = x.w;
    }
  }
}

// As linear_backward_kernel.  Four rounds of products a chunk: the scores and S's part of dQ; all that P and D are in, while R's limbs take the
// place of S's; R's part of dK and dV; the update of R, whose weighted queries take the place of its limbs.
template <class S>
__global__ void __launch_bounds__(S::THREADS, 1)
linear_tensor_backward_kernel(const __grid_constant__ ZenoLinearAttention p, const __grid_constant__ ZenoLinearAttentionGrads d, const Segments sg,
                              const BackwardOut extra, const uint64_t patience) {
  extern __shared__ char smem[];
  plane_t* const q = reinterpret_cast<plane_t*>((reinterpret_cast<uintptr_t>(smem) + 1023) / 1024 * 1024);
  plane_t *const k = q + kTok, *const v = k + kTok, *const o = v + kTok, *const pr = o + kTok, *const dp = pr + 2 * kPair, *const st = dp + 2 * kPair;
  Gates<C>& s = *reinterpret_cast<Gates<C>*>(st + 3 * kState);
  BackwardSums& sums = *reinterpret_cast<BackwardSums*>(&s + 1);
  Control& control = *reinterpret_cast<Control*>(&sums + 1);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rt = warp & 3, ct = warp >> 2, col = ct * 32;
  const int dk = S::FULL ? D : int(p.key_dim), dv = S::FULL ? D : int(p.value_dim);
  const At a = block_at(p, sg, 0, C);
  if (a.b >= p.batch) return;
  const Mover<S::THREADS> mv(tid);
  const int64_t state_size = int64_t(dk) * dv;
  const bool shared = extra.shared_q != nullptr;
  const bf16 *gq = place<bf16>(p.q, a.b, a.kh), *gk = place<bf16>(p.k, a.b, a.kh), *gv = place<bf16>(p.v, a.b, a.h), *go = place<bf16>(d.d_out, a.b, a.h);
  const float* gg = place<float>(p.g, a.b, a.h);
  const uint8_t* gr = p.reset.data ? static_cast<const uint8_t*>(p.reset.data) + int64_t(a.b) * p.reset.stride[0] : nullptr;
  bf16 *wq = place<bf16>(d.d_q, a.b, a.kh), *wk = place<bf16>(d.d_k, a.b, a.kh), *wv = place<bf16>(d.d_v, a.b, a.h);
  const int64_t shared_stride = int64_t(p.value_heads) * dk;
  begin<512>(control, warp, tid);
  const uint32_t tmem = control.tmem, quarter = uint32_t(rt * 32) << 16;
  // regions of 128 columns: scores, then P's part of dV, then the update; S's part of dQ, then R's of dK; D's part of dQ, then R's of dV; D's of dK
  const uint32_t t0_ = tmem, t1_ = tmem + 128, t2_ = tmem + 256, t3_ = tmem + 384;
  Products products{delta::smem_at(&control.bar), 0, patience};
  const uint32_t aq = delta::smem_at(q), ak = delta::smem_at(k), av = delta::smem_at(v), ao = delta::smem_at(o), ap = delta::smem_at(pr),
                 ad = delta::smem_at(dp), as = delta::smem_at(st);

  float *const sq = reinterpret_cast<float*>(k), *const sk = reinterpret_cast<float*>(st + 3 * kTok);
  const Part<S> part = part_of<S>(warp);
  float m[S::NM][2][4];
  const bool last_segment = a.c1 == a.chunks;
  const float* behind = !last_segment ? sg.state + (int64_t(a.row) * sg.count + a.seg) * state_size
                                      : d.d_final ? d.d_final + int64_t(a.row) * state_size : nullptr;
  early::wait_for_previous();
  if (behind) read_state<S>(m, behind, part, dk, dv, lane);
  else clear<S>(m);
  const bool each = d.d_g.data != nullptr;  // every token's decay has a gradient of its own
  double decay_sum = 0.0;
  bool ok = true;

  for (int c = a.c1 - 1; c >= a.c0; --c) {
    const int64_t t0 = int64_t(c) * C;
    const int n = int(min(int64_t(C), int64_t(p.tokens) - t0));
    const float* front = c > 0 ? p.saved + (int64_t(a.row) * (a.chunks - 1) + c - 1) * state_size
                               : p.initial_state ? p.initial_state + int64_t(a.row) * state_size : nullptr;
    const bool have_r = c + 1 < a.c1 || behind, goes_on = c > a.c0 || (c == 0 && d.d_initial);
    GateIn<C> in{};
    if (warp == S::NW - 1) in = fetch_gates<C>(gg, p.g.stride[1], gr, p.reset.stride[1], t0, n, lane);
    __syncthreads();  // the last chunk's results have left
    load_tile(q, gq + t0 * p.q.stride[1], p.q.stride[1], dk, sg.vec & kVecQ, n, mv);
    load_tile(k, gk + t0 * p.k.stride[1], p.k.stride[1], dk, sg.vec & kVecK, n, mv);
    load_tile(v, gv + t0 * p.v.stride[1], p.v.stride[1], dv, sg.vec & kVecV, n, mv);
    load_tile(o, go + t0 * d.d_out.stride[1], d.d_out.stride[1], dv, sg.vec & kVecOut, n, mv);
    if (warp == S::NW - 1) scan_gates<C>(s, in, p.g.stride[1] == 0, n, lane);
    float state_dot = 0.0f;  // <S, R> over this thread's elements
    if (front) {
      float x[S::NM][2][4];
      if (c > 0) read_saved<S>(x, front, part, dk, dv, lane, tid);
      else read_state<S>(x, front, part, dk, dv, lane);
      float dot = 0.0f;
#pragma unroll
      for (int j = 0; j < S::NM; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) dot = fmaf(x[j][e >> 2][e & 3], m[j][e >> 2][e & 3], dot);
      dump<S, 3>(x, st, part, lane);
      state_dot = have_r ? dot : 0.0f;
      if (each) {
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) dot += __shfl_xor_sync(kAll, dot, x);
        if (lane == 0) sums.state[warp] = dot;
      }
    }
    copies_landed();
    const bool odd = tile_odd(q, mv) || tile_odd(o, mv);
    fence_shared();
    fence_before();
    const bool bad_rows = __syncthreads_or(odd);  // (of the update's)
    if (tid == 0) {
      fence_after();
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) mma(t0_, along<C>(aq, kk), along<C>(ak, kk), kInstruction<64, 64, false, false>, kk > 0);
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) mma(t0_ + 64, along<C>(ao, kk), along<C>(av, kk), kInstruction<64, 64, false, false>, kk > 0);
      if (front) {
#pragma unroll
        for (int l = 2; l >= 0; --l)
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            mma(t1_, along<C>(ao, kk), along<D>(as + l * kState * 2, kk), kInstruction<64, 128, false, false>, l < 2 || kk > 0);
      }
    }
    products.issued(tid == 0);
    ok = products.done();
    if (!ok) break;

    // P, D, and what the pairs give the decays: this thread's part of their gradient, where all tokens of the head have one
    float decays = each || s.keep == 0.0f ? 0.0f : state_dot * s.keep * float(n);
    {
      float sp[1][2][4], so[1][2][4];
      fetch2(&sp[0][0][0], t0_ + quarter + ct * 16);
      fetch2(&so[0][0][0], t0_ + quarter + 64 + ct * 16);
      fetched(sp);
      fetched(so);
      const int i0 = rt * 16 + (lane >> 2);
      const Token ti[2] = {s.token[i0], s.token[i0 + 8]};
      float before[2] = {0.0f, 0.0f};  // of the quarter's columns so far, for each of the lane's two rows
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int cc = ct * 16 + h * 8 + (lane & 3) * 2;
        const Token u0 = s.token[cc], u1 = s.token[cc + 1];
        float pass[2][2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int i = i0 + r * 8, at = spot<C>(i, cc);
          const bool m0 = meets(ti[r], u0, i, cc), m1 = meets(ti[r], u1, i, cc + 1);
          const float f0 = pair_decay(ti[r], u0, m0) * p.scale, f1 = pair_decay(ti[r], u1, m1) * p.scale;
          const float o0 = so[0][h][2 * r], o1 = so[0][h][2 * r + 1];
          const float p0 = m0 ? sp[0][h][2 * r] * f0 : 0.0f, p1 = m1 ? sp[0][h][2 * r + 1] * f1 : 0.0f;
          uint32_t w[2];
          split<2>(p0, p1, w);
          *reinterpret_cast<uint32_t*>(pr + at) = w[0], *reinterpret_cast<uint32_t*>(pr + kPair + at) = w[1];
          split<2>(m0 ? o0 * f0 : 0.0f, m1 ? o1 * f1 : 0.0f, w);
          *reinterpret_cast<uint32_t*>(dp + at) = w[0], *reinterpret_cast<uint32_t*>(dp + kPair + at) = w[1];
          // (a token with itself passes none: where it is not finite that is not zero times it)
          pass[r][0] = m0 && i != cc ? p0 * o0 : 0.0f, pass[r][1] = m1 && i != cc + 1 ? p1 * o1 : 0.0f;
        }
        if (!each) {  // a pair passes i - j tokens
          const float far = float(i0 - cc);
          decays = fmaf(pass[0][0], far, fmaf(pass[0][1], far - 1.0f, fmaf(pass[1][0], far + 8.0f, fmaf(pass[1][1], far + 7.0f, decays))));
          continue;
        }
        float passes[2] = {0.0f, 0.0f};  // tokens cc and cc + 1, over the lane's rows
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int i = i0 + r * 8;
          float sum = pass[r][0] + pass[r][1];
          const float x1 = __shfl_up_sync(kAll, sum, 1, 4);
          if ((lane & 3) >= 1) sum += x1;
          const float x2 = __shfl_up_sync(kAll, sum, 2, 4);
          if ((lane & 3) >= 2) sum += x2;
          float left = __shfl_up_sync(kAll, sum, 1, 4);
          left = (lane & 3) ? before[r] + left : before[r];
          before[r] += __shfl_sync(kAll, sum, 3, 4);
          if (i >= cc) passes[0] += left;
          if (i >= cc + 1) passes[1] += left + pass[r][0];
        }
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
          passes[0] += __shfl_xor_sync(kAll, passes[0], x);
          passes[1] += __shfl_xor_sync(kAll, passes[1], x);
        }
        if (lane < 4) sums.pairs[rt][cc] = passes[0], sums.pairs[rt][cc + 1] = passes[1];
      }
      if (each && (lane & 3) == 0) sums.row[ct][i0] = before[0], sums.row[ct][i0 + 8] = before[1];
    }
    fence_shared();
    fence_before();
    __syncthreads();
    if (tid == 0) {
      fence_after();
#pragma unroll
      for (int l = 1; l >= 0; --l)
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          mma(t2_, along<C>(ad + l * kPair * 2, kk), across<C>(ak, kk), kInstruction<64, 128, false, true>, l == 0 || kk > 0);
          mma(t3_, across<C>(ad + l * kPair * 2, kk), across<C>(aq, kk), kInstruction<64, 128, true, true>, l == 0 || kk > 0);
          mma(t0_, across<C>(ap + l * kPair * 2, kk), across<C>(ao, kk), kInstruction<64, 128, true, true>, l == 0 || kk > 0);
        }
    }
    products.issued(tid == 0);
    if (c > a.c0) {  // the next chunk's rows, a line of 128 bytes a thread, and the state in front of it
      const int row = tid >> 3, half = (tid & 1) * 64;
      const int64_t t = t0 - C + row;
      const int which = tid >> 1 & 3;
      const bf16* at = which == 0 ? gq + t * p.q.stride[1] : which == 1 ? gk + t * p.k.stride[1] : which == 2 ? gv + t * p.v.stride[1]
                                                                                                             : go + t * d.d_out.stride[1];
      if (half < (which < 2 ? dk : dv)) delta::prefetch(at + half);
      const float* next = c > 1 ? front - state_size : p.initial_state ? p.initial_state + int64_t(a.row) * state_size : nullptr;
      if (next && tid * 32 < state_size) delta::prefetch(next + tid * 32);
    }
    if (have_r) {  // (S's limbs have been read)
      dump<S, 3>(m, st, part, lane);
      fence_shared();
    }
    ok = products.done();
    if (!ok) break;

    float dq[2][2][4], dk_[2][2][4], dv_[2][2][4];
    fetch4(&dq[0][0][0], t2_ + quarter + col);
    fetch4(&dk_[0][0][0], t3_ + quarter + col);
    fetch4(&dv_[0][0][0], t0_ + quarter + col);
    if (front) {
      float more[2][2][4];
      fetch4(&more[0][0][0], t1_ + quarter + col);
      fetched(more);
      fetched(dq);
      const float2 x = add_and_dot(dq, more, s.carried, p.scale, q, rt, col, lane);
      const float i = float(rt * 16 + (lane >> 2));
      if (each) keep_rows(sums.x[ct], x, rt, lane);
      else decays = fmaf(x.x, i + 1.0f, fmaf(x.y, i + 9.0f, decays));  // the state in front passes every token up to this one
    }
    fetched(dq), fetched(dk_), fetched(dv_);
    fence_before();
    __syncthreads();
    if (have_r) {
      if (tid == 0) {
        fence_after();
#pragma unroll
        for (int l = 2; l >= 0; --l)
#pragma unroll
          for (int kk = 0; kk < 8; ++kk) {
            mma(t1_, along<C>(av, kk), along<D>(as + l * kState * 2, kk), kInstruction<64, 128, false, false>, l < 2 || kk > 0);
            if (l < 2) mma(t2_, along<C>(ak, kk), across<D>(as + l * kState * 2, kk), kInstruction<64, 128, false, true>, l == 0 || kk > 0);
          }
      }
      products.issued(tid == 0);
      ok = products.done();
      if (!ok) break;
      float more[2][2][4];
      fetch4(&more[0][0][0], t1_ + quarter + col);
      fetched(more);
      const float2 y = add_and_dot(dk_, more, s.to_end, 1.0f, k, rt, col, lane);
      const float rest = float(n - 1 - rt * 16 - (lane >> 2));
      if (each) keep_rows(sums.y[ct], y, rt, lane);
      else decays += (rest == 0.0f ? 0.0f : y.x * rest) + (rest == 8.0f ? 0.0f : y.y * (rest - 8.0f));  // what begins here passes the tokens behind it
      fetch4(&more[0][0][0], t2_ + quarter + col);
      fetched(more);
      const float e0 = s.to_end[rt * 16 + (lane >> 2)], e1 = s.to_end[rt * 16 + (lane >> 2) + 8];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          float& z = dv_[j][x >> 2][x & 3];
          const float e = x & 2 ? e1 : e0;
          z = e == 0.0f ? z : fmaf(e, more[j][x >> 2][x & 3], z);
        }
    }
    decay_sum += double(decays);
    if (__syncthreads_or(not_finite(dq) || not_finite(dk_) || not_finite(dv_))) {
      again(dq, rt, col, n, dk, lane, [&](int i, int cc) {
        float y = 0.0f;
        if (front && s.carried[i] != 0.0f) {
          for (int e = 0; e < dv; ++e) y = fmaf(value_at<1, C>(o, 0, i, e), saved_value<S>(front, c > 0, cc, e, dv), y);
          y *= s.carried[i] * p.scale;
        }
        return over_pairs<true>(s, y, dp, k, i, cc, n);
      });
      again(dk_, rt, col, n, dk, lane, [&](int j, int cc) {
        float y = 0.0f;
        if (have_r && s.to_end[j] != 0.0f) {
          for (int e = 0; e < dv; ++e) y = fmaf(value_at<1, C>(v, 0, j, e), value_at<3, D>(st, kState, cc, e), y);
          y *= s.to_end[j];
        }
        return over_pairs<false>(s, y, dp, q, j, cc, n);
      });
      again(dv_, rt, col, n, dv, lane, [&](int j, int cc) {
        float y = 0.0f;
        if (have_r && s.to_end[j] != 0.0f) {
          for (int e = 0; e < dk; ++e) y = fmaf(value_at<1, C>(k, 0, j, e), value_at<3, D>(st, kState, e, cc), y);
          y *= s.to_end[j];
        }
        return over_pairs<false>(s, y, pr, o, j, cc, n);
      });
      __syncthreads();
    }
    if (goes_on && !bad_rows) {
      weigh(st, q, s.carried, p.scale, mv);
      fence_shared();
      fence_before();
      __syncthreads();
      if (tid == 0) {
        fence_after();
#pragma unroll
        for (int l = 2; l >= 0; --l)
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma(t0_, across<C>(as + l * kTok * 2, kk), across<C>(ao, kk), kInstruction<128, 128, true, true>, l < 2 || kk > 0);
      }
      products.issued(tid == 0);
    }
    // results by way of tiles that are not needed any more (Q and dO still are)
    if (shared) {
      // (32-bit rows where K and V, and the rest of the limbs, were)
      stage_float(sq, dq, rt, col, lane);
      stage_float(sk, dk_, rt, col, lane);
    } else {
      stage_tile(k, dq, rt, col, lane);
      stage_tile(v, dk_, rt, col, lane);
    }
    stage_tile(pr, dv_, rt, col, lane);
    if (each && warp == S::NW - 1) {
      // the decays: neighbouring tokens 2 lane and 2 lane + 1
      float z = 0.0f;
      if (front && have_r && s.keep != 0.0f) {
        for (int w = 0; w < S::NW; ++w) z += sums.state[w];
        z *= s.keep;
      }
      float dg[2], here[2] = {0.0f, 0.0f}, ahead[2] = {0.0f, 0.0f};  // what ends at this token; what begins at it
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int t = lane * 2 + u;
        dg[u] = z;
        if (t < n) {
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            if (front) here[u] += sums.x[x][t];
            if (have_r) ahead[u] += sums.y[x][t];
          }
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (r * 16 + 15 >= t) dg[u] += sums.pairs[r][t];
        }
      }
      // sums over the tokens in front, and from this one on: x_i, and pairs whose first token lies in an earlier quarter of the columns
      float in_front = ahead[0] + ahead[1];
#pragma unroll
      for (int x = 1; x < 32; x <<= 1) {
        const float y = __shfl_up_sync(kAll, in_front, x);
        if (lane >= x) in_front += y;
      }
      in_front = __shfl_up_sync(kAll, in_front, 1);
      if (lane == 0) in_front = 0.0f;
      dg[0] += in_front, dg[1] += in_front + ahead[0];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float rest[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) rest[u] = g == 3 ? here[u] : lane * 2 + u < n ? sums.row[g][lane * 2 + u] : 0.0f;
        float sum = rest[0] + rest[1];
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) {
          const float y = __shfl_down_sync(kAll, sum, x);
          if (lane + x < 32) sum += y;
        }
        float from = __shfl_down_sync(kAll, sum, 1);
        if (lane == 31) from = 0.0f;
        if (g == 3 || lane * 2 >= (g + 1) * 16) {  // (both tokens of a lane are in one quarter)
          dg[1] += from + rest[1];
          dg[0] += from + rest[1] + rest[0];
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int t = lane * 2 + u;
        if (t < n) {
          decay_sum += double(dg[u]);
          place<float>(d.d_g, a.b, a.h)[(t0 + t) * d.d_g.stride[1]] = dg[u];
        }
      }
    }
    if (goes_on) {
      if (bad_rows) {
        merge_masked<S>(m, q, o, s.carried, p.scale, s.keep, n, part, lane);
      } else {
        ok = products.done();
        if (!ok) break;
        merge<S>(m, t0_, s.keep, part);
      }
    }
    fence_before();
    __syncthreads();
    if (shared) {
      const int64_t at = (int64_t(a.b) * p.tokens + t0) * shared_stride + int64_t(a.h) * dk;
      store_staged(extra.shared_q + at, shared_stride, sq, dk, n, tid);
      store_staged(extra.shared_k + at, shared_stride, sk, dk, n, tid);
    } else {
      store_tile(wq + t0 * d.d_q.stride[1], d.d_q.stride[1], k, dk, sg.vec & kVecDq, n, mv);
      store_tile(wk + t0 * d.d_k.stride[1], d.d_k.stride[1], v, dk, sg.vec & kVecDk, n, mv);
    }
    store_tile(wv + t0 * d.d_v.stride[1], d.d_v.stride[1], pr, dv, sg.vec & kVecDv, n, mv);
  }
  if (!ok) {  // what this block would have written
    for (int64_t t = int64_t(a.c0) * C + warp; t < min(int64_t(a.c1) * C, int64_t(p.tokens)); t += S::NW) {
      for (int x = lane; x < max(dk, dv); x += 32) {
        if (x < dv) wv[t * d.d_v.stride[1] + x] = __float2bfloat16_rn(lost());
        if (x >= dk) continue;
        if (shared) {
          const int64_t at = (int64_t(a.b) * p.tokens + t) * shared_stride + int64_t(a.h) * dk + x;
          extra.shared_q[at] = extra.shared_k[at] = lost();
        } else {
          wq[t * d.d_q.stride[1] + x] = __float2bfloat16_rn(lost()), wk[t * d.d_k.stride[1] + x] = __float2bfloat16_rn(lost());
        }
      }
      if (each && lane == 0) place<float>(d.d_g, a.b, a.h)[t * d.d_g.stride[1]] = lost();
    }
#pragma unroll
    for (int j = 0; j < S::NM; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) m[j][e >> 2][e & 3] = lost();
    decay_sum = double(lost());
  }
  if (a.c0 == 0 && d.d_initial) write_state<S>(m, d.d_initial + int64_t(a.row) * state_size, part, dk, dv, lane);
  if (extra.decay) {
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) decay_sum += __shfl_xor_sync(kAll, decay_sum, x);
    double* part_sum = reinterpret_cast<double*>(&s);  // (where the gates were)
    __syncthreads();
    if (lane == 0) part_sum[warp] = decay_sum;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < S::NW; ++w) decay_sum += part_sum[w];
      extra.decay[(uint64_t(a.h) * p.batch + a.b) * sg.count + a.seg] = decay_sum;
    }
  }
  end<512>(tmem, warp);
}

}  // namespace tensor
}  // namespace linear
}  // namespace zb
