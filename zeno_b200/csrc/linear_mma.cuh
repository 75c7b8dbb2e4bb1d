// Building blocks of the chunked linear attention with decays: the chunk's rows in shared memory, matrix
// products on split operands, the gates of a chunk, and the state in the warps' accumulators.
//
// Precision.  The matrix instructions take bfloat16 operands and sum in 32 bits.  bfloat16 inputs enter as
// they are.  A 32-bit value x enters as limbs of 8 bits each: hi = x rounded to bfloat16, then the same of what
// is left; three limbs are x exactly, and since a bfloat16 has the exponents of a float nothing is scaled and
// nothing leaves the range (what would round to infinity is the largest bfloat16 and the rest).  What ends in a 32-bit result (the states, the decays' gradient, all of a 32-bit call)
// takes three limbs, products of two such values the six terms above 2^-25.  What ends in a bfloat16 result (P in
// out and dV, dP in dQ and dK of a bfloat16 call) takes two: 2^-17 of the value against the result's 2^-8.
// The instructions' sums truncate, so the state is not summed in them: each chunk's contribution is, and
// is added to the state by an ordinary multiply-add.
//
// Not finite values.  A masked pair is a product with zero, which an infinity or a NaN would leave the mask through.
// Every present token meets itself, so such an input leaves a result that is not finite; where a chunk has one,
// its results are taken again element by element over the pairs that the mask leaves.
#pragma once
#include <cuda_bf16.h>

#include <cstdint>
#include <type_traits>

#include "delta_mma.cuh"
#include "policy_ops.h"

namespace zb {
namespace linear {

using delta::kAll;
using bf16 = __nv_bfloat16;
using plane_t = uint16_t;  // bfloat16 bits

// D: the widths of a head, padded.  C: tokens of a chunk.  NW: warps.  The warps lie over a chunk's products as
// [C / 16 row tiles][NH groups of columns] and over the state as [D / 16 row tiles][MG groups of columns].
// FULL: keys and values have D channels each, so that offsets are known and no column is past an end.
template <class T_, int D_, int C_, int NW_, bool FULL_>
struct Shape {
  using T = T_;
  static constexpr bool FULL = FULL_;
  static constexpr int D = D_, C = C_, NW = NW_, THREADS = NW_ * 32;
  static constexpr int L = sizeof(T) == 2 ? 1 : 3;   // limbs of an input
  static constexpr int PL = sizeof(T) == 2 ? 2 : 3;  // limbs of P and dP
  static constexpr int P = D + 8, PLANE = C * P;     // rows 16 bytes apart in banks
  static constexpr int CP = C + 8, CPLANE = C * CP;
  static constexpr int SPLANE = D * P;
  static constexpr int RT = C / 16, NH = NW / RT, NHS = NH < RT ? NH : RT, SP = RT / NHS;
  static constexpr int NO = D / NH / 16;  // pairs of 8 columns of a warp's part of a product
  static constexpr int MR = D / 16, MG = NW / MR, NM = D / MG / 16;
  static_assert(NW % RT == 0 && NW % MR == 0 && NO >= 1 && NM >= 1 && SP >= 1);
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {  // d = a b
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

// Fragments of a 16 x 16 operand in shared memory, as in delta_mma.cuh.  TR: stored with the contracted axis first.
template <bool TR>
__device__ __forceinline__ void frag_a(uint32_t (&r)[4], const plane_t* at, int pitch, int lane) {
  if (TR) delta::ldsm4t(r, delta::smem_at(at + ((lane >> 4) * 8 + (lane & 7)) * pitch + ((lane >> 3) & 1) * 8));
  else delta::ldsm4(r, delta::smem_at(at + (lane & 15) * pitch + (lane >> 4) * 8));
}
template <bool TR>
__device__ __forceinline__ void frag_b(uint32_t (&r)[4], const plane_t* at, int pitch, int lane) {
  if (TR) delta::ldsm4t(r, delta::smem_at(at + (lane & 15) * pitch + (lane >> 4) * 8));
  else delta::ldsm4(r, delta::smem_at(at + ((lane >> 4) * 8 + (lane & 7)) * pitch + ((lane >> 3) & 1) * 8));
}

__device__ __forceinline__ float cut(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }
__device__ __forceinline__ uint32_t pack_cut(float x, float y) {  // the upper halves: x low, y high
  return __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
}
__device__ __forceinline__ uint32_t pack_round(float x, float y) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// The same, of infinities and what would round to one the largest bfloat16 (the rest is the second limb's: an infinity, or what is left).
__device__ __forceinline__ uint32_t pack_near(float x, float y) {
  uint32_t w;
  asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(y), "f"(x));
  return w;
}
__device__ __forceinline__ float lower(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float upper(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
// Two values as N packed limbs, each the rounding of what is left; three are exact, two leave 2^-17 of the value.
template <int N>
__device__ __forceinline__ void split(float x, float y, uint32_t (&r)[N]) {
  if constexpr (N == 1) {
    r[0] = pack_round(x, y);
  } else {
    r[0] = pack_near(x, y);
    x -= lower(r[0]), y -= upper(r[0]);
    r[1] = pack_round(x, y);
    if constexpr (N == 3) r[2] = pack_cut(x - lower(r[1]), y - upper(r[1]));  // (six bits are left)
  }
}

// The value that N planes hold at `at`; no further than a limb that is not finite.
template <int N>
__device__ __forceinline__ float value(const plane_t* at, int plane) {
  float x = __uint_as_float(uint32_t(at[0]) << 16);
#pragma unroll
  for (int l = 1; l < N; ++l)
    if (fabsf(x) < INFINITY) x += __uint_as_float(uint32_t(at[l * plane]) << 16);
  return x;
}
// Two neighbouring ones.
template <int N>
__device__ __forceinline__ float2 values(const plane_t* at, int plane) {
  uint32_t w = *reinterpret_cast<const uint32_t*>(at);
  float2 x = make_float2(lower(w), upper(w));
#pragma unroll
  for (int l = 1; l < N; ++l) {
    w = *reinterpret_cast<const uint32_t*>(at + l * plane);
    x.x += lower(w), x.y += upper(w);
  }
  return x;
}

// One 16-wide step: d += the products of the first limbs, low += the other terms above 2^-25 of the largest, smallest
// first.  The instructions' sums truncate at 2^-23 of what they hold, which is 2^-8 less for `low`.
template <int LA, int LB, bool FIRST = false>
__device__ __forceinline__ void mma_terms(float (&d)[2][4], float (&low)[2][4], const uint32_t (&a)[LA][4], const uint32_t (&b)[LB][4]) {
  bool begun = !FIRST;
#pragma unroll
  for (int s = 2; s >= 0; --s)
#pragma unroll
    for (int l = 0; l < LA; ++l)
      if (s - l >= 0 && s - l < LB) {
        float(&to)[2][4] = s ? low : d;
        if (begun && !(FIRST && s == 0)) {
          mma(to[0], a[l], b[s - l][0], b[s - l][1]);
          mma(to[1], a[l], b[s - l][2], b[s - l][3]);
        } else {
          mma_first(to[0], a[l], b[s - l][0], b[s - l][1]);
          mma_first(to[1], a[l], b[s - l][2], b[s - l][3]);
        }
        begun = true;
      }
}

// acc[j] += A B over the 16-wide steps [k0, k1): A 16 x 16 tiles of LA planes, B of LB planes.  pairs: 16-column tiles of B
// that exist.  Products of two limbs (of P and dP, for bfloat16 results) share one sum.
template <int LA, int LB, bool TA, bool TB, int N>
__device__ __forceinline__ void product(float (&acc)[N][2][4], const plane_t* a, int a_pitch, int a_plane, const plane_t* b, int b_pitch,
                                        int b_plane, int k0, int k1, int pairs, int lane) {
  constexpr bool APART = LA * LB > 2;
  float low[APART ? N : 1][2][4] = {};
#pragma unroll 2
  for (int kk = k0; kk < k1; ++kk) {
    uint32_t fa[LA][4];
#pragma unroll
    for (int l = 0; l < LA; ++l) frag_a<TA>(fa[l], a + l * a_plane + (TA ? kk * 16 * a_pitch : kk * 16), a_pitch, lane);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (j >= pairs) break;
      uint32_t fb[LB][4];
#pragma unroll
      for (int l = 0; l < LB; ++l)
        frag_b<TB>(fb[l], b + l * b_plane + (TB ? kk * 16 * b_pitch + j * 16 : j * 16 * b_pitch + kk * 16), b_pitch, lane);
      mma_terms<LA, LB>(acc[j], APART ? low[APART ? j : 0] : acc[j], fa, fb);
    }
  }
  if (APART) {
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
      for (int x = 0; x < 8; ++x) acc[j][x >> 2][x & 3] += low[APART ? j : 0][x >> 2][x & 3];
  }
}

// ---------------------------------------------------------------- gates
// One token of a chunk, as the pairs read it.
struct __align__(16) Token {
  float hi, lo;  // sum of the log decays since the last reset, base 2, in two parts (differences of long sums are exact enough)
  int episode;   // resets up to and including this token
  int pad;
};
template <int C>
struct __align__(16) Gates {
  Token token[C];
  float carried[C];  // c_i: decay from the state in front of the chunk; 0 behind a reset, and for absent tokens
  float to_end[C];   // e_j: decay from token j to the chunk's end; 0 in front of a reset, and for absent tokens
  float keep;        // what is left of the state in front of the chunk
};

// a_ij of a pair, 0 where the mask takes it out.
__device__ __forceinline__ bool meets(const Token& ti, const Token& tj, int i, int j) { return j <= i && ti.episode == tj.episode; }
__device__ __forceinline__ float pair_decay(const Token& ti, const Token& tj, bool meet) {
  return meet ? ex2((ti.hi - tj.hi) + (ti.lo - tj.lo)) : 0.0f;
}

// What is left of a state over two stretches: nothing where one of them drops it, whatever the other's decays are.
__device__ __forceinline__ float both_keep(float a, float b) { return a == 0.0f || b == 0.0f ? 0.0f : a * b; }

// One warp: log decays and marks of n tokens, C / 32 neighbouring ones a lane.  Fetched before the rows, whose loads would be waited for first.
template <int C>
struct GateIn {
  float x[C / 32];
  uint8_t mark[C / 32];  // as in memory: looked at when the rows are under way
};
template <int C>
__device__ __forceinline__ GateIn<C> fetch_gates(const float* g, int64_t g_stride, const uint8_t* reset, int64_t reset_stride, int64_t t0, int n, int lane) {
  constexpr int U = C / 32;
  GateIn<C> in;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = lane * U + u;
    in.x[u] = i < n ? g[(t0 + i) * g_stride] : 0.0f;
    in.mark[u] = i < n && reset ? reset[(t0 + i) * reset_stride] : uint8_t(0);
  }
  return in;
}

// One warp: their gates.  Sums run from the last reset on, so that what one episode's decays are, not finite included, stays in it.  They are
// taken in 64-bit integers, in units of 2^-40: exact in any order, with additions that every SM has many of where those in double are few.  A
// log decay of 2^16 and more counts as not a number.  One decay for all tokens (`fixed`) needs no sum.
template <int C>
__device__ __forceinline__ void scan_gates(Gates<C>& s, GateIn<C> in, bool fixed, int n, int lane) {
  constexpr int U = C / 32;
  const float one = __shfl_sync(kAll, in.x[0], 0);
  bool odd[U], mark[U];
  unsigned marks[U], odds = 0;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    // a decay to nothing is a reset: the sums behind it stay finite
    mark[u] = in.mark[u] || ex2(in.x[u] * 1.4426950408889634f) == 0.0f;
    if (mark[u]) in.x[u] = 0.0f;
    odd[u] = !(in.x[u] < 65536.0f);  // (the least that is no mark is -104)
    marks[u] = __ballot_sync(kAll, mark[u]);
    odds |= __ballot_sync(kAll, odd[u]);
  }
  int all = 0, episode = 0, from = -1;  // from: the last mark in front of the lane's tokens
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const unsigned m = marks[u] & ((1u << lane) - 1);
    all += __popc(marks[u]), episode += __popc(m);
    if (m) from = max(from, (31 - __clz(m)) * U + u);
  }
  float hi[U], lo[U];  // of the sums' products with log2(e)
  auto times_log2e = [](float p, float e, float unit, float& hi, float& lo) {
    constexpr float kL = 1.44269502f, kRest = 1.92596303e-8f;  // log2(e) in two parts
    hi = p * (kL * unit);
    lo = fmaf(p, kL * unit, -hi) + (p * (kRest * unit) + e * (kL * unit));
  };
  if (fixed) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = lane * U + u;
      if (mark[u]) from = i;
      const int steps = min(i, n - 1) - from;
      const float p = steps > 0 ? float(steps) * one : 0.0f, e = steps > 0 ? fmaf(float(steps), one, -p) : 0.0f;
      times_log2e(p, e, 1.0f, hi[u], lo[u]);
    }
  } else {
    constexpr float kUnit = 1.0f / 1099511627776.0f;
    long long sum[U];
#pragma unroll
    for (int u = 0; u < U; ++u) sum[u] = (odd[u] ? 0 : __float2ll_rn(in.x[u] * 1099511627776.0f)) + (u ? sum[u - 1] : 0);
    long long run = sum[U - 1];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long z = __shfl_up_sync(kAll, run, d);
      if (lane >= d) run += z;
    }
    run -= sum[U - 1];
#pragma unroll
    for (int u = 0; u < U; ++u) sum[u] += run;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = lane * U + u;
      if (mark[u]) from = i;
      long long y = sum[u];
      if (all) {  // less the sum at the reset
        long long at = 0;
#pragma unroll
        for (int w = 0; w < U; ++w) {
          const long long z = __shfl_sync(kAll, sum[w], max(from, 0) / U);
          if (from >= 0 && from % U == w) at = z;
        }
        y -= at;
      }
      const float p = __ll2float_rn(y);
      times_log2e(p, __ll2float_rn(y - __float2ll_rn(p)), kUnit, hi[u], lo[u]);
      if (odds) {
        bool lost = false;
#pragma unroll 1
        for (int t = 0; t < C; ++t) {
          bool z = false;
#pragma unroll
          for (int w = 0; w < U; ++w) {
            const bool x = __shfl_sync(kAll, int(odd[w]), t / U);
            if (t % U == w) z = x;
          }
          lost |= z && t > from && t <= i;
        }
        if (lost) hi[u] = __uint_as_float(0x7fffffffu);
      }
    }
  }
  const float last_hi = __shfl_sync(kAll, hi[U - 1], 31), last_lo = __shfl_sync(kAll, lo[U - 1], 31);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = lane * U + u;
    episode += mark[u];
    s.token[i] = Token{hi[u], lo[u], episode, 0};
    s.carried[i] = i < n && episode == 0 ? ex2(hi[u] + lo[u]) : 0.0f;
    s.to_end[i] = i < n && episode == all ? ex2((last_hi - hi[u]) + (last_lo - lo[u])) : 0.0f;
  }
  if (lane == 0) s.keep = all == 0 ? ex2(last_hi + last_lo) : 0.0f;
}

// ---------------------------------------------------------------- rows
__device__ __forceinline__ void copy16(plane_t* to, const void* from, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(delta::smem_at(to)), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_landed() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Which 8 columns of which rows of a chunk a thread moves: rows row, row + STEP, ...
template <class S>
struct Mover {
  static constexpr int LR = S::D / 8, STEP = S::THREADS / LR, TURNS = S::C / STEP;
  static_assert(S::THREADS % LR == 0 && S::C % STEP == 0);
  int row, c;
  __device__ __forceinline__ explicit Mover(int tid) : row(tid / LR), c(tid % LR * 8) {}
};

__device__ __forceinline__ void split_rows(plane_t* at, int plane, const delta::Eight& raw) {
  float x[8];
  delta::unpack8<float>(x, raw);
  uint32_t w[3][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t r[3];
    // an infinity or a NaN is its first limb alone
    const float x0 = x[2 * i], x1 = x[2 * i + 1];
    const bool f0 = fabsf(x0) < INFINITY, f1 = fabsf(x1) < INFINITY;
    split<3>(f0 ? x0 : 0.0f, f1 ? x1 : 0.0f, r);
    if (!f0) r[0] = (r[0] & 0xffff0000u) | (x0 != x0 ? 0x7fc0u : __float_as_uint(x0) >> 16);
    if (!f1) r[0] = (r[0] & 0xffffu) | (x1 != x1 ? 0x7fc00000u : __float_as_uint(x1));
    w[0][i] = r[0], w[1][i] = r[1], w[2][i] = r[2];
  }
#pragma unroll
  for (int l = 0; l < 3; ++l) *reinterpret_cast<uint4*>(at + l * plane) = make_uint4(w[l][0], w[l][1], w[l][2], w[l][3]);
}

// All threads: n rows of `width` values as planes [16 nt][P], zero for absent tokens and past the width up to
// the next 16 columns.  vec: rows are of whole 16-byte pieces.
template <class S>
__device__ __forceinline__ void load_rows(plane_t* to, const typename S::T* from, int64_t stride, int width, bool vec, int n, int nt, const Mover<S>& mv) {
  using M = Mover<S>;
  if (mv.c >= ((width + 15) & ~15)) return;
  const typename S::T* at = from + mv.row * stride + mv.c;
  to += mv.row * S::P + mv.c;
  if (vec) {
    const bool column = mv.c < width;
    if constexpr (S::L == 1) {
#pragma unroll
      for (int u = 0; u < M::TURNS; ++u) {
        const int row = mv.row + u * M::STEP;
        if (row >= nt * 16) break;
        const bool there = row < n && column;
        copy16(to + u * M::STEP * S::P, there ? at : from, there);
        at += M::STEP * stride;
      }
    } else {
      constexpr int BATCH = M::TURNS < 2 ? M::TURNS : 2;
#pragma unroll
      for (int first = 0; first < M::TURNS; first += BATCH) {
        delta::Eight raw[BATCH];
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
          raw[u] = delta::Eight{};
          if (mv.row + (first + u) * M::STEP < n && column) {
            raw[u].a = __ldg(reinterpret_cast<const uint4*>(at));
            raw[u].b = __ldg(reinterpret_cast<const uint4*>(at) + 1);
          }
          at += M::STEP * stride;
        }
#pragma unroll
        for (int u = 0; u < BATCH; ++u)
          if (mv.row + (first + u) * M::STEP < nt * 16) split_rows(to + (first + u) * M::STEP * S::P, S::PLANE, raw[u]);
      }
    }
    return;
  }
#pragma unroll 1
  for (int row = mv.row; row < nt * 16; row += M::STEP) {
    delta::Eight raw{};
    if (row < n && mv.c < width) raw = delta::fetch8_slow(at, width - mv.c);
    if constexpr (S::L == 1) *reinterpret_cast<uint4*>(to) = raw.a;
    else split_rows(to, S::PLANE, raw);
    at += M::STEP * stride;
    to += M::STEP * S::P;
  }
}

// Whether something that this thread brought is not finite (which its first limb shows).
template <class S>
__device__ __forceinline__ bool rows_odd(const plane_t* at, int width, int nt, const Mover<S>& mv) {
  if (mv.c >= ((width + 15) & ~15)) return false;
  __nv_bfloat162 z = __floats2bfloat162_rn(0.0f, 0.0f);
  const __nv_bfloat162 nothing = z;
#pragma unroll
  for (int u = 0; u < Mover<S>::TURNS; ++u) {
    if (mv.row + u * Mover<S>::STEP >= nt * 16) break;
    const uint4 w = *reinterpret_cast<const uint4*>(at + (mv.row + u * Mover<S>::STEP) * S::P + mv.c);
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) z = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&x[e]), nothing, z);
  }
  const float sum = __low2float(z) + __high2float(z);
  return sum != sum;
}

// ---------------------------------------------------------------- the state in the warps' accumulators
// A warp's part: rows [16 (warp % MR), +16), columns [16 NM (warp / MR), +16 NM) of a state [dk][dv].
template <class S>
struct Part {
  int row, col;    // first row and column
  int pairs;       // 16-column tiles that exist (0: none, or no rows)
  __device__ __forceinline__ Part(int warp, int dk, int dv) {
    row = warp % S::MR * 16, col = warp / S::MR * S::NM * 16;
    pairs = S::FULL ? S::NM : row < dk && col < dv ? min(S::NM, (dv - col + 15) / 16) : 0;
  }
};

// A lane's elements of a part are pairs of neighbouring columns: (j, h, r) is at row 8 r and column 16 j + 8 h of its first.
// f(j, h, r, at, second) over the pairs that exist; `second`: so does the second of the pair.
template <class S, class P, class F>
__device__ __forceinline__ void each_pair(P* state, const Part<S>& part, int dk, int dv, int lane, F&& f) {
  const int row = part.row + (lane >> 2), col = part.col + (lane & 3) * 2;
  P* const at[2] = {state + row * dv + col, state + (row + 8) * dv + col};
  if (S::FULL || (part.row + 16 <= dk && part.col + S::NM * 16 <= dv)) {  // all of it
#pragma unroll
    for (int j = 0; j < S::NM; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 2; ++r) f(j, h, r, at[r] + (j * 16 + h * 8), true);
    return;
  }
  const int left[2] = {row < dk ? dv - col : 0, row + 8 < dk ? dv - col : 0};
#pragma unroll
  for (int j = 0; j < S::NM; ++j)
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int r = 0; r < 2; ++r)
        if (j * 16 + h * 8 < left[r]) f(j, h, r, at[r] + (j * 16 + h * 8), j * 16 + h * 8 + 1 < left[r]);
}

template <class S>
__device__ __forceinline__ void clear(float (&m)[S::NM][2][4]) {
#pragma unroll
  for (int j = 0; j < S::NM; ++j)
#pragma unroll
    for (int x = 0; x < 8; ++x) m[j][x >> 2][x & 3] = 0.0f;
}

// Pairs of columns are 8-byte aligned.
__device__ __forceinline__ bool pairs_aligned(const void* p, int dv) { return dv % 2 == 0 && reinterpret_cast<uintptr_t>(p) % 8 == 0; }
__device__ __forceinline__ void write_pair(float* at, int col, int width, bool even, float x, float y) {
  if (even) {
    *reinterpret_cast<float2*>(at) = make_float2(x, y);
  } else {
    at[0] = x;
    if (col + 1 < width) at[1] = y;
  }
}

template <class S>
__device__ __forceinline__ void read_state(float (&m)[S::NM][2][4], const float* from, const Part<S>& part, int dk, int dv, int lane) {
  clear<S>(m);
  if (pairs_aligned(from, dv)) {
    each_pair<S>(from, part, dk, dv, lane, [&](int j, int h, int r, const float* at, bool) {
      const float2 v = *reinterpret_cast<const float2*>(at);
      m[j][h][2 * r] = v.x, m[j][h][2 * r + 1] = v.y;
    });
  } else {
    each_pair<S>(from, part, dk, dv, lane, [&](int j, int h, int r, const float* at, bool second) {
      m[j][h][2 * r] = at[0];
      if (second) m[j][h][2 * r + 1] = at[1];
    });
  }
}
template <class S>
__device__ __forceinline__ void write_state(const float (&m)[S::NM][2][4], float* to, const Part<S>& part, int dk, int dv, int lane) {
  if (pairs_aligned(to, dv)) {
    each_pair<S>(to, part, dk, dv, lane,
                 [&](int j, int h, int r, float* at, bool) { *reinterpret_cast<float2*>(at) = make_float2(m[j][h][2 * r], m[j][h][2 * r + 1]); });
  } else {
    each_pair<S>(to, part, dk, dv, lane, [&](int j, int h, int r, float* at, bool second) {
      at[0] = m[j][h][2 * r];
      if (second) at[1] = m[j][h][2 * r + 1];
    });
  }
}

// The part's limbs into planes [D][P] (whole 16 x 16 tiles).
template <class S, int N>
__device__ __forceinline__ void dump_state(const float (&m)[S::NM][2][4], plane_t* to, const Part<S>& part, int lane) {
#pragma unroll
  for (int j = 0; j < S::NM; ++j) {
    if (j >= part.pairs) break;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        uint32_t w[N];
        split<N>(m[j][h][2 * r], m[j][h][2 * r + 1], w);
        plane_t* at = to + (part.row + (lane >> 2) + r * 8) * S::P + part.col + j * 16 + h * 8 + (lane & 3) * 2;
#pragma unroll
        for (int l = 0; l < N; ++l) *reinterpret_cast<uint32_t*>(at + l * S::SPLANE) = w[l];
      }
  }
}

// m = keep m + sum_j factor weight[j] x_j y_j^T over a chunk's tokens, 32 of them at a time.  The weight goes into x's
// fragments, which then have three limbs.
template <class S>
__device__ __forceinline__ void update(float (&m)[S::NM][2][4], const plane_t* x, const plane_t* y, const float* weight, float factor,
                                       float keep, int nt, const Part<S>& part, int lane) {
#pragma unroll
  for (int half = 0; half < S::RT; half += 2) {
    if (half >= nt || !part.pairs) break;
    uint32_t a[2][3][4];
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      if (half + kk >= nt) break;
      const int t = (half + kk) * 16;
      uint32_t raw[S::L][4];
#pragma unroll
      for (int l = 0; l < S::L; ++l) frag_a<true>(raw[l], x + l * S::PLANE + t * S::P + part.row, S::P, lane);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float2 w = *reinterpret_cast<const float2*>(weight + t + (r >> 1) * 8 + (lane & 3) * 2);
        float x0 = lower(raw[0][r]), x1 = upper(raw[0][r]);
#pragma unroll
        for (int l = 1; l < S::L; ++l) x0 += lower(raw[l][r]), x1 += upper(raw[l][r]);
        uint32_t limbs[3];
        split<3>(x0 * (w.x * factor), x1 * (w.y * factor), limbs);
        a[kk][0][r] = limbs[0], a[kk][1][r] = limbs[1], a[kk][2][r] = limbs[2];
      }
    }
#pragma unroll
    for (int j = 0; j < S::NM; ++j) {
      if (j >= part.pairs) break;
      float acc[2][4], low[2][4];
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        if (kk && half + kk >= nt) break;
        uint32_t b[S::L][4];
#pragma unroll
        for (int l = 0; l < S::L; ++l) frag_b<true>(b[l], y + l * S::PLANE + (half + kk) * 16 * S::P + part.col + j * 16, S::P, lane);
        if (kk) mma_terms<3, S::L>(acc, low, a[kk], b);
        else mma_terms<3, S::L, true>(acc, low, a[kk], b);
      }
      const float k = half ? 1.0f : keep;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float add = acc[h][e] + low[h][e];
          m[j][h][e] = k == 0.0f ? add : fmaf(k, m[j][h][e], add);
        }
    }
  }
}
// The same, element by element, leaving out tokens of no weight.
template <class S>
__device__ __noinline__ float update_slow(float old, const plane_t* x, const plane_t* y, const float* weight, float factor, float keep, int n) {
  float sum = 0.0f;
  for (int j = 0; j < n; ++j)
    if (weight[j] != 0.0f) sum = fmaf(weight[j] * factor * value<S::L>(x + j * S::P, S::PLANE), value<S::L>(y + j * S::P, S::PLANE), sum);
  return keep == 0.0f ? sum : fmaf(keep, old, sum);
}
template <class S>
__device__ __forceinline__ void update_masked(float (&m)[S::NM][2][4], const plane_t* x, const plane_t* y, const float* weight, float factor,
                                              float keep, int n, const Part<S>& part, int dk, int dv, int lane) {
#pragma unroll
  for (int j = 0; j < S::NM; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int row = part.row + (lane >> 2) + ((e >> 1) & 1) * 8, col = part.col + j * 16 + (e >> 2) * 8 + (lane & 3) * 2 + (e & 1);
      if (row < dk && col < dv) m[j][e >> 2][e & 3] = update_slow<S>(m[j][e >> 2][e & 3], x + row, y + col, weight, factor, keep, n);
    }
}

// Whether any of a warp's accumulators is not finite (a sum that overflows counts too).
template <int N>
__device__ __forceinline__ bool not_finite(const float (&acc)[N][2][4]) {
  float sum = 0.0f;
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int x = 0; x < 8; ++x) sum = fmaf(acc[j][x >> 2][x & 3], 0.0f, sum);
  return sum != sum;
}

// ---------------------------------------------------------------- results
// A warp's part of a product, rows [16 r, +16) and columns [col, col + 16 N), rounded into rows of bfloat16.
template <class S, int N>
__device__ __forceinline__ void stage(plane_t* to, const float (&acc)[N][2][4], int row, int col, int pairs, int lane) {
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if (j >= pairs) break;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int r = 0; r < 2; ++r)
        *reinterpret_cast<uint32_t*>(to + (row + (lane >> 2) + r * 8) * S::P + col + j * 16 + h * 8 + (lane & 3) * 2) =
            pack_round(acc[j][h][2 * r], acc[j][h][2 * r + 1]);
  }
}
// All threads: staged rows to memory.
template <class S>
__device__ __forceinline__ void store_rows(bf16* to, int64_t stride, const plane_t* from, int width, bool vec, int n, const Mover<S>& mv) {
  using M = Mover<S>;
  if (mv.c >= width) return;
  plane_t* at = reinterpret_cast<plane_t*>(to) + mv.row * stride + mv.c;
  from += mv.row * S::P + mv.c;
  if (vec) {
#pragma unroll
    for (int u = 0; u < M::TURNS; ++u) {
      if (mv.row + u * M::STEP >= n) break;
      *reinterpret_cast<uint4*>(at) = *reinterpret_cast<const uint4*>(from + u * M::STEP * S::P);
      at += M::STEP * stride;
    }
    return;
  }
#pragma unroll 1
  for (int row = mv.row; row < n; row += M::STEP) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (mv.c + i < width) at[i] = from[i];
    at += M::STEP * stride;
    from += M::STEP * S::P;
  }
}
// A warp's part of a product as 32-bit values straight to memory (four lanes fill a 32-byte sector).
template <int N>
__device__ __forceinline__ void store_float(float* to, int64_t stride, const float (&acc)[N][2][4], int row, int col, int n, int width, int lane) {
  const bool even = reinterpret_cast<uintptr_t>(to) % 8 == 0 && stride % 2 == 0 && width % 2 == 0;
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int i = row + (lane >> 2) + r * 8, c = col + j * 16 + h * 8 + (lane & 3) * 2;
        if (i < n && c < width) write_pair(to + i * stride + c, c, width, even, acc[j][h][2 * r], acc[j][h][2 * r + 1]);
      }
}

// Where one (environment, value head) is in a tensor.
template <class T>
__device__ __forceinline__ T* place(const ZenoTensor& t, int64_t b, int64_t h) {
  return static_cast<T*>(t.data) + b * t.stride[0] + h * t.stride[2];
}

// Rows of whole 16-byte pieces, of each tensor.
enum : uint32_t { kVecQ = 1, kVecK = 2, kVecV = 4, kVecOut = 8, kVecDq = 16, kVecDk = 32, kVecDv = 64 };

// Rollouts in segments of `chunks` chunks, one block each.
struct Segments {
  uint32_t count, chunks;
  uint32_t vec;    // kVec...
  float* state;  // [rows][count][dk][dv]: first what a segment adds, then the state in front of it (behind it in reverse)
  float* keep;   // [rows][count]: what a segment leaves of the state in front of it
};

}  // namespace linear
}  // namespace zb
