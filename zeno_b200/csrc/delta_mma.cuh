// Building blocks of the chunked gated delta rule: 16-bit matrix products on split
// operands, and the token-by-token matrices of one chunk.
//
// Precision.  A 32-bit value x is taken into the 16-bit matrix instructions as two f16
// limbs of x s, hi = f16(x s) and lo = f16(x s - hi), with s a power of two that puts the
// largest value of the row (or tile) near 2^14: 22 bits of the row's largest value, and
// values 2^-16 of it still keep all of theirs.  Products are hi hi + lo hi + hi lo with
// 32-bit sums (lo lo is below 2^-22).  bfloat16 inputs are exact in one limb once their
// row is scaled, so a product of an input with a computed value takes two instructions.
// The backward pass gives dO, W, dE, S0 and R one scale for all channels and tokens of a chunk
// (their products contract over either): what lies 2^-16 below its largest value loses bits
// there, and below 2^-38 is dropped.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "policy_ops.h"

namespace zb {
namespace delta {

constexpr int C = kDeltaChunk;
constexpr int CP = C + 8;    // pitch of a chunk's token-by-token matrix: rows 16 bytes apart in banks
constexpr int TP = 16 + 8;   // pitch of a 16-column matrix
constexpr unsigned kAll = 0xffffffffu;

__device__ __forceinline__ uint32_t smem_at(const void* p) { return uint32_t(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 8 x 8 transpose of 16-bit values over the warp
__device__ __forceinline__ uint32_t movm(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Fragments of a 16 x 16 operand in shared memory (half, `pitch` a multiple of 8).
// a_rows: A[m][k] stored [m][k]; a_cols: A[m][k] stored [k][m];
// b_rows: B[k][n] stored [n][k]; b_cols: B[k][n] stored [k][n] (two n8 tiles: regs 0,1 and 2,3).
__device__ __forceinline__ void a_rows(uint32_t (&r)[4], const __half* at, int pitch, int lane) {
  ldsm4(r, smem_at(at + (lane & 15) * pitch + (lane >> 4) * 8));
}
__device__ __forceinline__ void a_cols(uint32_t (&r)[4], const __half* at, int pitch, int lane) {
  ldsm4t(r, smem_at(at + ((lane >> 4) * 8 + (lane & 7)) * pitch + ((lane >> 3) & 1) * 8));
}
__device__ __forceinline__ void b_rows(uint32_t (&r)[4], const __half* at, int pitch, int lane) {
  ldsm4(r, smem_at(at + ((lane >> 4) * 8 + (lane & 7)) * pitch + ((lane >> 3) & 1) * 8));
}
__device__ __forceinline__ void b_cols(uint32_t (&r)[4], const __half* at, int pitch, int lane) {
  ldsm4t(r, smem_at(at + (lane & 15) * pitch + (lane >> 4) * 8));
}

// The power of two that takes `most` (>= 0) to [2^14, 2^15), and its inverse.  Below
// 2^-86 the scale stays at 2^100: such values lose bits against 2^-110, not against one another.
__device__ __forceinline__ int pow2_exp(float most) { return max(int(__float_as_uint(most) >> 23), 41); }
__device__ __forceinline__ float pow2_scale(int e) { return __uint_as_float(uint32_t(268 - e) << 23); }
__device__ __forceinline__ float pow2_unscale(int e) { return __uint_as_float(uint32_t(e - 14) << 23); }

// Two scaled values as packed limbs.
__device__ __forceinline__ void split(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}

// The A fragment (16 x 16, two limbs) of two neighbouring accumulator tiles; row r and
// r + 8 of the thread are scaled by s0 and s1, the columns by col[4] (2q, 2q+1 of each tile).
__device__ __forceinline__ void split_a(uint32_t (&hi)[4], uint32_t (&lo)[4], const float (&t0)[4], const float (&t1)[4],
                                        float s0, float s1) {
  split(t0[0] * s0, t0[1] * s0, hi[0], lo[0]);
  split(t0[2] * s1, t0[3] * s1, hi[1], lo[1]);
  split(t1[0] * s0, t1[1] * s0, hi[2], lo[2]);
  split(t1[2] * s1, t1[3] * s1, hi[3], lo[3]);
}

__device__ __forceinline__ float quad_max(float x) {  // over the 4 lanes of one accumulator row
  x = fmaxf(x, __shfl_xor_sync(kAll, x, 1));
  return fmaxf(x, __shfl_xor_sync(kAll, x, 2));
}

template <class T>
struct In;
template <>
struct In<__nv_bfloat16> {
  static constexpr int limbs = 1;
  static __device__ __forceinline__ float up(__nv_bfloat16 x) { return __bfloat162float(x); }
};
template <>
struct In<float> {
  static constexpr int limbs = 2;
  static __device__ __forceinline__ float up(float x) { return x; }
};

// One token of a chunk, as the token-by-token matrices read it.
struct __align__(16) Token {
  float hi, lo;  // running sum of the log decays, base 2, in two parts (differences of long sums are exact enough)
  float fk;      // what takes the scaled row of K to the normalised one
  int episode;   // resets up to and including this token
};

// Gates of one chunk.
struct Gates {
  Token token[C];
  __align__(16) float carried[C];  // a_i: decay from the state in front of the chunk; 0 behind a reset, and for absent tokens
  float to_end[C];    // D_Ci: decay from token i to the chunk's end, 0 for absent tokens
  float beta[C];
  float fq[C];        // what takes the scaled row of Q to the normalised one
  float nk[C], nq[C]; // 1 / norm of the rows (1 where they are not normalised)
  float ak[C], aq[C], zk[C];  // a_i fk_i, a_i fq_i, D_Ci fk_i
  unsigned most[2];   // largest magnitudes of Q and K, as float bits (backward)
  unsigned marks;     // the tokens that clear the state
  float keep;         // a_C: what is left of the state in front of the chunk
  int bad;            // some input of this chunk is not finite
  int state_bad;      // some element of the state in front of this chunk is not finite
};

__device__ __forceinline__ float decay(const Token& i, const Token& j) {  // from token j to token i, j <= i
  return i.episode == j.episode ? exp2f((i.hi - j.hi) + (i.lo - j.lo)) : 0.0f;
}

// max.NaN: not a number where one of the two is none
__device__ __forceinline__ float max_nan(float x, float y) {
  float z;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(z) : "f"(x), "f"(y));
  return z;
}

// 1 / sqrt(x): the approximation and one Newton step
__device__ __forceinline__ float inverse_sqrt(float x) {
  const float y = rsqrtf(x);
  return fmaf(0.5f * y, fmaf(-x * y, y, 1.0f), y);
}

// Where one block's tokens are.
template <class T>
struct Rows {
  const T *q, *k, *v;
  const float *g, *beta;
  const uint8_t* reset;
  bool vec_qk, vec_v;
};

template <class T>
__device__ __forceinline__ bool vec_ok(const ZenoTensor& t, int width) {
  constexpr int64_t n = 16 / sizeof(T);
  return width % 8 == 0 && reinterpret_cast<uintptr_t>(t.data) % 16 == 0 && t.stride[0] % n == 0 && t.stride[1] % n == 0 &&
         t.stride[2] % n == 0;
}

template <class T>
__device__ __forceinline__ Rows<T> rows_of(const ZenoDeltaRule& p, uint32_t b, uint32_t h) {
  const uint32_t kh = h / (p.value_heads / p.key_heads);
  Rows<T> r;
  r.q = static_cast<const T*>(p.q.data) + int64_t(b) * p.q.stride[0] + int64_t(kh) * p.q.stride[2];
  r.k = static_cast<const T*>(p.k.data) + int64_t(b) * p.k.stride[0] + int64_t(kh) * p.k.stride[2];
  r.v = static_cast<const T*>(p.v.data) + int64_t(b) * p.v.stride[0] + int64_t(h) * p.v.stride[2];
  r.g = static_cast<const float*>(p.g.data) + int64_t(b) * p.g.stride[0] + int64_t(h) * p.g.stride[2];
  r.beta = static_cast<const float*>(p.beta.data) + int64_t(b) * p.beta.stride[0] + int64_t(h) * p.beta.stride[2];
  r.reset = p.reset.data ? static_cast<const uint8_t*>(p.reset.data) + int64_t(b) * p.reset.stride[0] : nullptr;
  r.vec_qk = vec_ok<T>(p.q, int(p.key_dim)) && vec_ok<T>(p.k, int(p.key_dim));
  r.vec_v = vec_ok<T>(p.v, int(p.value_dim));
  return r;
}

// Warp 0: the gates of tokens [t0, t0 + C) that lie in [lo, hi), a token a lane; the others are
// absent (no decay, nothing written).  Fetched first, scanned when the rows are under way.
struct GateIn {
  float g, beta;
  bool here, mark;
};
__device__ __forceinline__ GateIn fetch_gates(const ZenoDeltaRule& p, const float* g, const float* beta, const uint8_t* reset, int64_t t0,
                                              int64_t lo, int64_t hi, int lane) {
  const int64_t t = t0 + lane;
  GateIn r;
  r.here = t >= lo && t < hi;
  r.g = r.here ? g[t * p.g.stride[1]] : 0.0f;
  r.beta = r.here ? beta[t * p.beta.stride[1]] : 0.0f;
  r.mark = r.here && reset && reset[t * p.reset.stride[1]];
  return r;
}

__device__ __forceinline__ void scan_gates(Gates& s, const GateIn& in, int lane) {
  float x = in.g;
  const float be = in.beta;
  const bool here = in.here, mark = in.mark;
  const bool clear = mark || expf(x) == 0.0f;  // a decay to nothing is a reset: the sums behind it stay finite
  if (clear) x = 0.0f;
  double sum = x;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const double y = __shfl_up_sync(kAll, sum, d);
    if (lane >= d) sum += y;
  }
  const unsigned marks = __ballot_sync(kAll, clear);
  const int episode = __popc(marks & (kAll >> (31 - lane)));
  sum *= 1.4426950408889634;
  const double last = __shfl_sync(kAll, sum, 31);
  s.token[lane].hi = float(sum);
  s.token[lane].lo = float(sum - float(sum));
  s.token[lane].episode = episode;
  s.beta[lane] = be;
  s.carried[lane] = here && episode == 0 ? exp2f(float(sum)) : 0.0f;
  if (lane == 0) s.marks = marks;
  if (lane == 0) s.keep = marks == 0 ? exp2f(float(last)) : 0.0f;
  s.to_end[lane] = here && episode == __popc(marks) ? exp2f(float(last - sum)) : 0.0f;
  if (!(fabsf(x) < INFINITY) || !(fabsf(be) < INFINITY)) s.bad = 1;
}

// One warp, once the gates and the rows' factors are there.
__device__ __forceinline__ void join_factors(Gates& s, int lane) {
  const float fk = s.token[lane].fk, a = s.carried[lane];
  s.ak[lane] = a * fk, s.aq[lane] = a * s.fq[lane], s.zk[lane] = s.to_end[lane] * fk;
}

// 8 values of a row as they are in memory.
struct Eight {
  uint4 a, b;  // b: the second half of 32-bit values
};
template <class T>
__device__ __noinline__ Eight fetch8_slow(const T* at, int n) {  // rows that are not 16-byte aligned, ragged ends
  Eight r;
  {
    uint32_t w[8] = {};
    if constexpr (sizeof(T) == 2) {
      const unsigned short* u = reinterpret_cast<const unsigned short*>(at);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) w[i >> 1] |= uint32_t(u[i]) << (16 * (i & 1));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) w[i] = __float_as_uint(at[i]);
    }
    r.a = make_uint4(w[0], w[1], w[2], w[3]), r.b = make_uint4(w[4], w[5], w[6], w[7]);
  }
  return r;
}
template <class T>
__device__ __forceinline__ Eight fetch8(const T* at, int n, bool vec) {
  if (!vec || n < 8) return fetch8_slow<T>(at, n);
  Eight r;
  r.a = __ldg(reinterpret_cast<const uint4*>(at));
  if (sizeof(T) == 4) r.b = __ldg(reinterpret_cast<const uint4*>(at) + 1);
  return r;
}
__device__ __forceinline__ void prefetch(const void* at) { asm volatile("prefetch.global.L2 [%0];" ::"l"(at)); }
// The rows of Q, K and V of the chunk at t0 (only its first address of each row and 128 bytes: a hint).
template <int NW, class T>
__device__ __forceinline__ void prefetch_rows(const ZenoDeltaRule& p, const Rows<T>& r, int64_t t0, int v0, int tid) {
  constexpr int LINE = 128 / int(sizeof(T));
  const int64_t t = t0 + tid % C;
  if (t < 0 || t >= p.tokens) return;
  for (int part = tid / C; part < 3 * 128 / LINE; part += NW) {
    const int c = part / 3 * LINE;
    if (part % 3 == 0 && c < int(p.key_dim)) prefetch(r.q + t * p.q.stride[1] + c);
    if (part % 3 == 1 && c < int(p.key_dim)) prefetch(r.k + t * p.k.stride[1] + c);
    if (part % 3 == 2 && v0 + c < int(p.value_dim)) prefetch(r.v + t * p.v.stride[1] + v0 + c);
  }
}
template <class T>
__device__ __forceinline__ void unpack8(float (&x)[8], const Eight& r) {
  if constexpr (sizeof(T) == 2) {
    const uint32_t w[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
    const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(w[i]);
  }
}

// All warps: rows of Q and K as scaled limb planes [C][DK + 8], their factors, and V as it is
// [C][16 NW + 16 / sizeof(T)], zero for absent tokens and past the widths (dv: V's).  All loads of a batch are
// under way before the first is used.
//
// A row is scaled by its own largest value.  With normalised rows that leaves factors of nearly
// one size (a row far below the norms' 1e-3 is not scaled up further, and an empty one neither).
// UNIFORM (backward, which multiplies two rows' factors into one matrix and divides them out again):
// rows that are not normalised share the largest value of the chunk's Q or K instead, found in a
// pass of its own.
template <int DK, int NW, class T, bool UNIFORM>
__device__ __forceinline__ void load_rows(Gates& s, const ZenoDeltaRule& p, const Rows<T>& r, __half* qp, __half* kp, T* vp,
                                          int v0, int dv, int64_t t0, int64_t lo, int64_t hi, int tid) {
  constexpr int LR = DK / 8, PITCH = DK + 8, PLANE = C * PITCH, THREADS = NW * 32;
  constexpr int VC = 16 * NW, VP = VC + 16 / int(sizeof(T));
  constexpr int JOBS = 2 * C * LR / THREADS < 1 ? 1 : 2 * C * LR / THREADS, VJOBS = C * VC / 8 / THREADS;
  constexpr int BATCH = sizeof(T) == 2 ? (JOBS < 4 ? JOBS : 4) : (JOBS < 2 ? JOBS : 2);
  const int dk = int(p.key_dim);
  bool bad = false;
  if (UNIFORM && !p.normalize) {
    if (tid < 2) s.most[tid] = 0;
    __syncthreads();
#pragma unroll 1
    for (int j = tid; j < 2 * C * LR; j += THREADS) {
      const int row = (j / LR) % C, at = (j % LR) * 8;
      const int64_t t = t0 + row;
      if (t >= lo && t < hi && at < dk) {
        float x[8], most = 0.0f;
        unpack8<T>(x, fetch8(j >= C * LR ? r.k + t * p.k.stride[1] + at : r.q + t * p.q.stride[1] + at, dk - at, r.vec_qk));
#pragma unroll
        for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(x[i]));
        if (most < INFINITY) atomicMax(&s.most[j >= C * LR], __float_as_uint(most));
      }
    }
    __syncthreads();
  }
  Eight v[VJOBS];
#pragma unroll
  for (int u = 0; u < VJOBS; ++u) {
    const int j = tid + u * THREADS, row = j / (VC / 8), at = (j % (VC / 8)) * 8;
    const int64_t t = t0 + row;
    v[u] = Eight{};
    if (t >= lo && t < hi && v0 + at < dv) v[u] = fetch8(r.v + t * p.v.stride[1] + v0 + at, dv - v0 - at, r.vec_v);
  }
#pragma unroll
  for (int first = 0; first < JOBS; first += BATCH) {
    Eight raw[BATCH];
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const int j = tid + (first + u) * THREADS, row = (j / LR) % C, at = (j % LR) * 8;
      const int64_t t = t0 + row;
      raw[u] = Eight{};
      if (t >= lo && t < hi && at < dk && j < 2 * C * LR)
        raw[u] = fetch8(j >= C * LR ? r.k + t * p.k.stride[1] + at : r.q + t * p.q.stride[1] + at, dk - at, r.vec_qk);
    }
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const int j = tid + (first + u) * THREADS, row = (j / LR) % C, at = (j % LR) * 8;
      const bool is_k = j >= C * LR;
      float x[8];
      unpack8<T>(x, raw[u]);
      float sum = 0.0f, most = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = fmaf(x[i], x[i], sum), most = fmaxf(most, fabsf(x[i]));
#pragma unroll
      for (int d = 1; d < LR; d <<= 1) {
        sum += __shfl_xor_sync(kAll, sum, d);
        most = fmaxf(most, __shfl_xor_sync(kAll, most, d));
      }
      bad |= !(sum < INFINITY);
      if (p.normalize) most = fmaxf(most, 0x1p-12f);
      else if (UNIFORM) most = fmaxf(__uint_as_float(s.most[is_k]), 0x1p-40f);
      const int e = pow2_exp(most);
      const float sc = pow2_scale(e);
      uint4 hi4, lo4;
      split(x[0] * sc, x[1] * sc, hi4.x, lo4.x);
      split(x[2] * sc, x[3] * sc, hi4.y, lo4.y);
      split(x[4] * sc, x[5] * sc, hi4.z, lo4.z);
      split(x[6] * sc, x[7] * sc, hi4.w, lo4.w);
      const float n = p.normalize ? inverse_sqrt(sum + kNormEps) : 1.0f, f = n * pow2_unscale(e);
      if (2 * C * LR % THREADS == 0 || j < 2 * C * LR) {
        __half* to = (is_k ? kp : qp) + row * PITCH + at;
        *reinterpret_cast<uint4*>(to) = hi4;
        if (In<T>::limbs == 2) *reinterpret_cast<uint4*>(to + PLANE) = lo4;
        if (at == 0) {
          if (is_k) s.token[row].fk = f, s.nk[row] = n;
          else s.fq[row] = f, s.nq[row] = n;
        }
      }
    }
  }
#pragma unroll
  for (int u = 0; u < VJOBS; ++u) {
    const int j = tid + u * THREADS, row = j / (VC / 8), at = (j % (VC / 8)) * 8;
    float x[8], most = 0.0f;
    unpack8<T>(x, v[u]);
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max_nan(most, fabsf(x[i]));
    bad |= !(most < INFINITY);
    T* to = vp + row * VP + at;
    *reinterpret_cast<uint4*>(to) = v[u].a;
    if (sizeof(T) == 4) *(reinterpret_cast<uint4*>(to) + 1) = v[u].b;
  }
  if (bad) s.bad = 1;
}

// All warps, where a chunk has rows that are not finite or whose squares are not: the factors of the latter,
// from values 2^80 times smaller.  load_rows' planes are right for them.  A warp a row.
template <int NW, class T>
__device__ __forceinline__ void mend_norms(Gates& s, const ZenoDeltaRule& p, const Rows<T>& r, int64_t t0, int64_t lo, int64_t hi, int tid) {
  const int lane = tid & 31;
#pragma unroll 1
  for (int j = tid >> 5; j < 2 * C; j += NW) {
    const int row = j % C;
    const int64_t t = t0 + row;
    if (t < lo || t >= hi) continue;
    const T* at = j >= C ? r.k + t * p.k.stride[1] : r.q + t * p.q.stride[1];
    float sum = 0.0f, most = 0.0f;
#pragma unroll 1
    for (int c = lane; c < int(p.key_dim); c += 32) {
      const float x = In<T>::up(at[c]), y = x * 0x1p-80f;
      sum = fmaf(y, y, sum), most = max_nan(most, fabsf(x));
    }
#pragma unroll 1
    for (int d = 1; d < 32; d <<= 1) {
      sum += __shfl_xor_sync(kAll, sum, d);
      most = max_nan(most, __shfl_xor_sync(kAll, most, d));
    }
    // below 2^60 the squares of 128 values stay in 32 bits
    if (!(most >= 0x1p60f && most < INFINITY) || lane != 0) continue;
    const float n = inverse_sqrt(sum), f = n * (pow2_unscale(pow2_exp(most)) * 0x1p-80f);
    if (j >= C) s.token[row].fk = f, s.nk[row] = n * 0x1p-80f;
    else s.fq[row] = f, s.nq[row] = n * 0x1p-80f;
  }
}

// Products of 16 rows of X with 16 rows of Y over the key channels: acc[2] tiles (n8 each).
template <int DK, int LIMBS>
__device__ __forceinline__ void rows_times_rows(float (&acc)[2][4], const __half* x, const __half* y, int lane) {
  constexpr int PITCH = DK + 8, PLANE = C * PITCH;
#pragma unroll
  for (int kk = 0; kk < DK; kk += 16) {
    uint32_t a[4], b[4];
    a_rows(a, x + kk, PITCH, lane);
    b_rows(b, y + kk, PITCH, lane);
    mma(acc[0], a, b[0], b[1]);
    mma(acc[1], a, b[2], b[3]);
    if (LIMBS == 2) {
      uint32_t al[4], bl[4];
      a_rows(al, x + PLANE + kk, PITCH, lane);
      b_rows(bl, y + PLANE + kk, PITCH, lane);
      mma(acc[0], al, b[0], b[1]);
      mma(acc[1], al, b[2], b[3]);
      mma(acc[0], a, bl[0], bl[1]);
      mma(acc[1], a, bl[2], bl[3]);
    }
  }
}

// Token-by-token matrices of a chunk, as limb planes:
//   n: N_10 = D k_i.k_j beta_j, rows of the second half against the first, one scale [16][TP]
//   t: (I + N_rr)^-1 of the two diagonal blocks, a scale each [C][TP]
//   p: P_ij = D q_i.k_j (j <= i) with a scale for each row; backward: its transpose [C][CP]
// gram (backward): D k_i.k_j, j < i.
constexpr int kSquarePitch = 20;
struct Squares {  // diagonal blocks of N, transposed, on their way to the inverses
  __align__(16) float at[2][16 * kSquarePitch];
};
struct Pairs {
  __align__(16) __half n[2][16 * TP];
  __align__(16) __half t[2][C * TP];
  __align__(16) __half p[2][C * CP];
  __align__(16) float fp[C];
  float fn, ft[2];
};
struct Gram {
  float at[C][C + 1];
};

__device__ __forceinline__ void store_split(__half* hi, __half* lo, int at, float x, float y) {
  uint32_t h, l;
  split(x, y, h, l);
  *reinterpret_cast<uint32_t*>(hi + at) = h;
  *reinterpret_cast<uint32_t*>(lo + at) = l;
}

// One warp: N of both diagonal blocks and the inverses of I + N.  Lane c + 16 r solves column c of
// block r by forward substitution, right-looking: a step's updates do not wait for one another.
template <int DK, int LIMBS>
__device__ __forceinline__ void diagonal_inverses(const Gates& s, Pairs& m, Squares& q, Gram* gram, const __half* kp, int halves,
                                                  int lane) {
  constexpr int PITCH = DK + 8;
  const int gi = lane >> 2, qj = (lane & 3) * 2;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    if (r == halves) break;
    float acc[2][4] = {};
    rows_times_rows<DK, LIMBS>(acc, kp + r * 16 * PITCH, kp + r * 16 * PITCH, lane);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int i = gi + half * 8;
      const Token ti = s.token[r * 16 + i];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int j = (x >> 1) * 8 + qj + (x & 1);
        const Token tj = s.token[r * 16 + j];
        const float y = j < i ? acc[x >> 1][half * 2 + (x & 1)] * (ti.fk * tj.fk) * decay(ti, tj) : 0.0f;
        q.at[r][j * kSquarePitch + i] = y * s.beta[r * 16 + j];
        if (gram) gram->at[r * 16 + i][r * 16 + j] = y;
      }
    }
  }
  __syncwarp();
  float t[16];
  const int c = lane & 15, r = lane >> 4;
  const float* sq = q.at[r];
#pragma unroll
  for (int i = 0; i < 16; ++i) t[i] = i == c ? 1.0f : 0.0f;
#pragma unroll
  for (int j = 0; j < 15; ++j) {
#pragma unroll
    for (int i = (j + 1) & ~3; i < 16; i += 4) {
      const float4 n = *reinterpret_cast<const float4*>(sq + j * kSquarePitch + i);
      const float w[4] = {n.x, n.y, n.z, n.w};
#pragma unroll
      for (int x = 0; x < 4; ++x)
        if (i + x > j) t[i + x] = fmaf(-w[x], t[j], t[i + x]);
    }
  }
  float most = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) most = fmaxf(most, fabsf(t[i]));
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) most = fmaxf(most, __shfl_xor_sync(kAll, most, d));
  const int e = pow2_exp(most);
  const float sc = pow2_scale(e);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float x = t[i] * sc;
    const __half hi = __float2half_rn(x);
    m.t[0][(r * 16 + i) * TP + c] = hi;
    m.t[1][(r * 16 + i) * TP + c] = __float2half_rn(x - __half2float(hi));
  }
  if (c == 0) m.ft[r] = pow2_unscale(e);
}

// One warp: N_10.
template <int DK, int LIMBS>
__device__ __forceinline__ void lower_block(const Gates& s, Pairs& m, Gram* gram, const __half* kp, int lane) {
  constexpr int PITCH = DK + 8;
  float acc[2][4] = {};
  rows_times_rows<DK, LIMBS>(acc, kp + 16 * PITCH, kp, lane);
  const int gi = lane >> 2, qj = (lane & 3) * 2;
  float most = 0.0f;
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int i = gi + (x >> 1) * 8, j = n * 8 + qj + (x & 1);
      const Token ti = s.token[16 + i], tj = s.token[j];
      const float y = acc[n][x] * (ti.fk * tj.fk) * decay(ti, tj);
      if (gram) gram->at[16 + i][j] = y;
      acc[n][x] = y * s.beta[j];
      most = fmaxf(most, fabsf(acc[n][x]));
    }
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) most = fmaxf(most, __shfl_xor_sync(kAll, most, d));
  const int e = pow2_exp(most);
  const float sc = pow2_scale(e);
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int half = 0; half < 2; ++half)
      store_split(m.n[0], m.n[1], (gi + half * 8) * TP + n * 8 + qj, acc[n][2 * half] * sc, acc[n][2 * half + 1] * sc);
  if (lane == 0) m.fn = pow2_unscale(e);
}

// One warp: rows [16 r, 16 r + 16) of P.
template <int DK, int LIMBS>
__device__ __forceinline__ void score_rows(const Gates& s, Pairs& m, const __half* qp, const __half* kp, int r, int lane) {
  constexpr int PITCH = DK + 8;
  float acc[4][4] = {};
  rows_times_rows<DK, LIMBS>(reinterpret_cast<float(&)[2][4]>(acc[0]), qp + r * 16 * PITCH, kp, lane);
  if (r == 1) rows_times_rows<DK, LIMBS>(reinterpret_cast<float(&)[2][4]>(acc[2]), qp + 16 * PITCH, kp + 16 * PITCH, lane);
  const int gi = lane >> 2, qj = (lane & 3) * 2;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int i = r * 16 + gi + half * 8;
    const Token ti = s.token[i];
    const float fq = s.fq[i];
    float x[8], most = 0.0f;
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      const int j = (n >> 1) * 8 + qj + (n & 1);
      x[n] = 0.0f;
      if (n >= 4 && r == 0) continue;
      const Token tj = s.token[j];
      if (j <= i) x[n] = acc[n >> 1][half * 2 + (n & 1)] * (fq * tj.fk) * decay(ti, tj);
      most = fmaxf(most, fabsf(x[n]));
    }
    most = quad_max(most);
    const int e = pow2_exp(most);
    const float sc = pow2_scale(e);
#pragma unroll
    for (int n = 0; n < 4; ++n) store_split(m.p[0], m.p[1], i * CP + n * 8 + qj, x[2 * n] * sc, x[2 * n + 1] * sc);
    if ((lane & 3) == 0) m.fp[i] = pow2_unscale(e);
  }
}

// One warp: rows [16 r, 16 r + 16) of P transposed.
template <int DK, int LIMBS>
__device__ __forceinline__ void score_columns(const Gates& s, Pairs& m, const __half* qp, const __half* kp, int r, int lane) {
  constexpr int PITCH = DK + 8;
  float acc[4][4] = {};
  if (r == 0) rows_times_rows<DK, LIMBS>(reinterpret_cast<float(&)[2][4]>(acc[0]), kp, qp, lane);
  rows_times_rows<DK, LIMBS>(reinterpret_cast<float(&)[2][4]>(acc[2]), kp + r * 16 * PITCH, qp + 16 * PITCH, lane);
  const int gi = lane >> 2, qi = (lane & 3) * 2;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int j = r * 16 + gi + half * 8;
    const Token tj = s.token[j];
    float x[8], most = 0.0f;
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      const int i = (n >> 1) * 8 + qi + (n & 1);
      x[n] = 0.0f;
      if (n < 4 && r == 1) continue;
      const Token ti = s.token[i];
      if (j <= i) x[n] = acc[n >> 1][half * 2 + (n & 1)] * (s.fq[i] * tj.fk) * decay(ti, tj);
      most = fmaxf(most, fabsf(x[n]));
    }
    most = quad_max(most);
    const int e = pow2_exp(most);
    const float sc = pow2_scale(e);
#pragma unroll
    for (int n = 0; n < 4; ++n) store_split(m.p[0], m.p[1], j * CP + n * 8 + qi, x[2 * n] * sc, x[2 * n + 1] * sc);
    if ((lane & 3) == 0) m.fp[j] = pow2_unscale(e);
  }
}

// All warps: the three kinds of matrices, spread over the warps (P only where it is asked for).  halves: 1 where
// the chunk has no tokens past the 16th; nothing of the second half is made then, nor read (forward: 8192 rollouts of
// 16 tokens 650 -> 560 us, 4096 of 32 tokens 342 -> 344 us; the backward pass always takes 2, because its whole
// chunks lost 5 % to the branches).
template <int DK, int NW, int LIMBS, bool BACKWARD>
__device__ __forceinline__ void pair_matrices(Gates& s, Pairs& m, Squares& q, Gram* gram, const __half* qp, const __half* kp, bool scores, int halves, int warp,
                                              int lane) {
#pragma unroll 1
  for (int job = warp; job < 4; job += NW) {
    if (job == 0) {
      diagonal_inverses<DK, LIMBS>(s, m, q, gram, kp, halves, lane);
    } else if (job < 3) {
      if (!scores || (halves == 1 && job == 1)) continue;
      if (BACKWARD) score_columns<DK, LIMBS>(s, m, qp, kp, job - 1, lane);
      else score_rows<DK, LIMBS>(s, m, qp, kp, 2 - job, lane);
    } else {
      if (halves == 2) lower_block<DK, LIMBS>(s, m, gram, kp, lane);
      join_factors(s, lane);
    }
  }
}

// One warp's 16 value channels: W^T = E^T (I + N)^-T, in place.  e: [4][4] accumulator tiles, E^T[channel][token].
__device__ __forceinline__ void times_block(float (&out)[2][4], const float (&t0)[4], const float (&t1)[4], const __half* hi,
                                            const __half* lo, bool rows, int lane, float& f0, float& f1) {
  const float m0 = quad_max(fmaxf(fmaxf(fabsf(t0[0]), fabsf(t0[1])), fmaxf(fabsf(t1[0]), fabsf(t1[1]))));
  const float m1 = quad_max(fmaxf(fmaxf(fabsf(t0[2]), fabsf(t0[3])), fmaxf(fabsf(t1[2]), fabsf(t1[3]))));
  const int e0 = pow2_exp(m0), e1 = pow2_exp(m1);
  f0 = pow2_unscale(e0), f1 = pow2_unscale(e1);
  uint32_t ah[4], al[4], bh[4], bl[4];
  split_a(ah, al, t0, t1, pow2_scale(e0), pow2_scale(e1));
  if (rows) b_rows(bh, hi, TP, lane), b_rows(bl, lo, TP, lane);
  else b_cols(bh, hi, TP, lane), b_cols(bl, lo, TP, lane);
#pragma unroll
  for (int n = 0; n < 2; ++n) {
#pragma unroll
    for (int x = 0; x < 4; ++x) out[n][x] = 0.0f;
    mma(out[n], ah, bh[2 * n], bh[2 * n + 1]);
    mma(out[n], al, bh[2 * n], bh[2 * n + 1]);
    mma(out[n], ah, bl[2 * n], bl[2 * n + 1]);
  }
}

__device__ __forceinline__ void solve_forward(float (&e)[4][4], const Pairs& m, int halves, int lane) {
  float f0, f1, x[2][4];
  times_block(x, e[0], e[1], m.t[0], m.t[1], true, lane, f0, f1);  // W_0 = E_0 T_00^T
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int c = 0; c < 4; ++c) e[n][c] = x[n][c] * ((c < 2 ? f0 : f1) * m.ft[0]);
  if (halves == 1) return;
  times_block(x, e[0], e[1], m.n[0], m.n[1], true, lane, f0, f1);  // E_1 -= W_0 N_10^T
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int c = 0; c < 4; ++c) e[2 + n][c] -= x[n][c] * ((c < 2 ? f0 : f1) * m.fn);
  times_block(x, e[2], e[3], m.t[0] + 16 * TP, m.t[1] + 16 * TP, true, lane, f0, f1);  // W_1 = E_1 T_11^T
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int c = 0; c < 4; ++c) e[2 + n][c] = x[n][c] * ((c < 2 ? f0 : f1) * m.ft[1]);
}

// dE^T = dW^T (I + N)^-1, in place: from the chunk's end to its begin.
__device__ __forceinline__ void solve_backward(float (&e)[4][4], const Pairs& m, int lane) {
  float f0, f1, x[2][4];
  times_block(x, e[2], e[3], m.t[0] + 16 * TP, m.t[1] + 16 * TP, false, lane, f0, f1);
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int c = 0; c < 4; ++c) e[2 + n][c] = x[n][c] * ((c < 2 ? f0 : f1) * m.ft[1]);
  times_block(x, e[2], e[3], m.n[0], m.n[1], false, lane, f0, f1);
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int c = 0; c < 4; ++c) e[n][c] -= x[n][c] * ((c < 2 ? f0 : f1) * m.fn);
  times_block(x, e[0], e[1], m.t[0], m.t[1], false, lane, f0, f1);
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int c = 0; c < 4; ++c) e[n][c] = x[n][c] * ((c < 2 ? f0 : f1) * m.ft[0]);
}

// The largest magnitude of the thread's two rows over all tiles of an accumulator array.
template <int N>
__device__ __forceinline__ void row_exps(const float (&t)[N][4], int& e0, int& e1) {
  float m0 = 0.0f, m1 = 0.0f;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    m0 = fmaxf(m0, fmaxf(fabsf(t[n][0]), fabsf(t[n][1])));
    m1 = fmaxf(m1, fmaxf(fabsf(t[n][2]), fabsf(t[n][3])));
  }
  e0 = pow2_exp(quad_max(m0)), e1 = pow2_exp(quad_max(m1));
}
// ... and whether all of the thread's values are finite.
template <int N>
__device__ __forceinline__ bool row_exps_finite(const float (&t)[N][4], int& e0, int& e1) {
  float m0 = 0.0f, m1 = 0.0f;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    m0 = max_nan(m0, max_nan(fabsf(t[n][0]), fabsf(t[n][1])));
    m1 = max_nan(m1, max_nan(fabsf(t[n][2]), fabsf(t[n][3])));
  }
  const bool finite = max_nan(m0, m1) < INFINITY;
  e0 = pow2_exp(quad_max(m0)), e1 = pow2_exp(quad_max(m1));
  return finite;
}
// V^T[channel][token] of a warp's 16 channels from the rows [C][pitch].
__device__ __forceinline__ void load_values(float (&t)[4][4], const __nv_bfloat16* v, int pitch, int lane) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {  // 16 tokens: tiles 2 h, 2 h + 1
    uint32_t r[4];
    ldsm4t(r, smem_at(v + (h * 16 + (lane >> 4) * 8 + (lane & 7)) * pitch + ((lane >> 3) & 1) * 8));
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      t[2 * h + (x >> 1)][(x & 1) * 2] = __uint_as_float(r[x] << 16);
      t[2 * h + (x >> 1)][(x & 1) * 2 + 1] = __uint_as_float(r[x] & 0xffff0000u);
    }
  }
}
__device__ __forceinline__ void load_values(float (&t)[4][4], const float* v, int pitch, int lane) {
#pragma unroll
  for (int n = 0; n < 4; ++n)
#pragma unroll
    for (int x = 0; x < 4; ++x) t[n][x] = v[(n * 8 + (lane & 3) * 2 + (x & 1)) * pitch + (lane >> 2) + (x >> 1) * 8];
}
// A state [dk][dv] to and from a warp's transposed accumulators.
template <int DK, class F>
__device__ __forceinline__ void for_state(float (&st)[DK / 8][4], int dk, int dv, int c0, int lane, F f) {
  const int gi = lane >> 2, qj = (lane & 3) * 2;
  if (dk == DK && dv % 16 == 0) {  // nothing to leave out
    if (c0 >= dv) return;
    int64_t at = int64_t(qj) * dv + c0 + gi;
#pragma unroll
    for (int n = 0; n < DK / 8; ++n, at += 8 * dv)
#pragma unroll
      for (int x = 0; x < 4; ++x) f(st[n][x], at + (x & 1 ? dv : 0) + (x >> 1) * 8);
  } else {
#pragma unroll
    for (int n = 0; n < DK / 8; ++n)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int c = c0 + gi + (x >> 1) * 8, r = n * 8 + qj + (x & 1);
        if (c < dv && r < dk) f(st[n][x], int64_t(r) * dv + c);
      }
  }
}

// out[4][4] += S^T X^T for the chunk's rows X (limb planes [C][DK + 8]), S scaled by s0, s1: [16 channels][C tokens].
template <int DK, int LIMBS>
__device__ __forceinline__ void state_times_rows(float (&out)[4][4], const uint32_t (&hi)[4], const uint32_t (&lo)[4],
                                                 const __half* x, int kk, int halves, int lane) {
  constexpr int PITCH = DK + 8, PLANE = C * PITCH;
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    if (n == 1 && halves == 1) break;
    uint32_t b[4];
    b_rows(b, x + n * 16 * PITCH + kk, PITCH, lane);
    mma(out[2 * n], hi, b[0], b[1]);
    mma(out[2 * n + 1], hi, b[2], b[3]);
    mma(out[2 * n], lo, b[0], b[1]);
    mma(out[2 * n + 1], lo, b[2], b[3]);
    if (LIMBS == 2) {
      b_rows(b, x + PLANE + n * 16 * PITCH + kk, PITCH, lane);
      mma(out[2 * n], hi, b[0], b[1]);
      mma(out[2 * n + 1], hi, b[2], b[3]);
    }
  }
}

// S^T <- keep S^T + A X, A^T[16 channels][C tokens] unscaled accumulator tiles, X rows [C][DK + 8].
template <int DK, int LIMBS>
__device__ __forceinline__ void state_update(float (&st)[DK / 8][4], float keep, const float (&a)[4][4], const __half* x, int halves,
                                             int lane) {
  constexpr int PITCH = DK + 8, PLANE = C * PITCH;
  int e0, e1;
  row_exps<4>(a, e0, e1);
  const float s0 = pow2_scale(e0), s1 = pow2_scale(e1), f0 = pow2_unscale(e0), f1 = pow2_unscale(e1);
  uint32_t hi[2][4], lo[2][4];
#pragma unroll
  for (int r = 0; r < 2; ++r) split_a(hi[r], lo[r], a[2 * r], a[2 * r + 1], s0, s1);
#pragma unroll
  for (int kk = 0; kk < DK; kk += 16) {
    float acc[2][4] = {};
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      if (r == 1 && halves == 1) break;
      uint32_t b[4];
      b_cols(b, x + r * 16 * PITCH + kk, PITCH, lane);
      mma(acc[0], hi[r], b[0], b[1]);
      mma(acc[1], hi[r], b[2], b[3]);
      mma(acc[0], lo[r], b[0], b[1]);
      mma(acc[1], lo[r], b[2], b[3]);
      if (LIMBS == 2) {
        b_cols(b, x + PLANE + r * 16 * PITCH + kk, PITCH, lane);
        mma(acc[0], hi[r], b[0], b[1]);
        mma(acc[1], hi[r], b[2], b[3]);
      }
    }
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float& y = st[kk / 8 + n][c];
        // a cleared state is zero whatever it held
        y = fmaf(acc[n][c], c < 2 ? f0 : f1, keep == 0.0f ? 0.0f : keep * y);
      }
  }
}

// Transposed tiles [16 channels][C tokens] of a warp to rows of `out`: bfloat16 pairs of tokens are transposed in the
// registers so that a lane writes neighbouring channels.
template <class T>
__device__ __forceinline__ void store_out(const float (&o)[4][4], T* out, int64_t stride, int64_t t0, int64_t lo, int64_t hi,
                                          int c0, int dv, bool pairs_ok, int lane) {
  const int gi = lane >> 2, qj = (lane & 3) * 2;
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const __nv_bfloat162 x = __floats2bfloat162_rn(o[n][half * 2], o[n][half * 2 + 1]);
        const uint32_t y = movm(*reinterpret_cast<const uint32_t*>(&x));
        const int64_t t = t0 + n * 8 + gi;
        const int c = c0 + half * 8 + qj;
        if (t >= lo && t < hi && c < dv) {
          T* at = out + t * stride + c;
          const __nv_bfloat162 z = *reinterpret_cast<const __nv_bfloat162*>(&y);
          if (pairs_ok) {
            *reinterpret_cast<__nv_bfloat162*>(at) = z;
          } else {
            at[0] = z.x;
            if (c + 1 < dv) at[1] = z.y;
          }
        }
      }
    } else {
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int64_t t = t0 + n * 8 + qj + (x & 1);
        const int c = c0 + gi + (x >> 1) * 8;
        if (t >= lo && t < hi && c < dv) out[t * stride + c] = o[n][x];
      }
    }
  }
}

// Padded widths of a call's kernels: key channels, and value channels in groups of 16, a warp each.
inline int key_width(const ZenoDeltaRule& p) { return p.key_dim <= 32 ? 32 : p.key_dim <= 64 ? 64 : 128; }
inline int value_groups(const ZenoDeltaRule& p) {
  const int nw = p.value_dim <= 32 ? 2 : p.value_dim <= 64 ? 4 : 8;
  return key_width(p) == 128 && nw < 4 ? 4 : nw;  // backward: a warp's share of the key channels is 64 at most
}

}  // namespace delta
}  // namespace zb
