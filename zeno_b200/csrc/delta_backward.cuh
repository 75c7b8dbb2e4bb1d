// Gradients of the gated delta rule over a rollout, chunked, from the last chunk to the first.
//
// With the forward chunk's quantities (S0, W, U = beta W, D, a, P as there), R the gradient of
// the state behind the chunk and dO that of its outputs (times the scale):
//   dU = P^T dO + D_C K R             (what outputs and later chunks ask of u)
//   (I + N)^T dE = beta dU,           dV = dE
//   X_ij = -D_ij dE_i . u_j (j < i),  M_ij = D_ij dO_i . u_j (j <= i)
//   dQ = a dO S0^T + M K
//   dK = [-a dE S0^T + X K] + [M^T Q + X^T K + D_C U R^T]
//   dbeta_j = dU_j . w_j - sum_i (dE_i . w_j) D_ij (k_i . k_j)
//   R <- a_C R + Q^T (a dO) - K^T (a dE)
// The log decays enter as exp(G_i) at a row's later token and exp(-G_j) at its earlier one, so
// dG_i = q_i . dq_i + k_i . dk_i[first bracket] - k_i . dk_i[second], the chunk's end adds <S_C, R> =
// sum_j u_j . (D_Cj R^T k_j) + a_C <S0, R>, and dg is the sum of dG from the token to its episode's end.
//
// Phase A as forward: a warp owns 16 value channels, everything transposed, R in its
// accumulators for the whole rollout.  Phase B sums over the value channels, so W, dE, S0
// and R pass through shared memory as limb planes, and a warp has 16 tokens and a share of
// the key channels.
//
// Few long rollouts are cut into segments here too (see the forward pass): all but the first are run
// for the R they leave alone, a walk back over the segments gives the R behind each, and all
// segments run at once for the gradients.
#pragma once
#include "delta_mma.cuh"

namespace zb {
namespace delta {
namespace {

template <int DK, int NW, class T>
struct BackwardSmem {
  static constexpr int L = In<T>::limbs;
  static constexpr int VC = 16 * NW;
  static constexpr int GROUPS = DK / (2 * DK / NW < 16 ? 16 : 2 * DK / NW);
  Gates gates;
  Gram gram;
  struct Early {  // up to phase A
    Pairs pairs;
    __align__(16) T v[C * (VC + 16 / int(sizeof(T)))];
  };
  struct Late {  // from the token-by-token gradients on: M and X with the rows' factors, later token by earlier one
    __align__(16) __half m[2][C * CP];
    __align__(16) __half x[2][C * CP];
  };
  __align__(16) unsigned char pair_space[sizeof(Early) > sizeof(Late) ? sizeof(Early) : sizeof(Late)];
  __align__(16) __half q[L][C * (DK + 8)];
  __align__(16) __half k[L][C * (DK + 8)];
  __align__(16) __half d_out[L][C * (VC + 8)];
  __align__(16) __half w[2][VC * CP];            // W^T [channel][token]; before, the squares on their way to the inverses
  __align__(16) __half d_e[2][VC * CP];          // dE^T
  __align__(16) __half state[2][VC * (DK + 8)];  // S0^T, then R^T [channel][key channel]
  float fm[3], fx[3];                            // scales of the blocks (0,0), (1,0), (1,1) of M and X
  float fk[C], inv_fk[C], inv_fq[C];
  float beta_part[NW][C], beta_pairs[2][C];
  float dot_q[GROUPS][C], dot_row[GROUPS][C], dot_col[GROUPS][C];
  float end_part[NW];
  unsigned most_out, most_state, most_r, most_w, most_e;  // largest finite magnitudes (float bits)
  int r_bad;
};

// Takes a warp's largest magnitude to `at` (float bits), and notes in `bad` if one is not finite.
__device__ __forceinline__ void raise(unsigned* at, int& bad, float x) {
  unsigned u = __reduce_max_sync(kAll, __float_as_uint(x));  // NaN and infinity above all others
  if (u >= 0x7f800000u) {
    bad = 1;
    u = __reduce_max_sync(kAll, fabsf(x) < INFINITY ? __float_as_uint(x) : 0u);
  }
  if ((threadIdx.x & 31) == 0) atomicMax(at, u);
}

template <int N>
__device__ __forceinline__ float most_of(const float (&t)[N][4]) {  // NaN where one is
  float m = 0.0f;
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int x = 0; x < 4; ++x) m = max_nan(m, fabsf(t[n][x]));
  return m;
}

// A warp's transposed tiles (channel rows) to limb planes of the given pitch.
template <int N>
__device__ __forceinline__ void store_planes(__half* hi, __half* lo, int pitch, const float (&t)[N][4], float sc, int warp, int lane) {
  const int gi = lane >> 2, qj = (lane & 3) * 2;
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int half = 0; half < 2; ++half)
      store_split(hi, lo, (warp * 16 + gi + half * 8) * pitch + n * 8 + qj, t[n][2 * half] * sc, t[n][2 * half + 1] * sc);
}

// acc += A B for 16-wide pieces: A limbs ah (al where LA == 2), B limbs bh (bl where LB == 2).
template <int LA, int LB>
__device__ __forceinline__ void mma2(float (&acc0)[4], float (&acc1)[4], const uint32_t (&ah)[4], const uint32_t (&al)[4],
                                     const uint32_t (&bh)[4], const uint32_t (&bl)[4]) {
  mma(acc0, ah, bh[0], bh[1]);
  mma(acc1, ah, bh[2], bh[3]);
  if (LA == 2) mma(acc0, al, bh[0], bh[1]), mma(acc1, al, bh[2], bh[3]);
  if (LB == 2) mma(acc0, ah, bl[0], bl[1]), mma(acc1, ah, bl[2], bl[3]);
}

// The blocks of M or X that rows [16 r, 16 r + 16) meet, times rows of K or Q (limb planes), into
// 16 x 8 N tiles from column c0 on.  TRANSPOSED: the rows are the earlier tokens.  Each block has a scale
// of its own, each row of the result a factor.
template <int DK, int N, int L, bool TRANSPOSED>
__device__ __forceinline__ void pairs_times_rows(float (&out)[N][4], const __half* plane, const float* scales, const float* row_factor,
                                                 const __half* x, int r, int c0, int lane) {
  constexpr int PITCH = DK + 8, PLANE = C * PITCH;
  const float r0 = row_factor[r * 16 + (lane >> 2)], r1 = row_factor[r * 16 + (lane >> 2) + 8];
#pragma unroll 1
  for (int j = TRANSPOSED ? r : 0; j < (TRANSPOSED ? 2 : r + 1); ++j) {
    uint32_t ah[4], al[4];
    if (TRANSPOSED) {
      a_cols(ah, plane + j * 16 * CP + r * 16, CP, lane);
      a_cols(al, plane + C * CP + j * 16 * CP + r * 16, CP, lane);
    } else {
      a_rows(ah, plane + r * 16 * CP + j * 16, CP, lane);
      a_rows(al, plane + C * CP + r * 16 * CP + j * 16, CP, lane);
    }
    const float f = scales[r + j], f0 = f * r0, f1 = f * r1;
#pragma unroll
    for (int n = 0; n < N; n += 2) {
      float acc[2][4] = {};
      uint32_t bh[4], bl[4] = {};
      b_cols(bh, x + j * 16 * PITCH + c0 + n * 8, PITCH, lane);
      if (L == 2) b_cols(bl, x + PLANE + j * 16 * PITCH + c0 + n * 8, PITCH, lane);
      mma2<2, L>(acc[0], acc[1], ah, al, bh, bl);
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int c = 0; c < 4; ++c) out[n + u][c] = fmaf(acc[u][c], c < 2 ? f0 : f1, out[n + u][c]);
    }
  }
}

// Rows of a [tokens] x [channels] operand times the state planes.  LA limbs; COLS: stored [channel][token].
template <int DK, int NW, int N, int LA, bool COLS>
__device__ __forceinline__ void rows_times_state(float (&acc)[N][4], const __half* a, int a_pitch, int a_plane, const __half* state,
                                                 int r, int c0, int lane) {
  constexpr int PITCH = DK + 8, PLANE = 16 * NW * PITCH;
#pragma unroll 2
  for (int kk = 0; kk < 16 * NW; kk += 16) {
    uint32_t ah[4], al[4] = {};
    if (COLS) a_cols(ah, a + kk * a_pitch + r * 16, a_pitch, lane);
    else a_rows(ah, a + r * 16 * a_pitch + kk, a_pitch, lane);
    if (LA == 2) {
      if (COLS) a_cols(al, a + a_plane + kk * a_pitch + r * 16, a_pitch, lane);
      else a_rows(al, a + a_plane + r * 16 * a_pitch + kk, a_pitch, lane);
    }
#pragma unroll
    for (int n = 0; n < N; n += 2) {
      uint32_t bh[4], bl[4];
      b_cols(bh, state + kk * PITCH + c0 + n * 8, PITCH, lane);
      b_cols(bl, state + PLANE + kk * PITCH + c0 + n * 8, PITCH, lane);
      mma2<LA, 2>(acc[n], acc[n + 1], ah, al, bh, bl);
    }
  }
}

// Sum over a row's channels of x times the normalised row of K or Q, over the quad: rows gi and gi + 8.
template <int DK, int N, int L>
__device__ __forceinline__ void row_dots(const float (&x)[N][4], const __half* plane, const float* factor, int r, int c0, int lane,
                                         float& d0, float& d1) {
  constexpr int PITCH = DK + 8, PLANE = C * PITCH;
  const int gi = lane >> 2, qj = (lane & 3) * 2;
  d0 = d1 = 0.0f;
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const __half* at = plane + (r * 16 + gi + half * 8) * PITCH + c0 + n * 8 + qj;
      float2 y = __half22float2(*reinterpret_cast<const __half2*>(at));
      if (L == 2) {
        const float2 z = __half22float2(*reinterpret_cast<const __half2*>(at + PLANE));
        y.x += z.x, y.y += z.y;
      }
      float& d = half ? d1 : d0;
      d = fmaf(x[n][2 * half], y.x, fmaf(x[n][2 * half + 1], y.y, d));
    }
  d0 += __shfl_xor_sync(kAll, d0, 1), d1 += __shfl_xor_sync(kAll, d1, 1);
  d0 += __shfl_xor_sync(kAll, d0, 2), d1 += __shfl_xor_sync(kAll, d1, 2);
  d0 *= factor[r * 16 + gi], d1 *= factor[r * 16 + gi + 8];
}

// Gradient of a row of Q or K through its norm, written to `out` (rows of the call's type, or
// 32-bit rows of the shared heads' workspace).
template <int DK, int N, int L, class O>
__device__ __forceinline__ void write_rows(const float (&x)[N][4], const __half* plane, const float* factor, const float* norm,
                                           bool normalize, const float (*dots)[C], int groups, const float (*dots2)[C], O* out,
                                           int64_t stride, int64_t t0, int64_t lo, int64_t hi, int r, int c0, int dk, bool pairs_ok,
                                           int lane) {
  constexpr int PITCH = DK + 8, PLANE = C * PITCH;
  const int gi = lane >> 2, qj = (lane & 3) * 2;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int row = r * 16 + gi + half * 8;
    const int64_t t = t0 + row;
    if (t < lo || t >= hi) continue;
    float dot = 0.0f, n1 = 1.0f;
    if (normalize) {
      for (int g = 0; g < groups; ++g) dot += dots[g][row];
      if (dots2)
        for (int g = 0; g < groups; ++g) dot += dots2[g][row];
      n1 = norm[row];
      dot *= factor[row];
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int c = c0 + n * 8 + qj;
      float y0 = x[n][2 * half], y1 = x[n][2 * half + 1];
      if (normalize) {
        const __half* at = plane + row * PITCH + c;
        float2 y = __half22float2(*reinterpret_cast<const __half2*>(at));
        if (L == 2) {
          const float2 z = __half22float2(*reinterpret_cast<const __half2*>(at + PLANE));
          y.x += z.x, y.y += z.y;
        }
        y0 = n1 * (y0 - y.x * dot), y1 = n1 * (y1 - y.y * dot);
      }
      O* at = out + t * stride + c;
      if constexpr (sizeof(O) == 2) {
        if (pairs_ok && c + 1 < dk) {
          *reinterpret_cast<__nv_bfloat162*>(at) = __floats2bfloat162_rn(y0, y1);
        } else {
          if (c < dk) at[0] = __float2bfloat16_rn(y0);
          if (c + 1 < dk) at[1] = __float2bfloat16_rn(y1);
        }
      } else {
        if (pairs_ok && c + 1 < dk) {
          *reinterpret_cast<float2*>(at) = make_float2(y0, y1);
        } else {
          if (c < dk) at[0] = y0;
          if (c + 1 < dk) at[1] = y1;
        }
      }
    }
  }
}

template <class T>
__device__ __forceinline__ bool even(const ZenoTensor& t, int width) {
  return width % 2 == 0 && reinterpret_cast<uintptr_t>(t.data) % (2 * sizeof(T)) == 0 &&
         ((t.stride[0] | t.stride[1] | t.stride[2]) & 1) == 0;
}

// Blocks of an SM: 384 threads of it where the registers allow (64 x 64, 4096 x 32 tokens: 1.9 ms with 256 threads,
// before other changes), 256 where a warp's share of the key channels or the state takes 64 registers.
template <int DK, int NW>
constexpr int kBlocks = (DK == 32 || (DK == 64 && NW > 2) ? 384 : 256) / (NW * 32);

struct BackSplit {
  uint32_t segments, chunks;  // chunks of a segment
  bool r_only;                // no gradients: the R in front of each segment, from zero behind it (the last: from d_final)
  float* n;                   // ... [batch * heads][segments][dk][dv]
  const float* state;         // else, with more than one segment: the R behind each
};

// OUT: type of the dq and dk rows (float: the workspace of shared heads, reduced afterwards).
template <int DK, int NW, class T, class OUT>
__global__ void __launch_bounds__(NW * 32, kBlocks<DK, NW>)
delta_backward_kernel(const __grid_constant__ ZenoDeltaRule p, const __grid_constant__ ZenoDeltaRuleGrads d,
                      const __grid_constant__ BackSplit sp) {
  extern __shared__ __align__(16) unsigned char raw[];
  using Smem = BackwardSmem<DK, NW, T>;
  constexpr int L = In<T>::limbs, VC = 16 * NW, VP = VC + 16 / int(sizeof(T)), DP = VC + 8, SP = DK + 8;
  Smem& sm = *reinterpret_cast<Smem*>(raw);
  typename Smem::Early& early = *reinterpret_cast<typename Smem::Early*>(sm.pair_space);
  typename Smem::Late& late = *reinterpret_cast<typename Smem::Late*>(sm.pair_space);
  Squares& squares = *reinterpret_cast<Squares*>(sm.w[0]);
  static_assert(sizeof(Squares) <= sizeof(sm.w), "the squares fit in W's place");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int gi = lane >> 2, qj = (lane & 3) * 2;
  const uint32_t h = blockIdx.x % p.value_heads, b = blockIdx.x / p.value_heads;
  const int dk = int(p.key_dim), dv = int(p.value_dim);
  const int c0 = warp * 16;
  const Rows<T> rows = rows_of<T>(p, b, h);
  const T* d_out = static_cast<const T*>(d.d_out.data) + int64_t(b) * d.d_out.stride[0] + int64_t(h) * d.d_out.stride[2];
  const bool vec_do = vec_ok<T>(d.d_out, dv);
  T* d_v = static_cast<T*>(d.d_v.data) + int64_t(b) * d.d_v.stride[0] + int64_t(h) * d.d_v.stride[2];
  const bool dv_pairs = even<T>(d.d_v, dv);
  // with OUT float for a 16-bit type (or shared heads) dq and dk have a row for each value head
  OUT* d_q = static_cast<OUT*>(d.d_q.data) + int64_t(b) * d.d_q.stride[0] + int64_t(h) * d.d_q.stride[2];
  OUT* d_k = static_cast<OUT*>(d.d_k.data) + int64_t(b) * d.d_k.stride[0] + int64_t(h) * d.d_k.stride[2];
  const bool dq_pairs = even<OUT>(d.d_q, dk), dk_pairs = even<OUT>(d.d_k, dk);
  float* d_g = static_cast<float*>(d.d_g.data) + int64_t(b) * d.d_g.stride[0] + int64_t(h) * d.d_g.stride[2];
  float* d_beta = static_cast<float*>(d.d_beta.data) + int64_t(b) * d.d_beta.stride[0] + int64_t(h) * d.d_beta.stride[2];
  const int64_t state_at = int64_t(blockIdx.x) * dk * dv;

  const bool r_only = sp.r_only;
  const uint32_t segment = blockIdx.z;
  if (r_only && segment == 0) return;
  const int64_t segment_at = (int64_t(blockIdx.x) * sp.segments + segment) * dk * dv;
  const float* r_from = !r_only && sp.segments > 1                          ? sp.state + segment_at
                        : d.d_final && segment + 1 == sp.segments ? d.d_final + state_at
                                                                  : nullptr;
  float* r_to = r_only ? sp.n + segment_at : d.d_initial && segment == 0 ? d.d_initial + state_at : nullptr;

  float rt[DK / 8][4] = {};  // R^T
  if (r_from) for_state<DK>(rt, dk, dv, c0, lane, [&](float& x, int64_t at) { x = r_from[at]; });
  bool has_r = r_from != nullptr;  // R is not zero
  if (tid == 0) sm.gates.bad = 0, sm.gates.state_bad = 0, sm.r_bad = 0, sm.most_out = sm.most_state = sm.most_r = sm.most_w = sm.most_e = 0;
  __syncthreads();
  if (has_r) raise(&sm.most_r, sm.r_bad, most_of<DK / 8>(rt));

  const int64_t T_ = p.tokens;
  const int64_t chunks = (T_ + C - 1) / C;
  const int64_t first = int64_t(segment) * sp.chunks, last = min(chunks, first + sp.chunks);
  for (int64_t chunk = last - 1; chunk >= first; --chunk) {
    const int64_t t0 = chunk * C, t1 = min(t0 + C, T_);
    for (int64_t hi = t1; hi > t0;) {
      int64_t lo = t0;
      // ---- loads
      bool has_state = !r_only && (chunk > 0 || p.initial_state != nullptr);
      float st[DK / 8][4] = {};  // S0^T
      if (r_only) {
      } else if (chunk > 0) {
        const float4* from = reinterpret_cast<const float4*>(p.saved + ((int64_t(blockIdx.x) * (chunks - 1) + chunk - 1) * VC + c0) * DK);
#pragma unroll
        for (int n = 0; n < DK / 8; ++n) {
          const float4 x = __ldcs(from + n * 32 + lane);
          st[n][0] = x.x, st[n][1] = x.y, st[n][2] = x.z, st[n][3] = x.w;
        }
      } else if (has_state) {
        for_state<DK>(st, dk, dv, c0, lane, [&](float& x, int64_t at) { x = p.initial_state[state_at + at]; });
      }
      Eight raw_out[2];
#pragma unroll 1
      for (;;) {
        GateIn gates{};
        if (warp == 0) gates = fetch_gates(p, rows.g, rows.beta, rows.reset, t0, lo, hi, lane);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int j = tid + u * NW * 32, row = j / (VC / 8), at = (j % (VC / 8)) * 8;
          const int64_t t = t0 + row;
          raw_out[u] = Eight{};
          if (t >= lo && t < hi && at < dv) raw_out[u] = fetch8(d_out + t * d.d_out.stride[1] + at, dv - at, vec_do);
        }
        load_rows<DK, NW, T, true>(sm.gates, p, rows, sm.q[0], sm.k[0], early.v, 0, r_only ? 0 : dv, t0, lo, hi, tid);
        if (warp == 0) scan_gates(sm.gates, gates, lane);
        float most = 0.0f;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float x[8];
          unpack8<T>(x, raw_out[u]);
#pragma unroll
          for (int i = 0; i < 8; ++i) most = max_nan(most, fabsf(x[i]));
        }
        raise(&sm.most_out, sm.gates.bad, most);
        if (has_state) raise(&sm.most_state, sm.gates.state_bad, most_of<DK / 8>(st));
        __syncthreads();
        if (sm.gates.bad && p.normalize) {
          mend_norms<NW, T>(sm.gates, p, rows, t0, lo, hi, tid);
          __syncthreads();
        }
        // A value that is not finite must not reach another episode through a product with
        // zero: such a chunk is taken episode by episode.
        if (lo > t0 || !(sm.gates.bad || sm.gates.state_bad || sm.r_bad) || (sm.gates.marks >> 1) == 0) break;
        lo = t0 + 31 - __clz(int(sm.gates.marks));
        has_state = false;  // the episode's first token drops it
        __syncthreads();
        if (tid == 0) sm.most_out = 0;
        __syncthreads();
      }
      if (chunk > first) {  // the next chunk on its way
        prefetch_rows<NW>(p, rows, t0 - C, 0, tid);
        if (tid < C) {
          const T* at = d_out + (t0 - C + tid) * d.d_out.stride[1];
          for (int c = 0; c < dv; c += 128 / int(sizeof(T))) prefetch(at + c);
        }
        if (chunk > 1 && !r_only) {
          const float* at = p.saved + ((int64_t(blockIdx.x) * (chunks - 1) + chunk - 2) * VC) * DK;
          for (int c = tid * 32; c < VC * DK; c += NW * 32 * 32) prefetch(at + c);
        }
      }
      const int e_out = pow2_exp(__uint_as_float(sm.most_out));
      const float u_out = pow2_unscale(e_out) * p.scale;
      {
        const float sc = pow2_scale(e_out);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int j = tid + u * NW * 32, row = j / (VC / 8), at = (j % (VC / 8)) * 8;
          float x[8];
          unpack8<T>(x, raw_out[u]);
          uint4 h4, l4;
          split(x[0] * sc, x[1] * sc, h4.x, l4.x);
          split(x[2] * sc, x[3] * sc, h4.y, l4.y);
          split(x[4] * sc, x[5] * sc, h4.z, l4.z);
          split(x[6] * sc, x[7] * sc, h4.w, l4.w);
          *reinterpret_cast<uint4*>(&sm.d_out[0][row * DP + at]) = h4;
          if (L == 2) *reinterpret_cast<uint4*>(&sm.d_out[L - 1][row * DP + at]) = l4;
        }
      }
      if (tid < C) {
        const float fk = sm.gates.token[tid].fk;
        sm.fk[tid] = fk, sm.inv_fk[tid] = 1.0f / fk, sm.inv_fq[tid] = 1.0f / sm.gates.fq[tid];
      }
      pair_matrices<DK, NW, L, true>(sm.gates, early.pairs, squares, &sm.gram, sm.q[0], sm.k[0], true, 2, warp, lane);

      // S0^T times K^T as the limbs are made; they also go to shared memory, for phase B
      float w[4][4] = {}, e[4][4] = {};
      const float keep = sm.gates.keep;
      float end = 0.0f, u_state = 0.0f;  // end: this warp's part of <S_C, R>
      if (has_state) {
        if (has_r && keep != 0.0f) {
#pragma unroll
          for (int n = 0; n < DK / 8; ++n)
#pragma unroll
            for (int x = 0; x < 4; ++x) end = fmaf(st[n][x], rt[n][x], end);
          end *= keep;
        }
        const int ex = pow2_exp(__uint_as_float(sm.most_state));
        const float sc = pow2_scale(ex);
        u_state = pow2_unscale(ex);
#pragma unroll
        for (int kk = 0; kk < DK; kk += 16) {
          uint32_t ah[4], al[4];
          split_a(ah, al, st[kk / 8], st[kk / 8 + 1], sc, sc);
          state_times_rows<DK, L>(w, ah, al, sm.k[0], kk, 2, lane);
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            const int at = (c0 + gi + (h & 1) * 8) * SP + kk + (h >> 1) * 8 + qj;
            *reinterpret_cast<uint32_t*>(&sm.state[0][at]) = ah[h];
            *reinterpret_cast<uint32_t*>(&sm.state[1][at]) = al[h];
          }
        }
      }
      const int e_r = pow2_exp(__uint_as_float(sm.most_r));
      const float u_r = pow2_unscale(e_r);
      if (has_r) {
        const float sc = pow2_scale(e_r);
#pragma unroll
        for (int kk = 0; kk < DK; kk += 16) {
          uint32_t ah[4], al[4];
          split_a(ah, al, rt[kk / 8], rt[kk / 8 + 1], sc, sc);
          state_times_rows<DK, L>(e, ah, al, sm.k[0], kk, 2, lane);
        }
      }
      __syncthreads();

      // ---- phase A: this warp's value channels
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const float2 zk = *reinterpret_cast<const float2*>(&sm.gates.zk[n * 8 + qj]);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float z = x & 1 ? zk.y : zk.x;
          e[n][x] = z == 0.0f ? 0.0f : e[n][x] * (u_r * z);
        }
      }
      if (!r_only) {
        float v[4][4];
        load_values(v, early.v + c0, VP, lane);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const float2 ak = *reinterpret_cast<const float2*>(&sm.gates.ak[n * 8 + qj]);
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const float a = x & 1 ? ak.y : ak.x;
            w[n][x] = a == 0.0f ? v[n][x] : fmaf(-w[n][x], u_state * a, v[n][x]);
          }
        }
        solve_forward(w, early.pairs, 2, lane);
        if (has_r) {
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const float2 be = *reinterpret_cast<const float2*>(&sm.gates.beta[n * 8 + qj]);
#pragma unroll
            for (int x = 0; x < 4; ++x) end = fmaf(e[n][x], w[n][x] * (x & 1 ? be.y : be.x), end);
          }
#pragma unroll
          for (int m = 1; m < 32; m <<= 1) end += __shfl_xor_sync(kAll, end, m);
        }
        if (lane == 0) sm.end_part[warp] = end;
      }
      // dU^T += dO^T P
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float acc[2][4] = {};
#pragma unroll
        for (int i = r; i < 2; ++i) {
          uint32_t ah[4], al[4] = {}, bh[4], bl[4];
          a_cols(ah, sm.d_out[0] + i * 16 * DP + c0, DP, lane);
          if (L == 2) a_cols(al, sm.d_out[L - 1] + i * 16 * DP + c0, DP, lane);
          b_rows(bh, early.pairs.p[0] + r * 16 * CP + i * 16, CP, lane);
          b_rows(bl, early.pairs.p[1] + r * 16 * CP + i * 16, CP, lane);
          mma2<L, 2>(acc[0], acc[1], ah, al, bh, bl);
        }
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x)
            e[2 * r + n][x] = fmaf(acc[n][x], u_out * early.pairs.fp[r * 16 + n * 8 + qj + (x & 1)], e[2 * r + n][x]);
      }
      // dbeta: dU . w over this warp's channels; then dW = beta dU
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          if (!r_only) {
            float s = fmaf(e[n][x], w[n][x], e[n][x + 2] * w[n][x + 2]);
            s += __shfl_xor_sync(kAll, s, 4);
            s += __shfl_xor_sync(kAll, s, 8);
            s += __shfl_xor_sync(kAll, s, 16);
            if (gi == 0) sm.beta_part[warp][n * 8 + qj + x] = s;
          }
          const float be = sm.gates.beta[n * 8 + qj + x];
          e[n][x] *= be, e[n][x + 2] *= be;
        }
      solve_backward(e, early.pairs, lane);  // now dE^T
      if (!r_only) {
      store_out(e, d_v, d.d_v.stride[1], t0, lo, hi, c0, dv, dv_pairs, lane);
      int unused;
      raise(&sm.most_w, unused, most_of<4>(w));
      raise(&sm.most_e, unused, most_of<4>(e));
      __syncthreads();
      const int e_w = pow2_exp(__uint_as_float(sm.most_w)), e_e = pow2_exp(__uint_as_float(sm.most_e));
      const float u_w = pow2_unscale(e_w), u_e = pow2_unscale(e_e);
      store_planes<4>(sm.w[0], sm.w[1], CP, w, pow2_scale(e_w), warp, lane);
      store_planes<4>(sm.d_e[0], sm.d_e[1], CP, e, pow2_scale(e_e), warp, lane);
      __syncthreads();

      // ---- M and X, one 16 x 16 block a job: rows later tokens i, columns earlier tokens j
#pragma unroll 1
      for (int job = warp; job < 3; job += NW) {
        const int r = (job + 1) >> 1, c = job >> 1;  // (0,0), (1,0), (1,1)
        float am[2][4] = {}, ax[2][4] = {};
#pragma unroll 2
        for (int kk = 0; kk < VC; kk += 16) {
          uint32_t ah[4], al[4] = {}, bh[4], bl[4];
          b_cols(bh, sm.w[0] + kk * CP + c * 16, CP, lane);
          b_cols(bl, sm.w[1] + kk * CP + c * 16, CP, lane);
          a_rows(ah, sm.d_out[0] + r * 16 * DP + kk, DP, lane);
          if (L == 2) a_rows(al, sm.d_out[L - 1] + r * 16 * DP + kk, DP, lane);
          mma2<L, 2>(am[0], am[1], ah, al, bh, bl);
          a_cols(ah, sm.d_e[0] + kk * CP + r * 16, CP, lane);
          a_cols(al, sm.d_e[1] + kk * CP + r * 16, CP, lane);
          mma2<2, 2>(ax[0], ax[1], ah, al, bh, bl);
        }
        const float um = u_out * u_w, ux = -u_e * u_w;
        float mm = 0.0f, mx = 0.0f, db[4] = {};
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int i = r * 16 + gi + half * 8;
          const Token ti = sm.gates.token[i];
          const float fq = sm.gates.fq[i];
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const int j = c * 16 + (n >> 1) * 8 + qj + (n & 1);
            const Token tj = sm.gates.token[j];
            float& ym = am[n >> 1][half * 2 + (n & 1)];
            float& yx = ax[n >> 1][half * 2 + (n & 1)];
            const float f = j <= i ? sm.gates.beta[j] * decay(ti, tj) * tj.fk : 0.0f;
            const float x = yx * ux;  // -dE_i . w_j
            if (j < i) db[n] = fmaf(x, sm.gram.at[i][j], db[n]);
            ym = j <= i ? ym * um * (f * fq) : 0.0f;
            yx = j < i ? x * (f * ti.fk) : 0.0f;
            mm = fmaxf(mm, fabsf(ym)), mx = fmaxf(mx, fabsf(yx));
          }
        }
#pragma unroll
        for (int m = 1; m < 32; m <<= 1) {
          mm = fmaxf(mm, __shfl_xor_sync(kAll, mm, m)), mx = fmaxf(mx, __shfl_xor_sync(kAll, mx, m));
          if (m >= 4) {
#pragma unroll
            for (int n = 0; n < 4; ++n) db[n] += __shfl_xor_sync(kAll, db[n], m);
          }
        }
        if (gi == 0) {  // of the earlier tokens: block column 0 has two blocks
#pragma unroll
          for (int n = 0; n < 4; ++n) sm.beta_pairs[r][c * 16 + (n >> 1) * 8 + qj + (n & 1)] = db[n];
        }
        const int em = pow2_exp(mm), ex = pow2_exp(mx);
        const float sm_m = pow2_scale(em), sm_x = pow2_scale(ex);
        if (lane == 0) sm.fm[job] = pow2_unscale(em), sm.fx[job] = pow2_unscale(ex);
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const int at = (r * 16 + gi + half * 8) * CP + c * 16 + n * 8 + qj;
            store_split(late.m[0], late.m[1], at, am[n][2 * half] * sm_m, am[n][2 * half + 1] * sm_m);
            store_split(late.x[0], late.x[1], at, ax[n][2 * half] * sm_x, ax[n][2 * half + 1] * sm_x);
          }
      }
      __syncthreads();

      // ---- phase B: 16 tokens and a share of the key channels
      constexpr int DKW = 2 * DK / NW < 16 ? 16 : 2 * DK / NW, N = DKW / 8, GROUPS = DK / DKW;
      const int r = warp & 1, group = warp >> 1, k0 = group * DKW;
      const bool works = group < GROUPS;
      float gq[N][4] = {}, g_row[N][4] = {}, g_col[N][4] = {};
      if (works) {
        if (has_state) {
          const float a0 = sm.gates.carried[r * 16 + gi], a1 = sm.gates.carried[r * 16 + gi + 8];
          float acc[N][4] = {};
          rows_times_state<DK, NW, N, L, false>(acc, sm.d_out[0], DP, C * DP, sm.state[0], r, k0, lane);
#pragma unroll
          for (int n = 0; n < N; ++n)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const float a = x < 2 ? a0 : a1;
              gq[n][x] = a == 0.0f ? 0.0f : acc[n][x] * (a * u_out * u_state);
              acc[n][x] = 0.0f;
            }
          rows_times_state<DK, NW, N, 2, true>(acc, sm.d_e[0], CP, VC * CP, sm.state[0], r, k0, lane);
#pragma unroll
          for (int n = 0; n < N; ++n)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const float a = x < 2 ? a0 : a1;
              g_row[n][x] = a == 0.0f ? 0.0f : acc[n][x] * (-a * u_e * u_state);
            }
        }
        pairs_times_rows<DK, N, L, false>(gq, late.m[0], sm.fm, sm.inv_fq, sm.k[0], r, k0, lane);
        pairs_times_rows<DK, N, L, false>(g_row, late.x[0], sm.fx, sm.inv_fk, sm.k[0], r, k0, lane);
        pairs_times_rows<DK, N, L, true>(g_col, late.m[0], sm.fm, sm.inv_fk, sm.q[0], r, k0, lane);
        pairs_times_rows<DK, N, L, true>(g_col, late.x[0], sm.fx, sm.inv_fk, sm.k[0], r, k0, lane);
      }
      if (has_r) {
        if (has_state) __syncthreads();
        store_planes<DK / 8>(sm.state[0], sm.state[1], SP, rt, pow2_scale(e_r), warp, lane);
        __syncthreads();
      }
      if (works) {
        const int i0 = r * 16 + gi;
        if (has_r) {
          float acc[N][4] = {};
          rows_times_state<DK, NW, N, 2, true>(acc, sm.w[0], CP, VC * CP, sm.state[0], r, k0, lane);
          const float u = u_w * u_r;
          const float z0 = sm.gates.to_end[i0] * sm.gates.beta[i0] * u, z1 = sm.gates.to_end[i0 + 8] * sm.gates.beta[i0 + 8] * u;
#pragma unroll
          for (int n = 0; n < N; ++n)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const float z = x < 2 ? z0 : z1;
              if (z != 0.0f) g_col[n][x] = fmaf(acc[n][x], z, g_col[n][x]);
            }
        }
        float x0, x1;
        row_dots<DK, N, L>(gq, sm.q[0], sm.gates.fq, r, k0, lane, x0, x1);
        if ((lane & 3) == 0) sm.dot_q[group][i0] = x0, sm.dot_q[group][i0 + 8] = x1;
        row_dots<DK, N, L>(g_row, sm.k[0], sm.fk, r, k0, lane, x0, x1);
        if ((lane & 3) == 0) sm.dot_row[group][i0] = x0, sm.dot_row[group][i0 + 8] = x1;
        row_dots<DK, N, L>(g_col, sm.k[0], sm.fk, r, k0, lane, x0, x1);
        if ((lane & 3) == 0) sm.dot_col[group][i0] = x0, sm.dot_col[group][i0 + 8] = x1;
      }
      __syncthreads();
      if (works) {
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x) g_row[n][x] += g_col[n][x];
        write_rows<DK, N, L, OUT>(gq, sm.q[0], sm.gates.fq, sm.gates.nq, p.normalize, sm.dot_q, GROUPS, nullptr, d_q, d.d_q.stride[1],
                                  t0, lo, hi, r, k0, dk, dq_pairs, lane);
        write_rows<DK, N, L, OUT>(g_row, sm.k[0], sm.fk, sm.gates.nk, p.normalize, sm.dot_row, GROUPS, sm.dot_col, d_k,
                                  d.d_k.stride[1], t0, lo, hi, r, k0, dk, dk_pairs, lane);
      }
      if (warp == 0) {  // gates
        float dg = 0.0f, db = sm.beta_pairs[1][lane] + (lane < 16 ? sm.beta_pairs[0][lane] : 0.0f);
        for (int g = 0; g < GROUPS; ++g) dg += sm.dot_q[g][lane] + sm.dot_row[g][lane] - sm.dot_col[g][lane];
        for (int v = 0; v < NW; ++v) db += sm.beta_part[v][lane];
        const int mine = sm.gates.token[lane].episode;
        if (lane == 31)
          for (int v = 0; v < NW; ++v) dg += sm.end_part[v];
        // sum over the later tokens of the same episode
#pragma unroll
        for (int m = 1; m < 32; m <<= 1) {
          const float y = __shfl_down_sync(kAll, dg, m);
          const int other = __shfl_down_sync(kAll, mine, m);
          if (lane + m < 32 && other == mine) dg += y;
        }
        const int64_t t = t0 + lane;
        if (t >= lo && t < hi) {
          d_g[t * d.d_g.stride[1]] = (sm.gates.marks >> lane) & 1 ? 0.0f : dg;
          d_beta[t * d.d_beta.stride[1]] = db;
        }
      }
      }

      // ---- R^T <- a_C R^T + (a dO)^T Q - (a dE)^T K, where something still asks for it
      const bool more = chunk > first || lo > t0 || r_to != nullptr;
      if (sm.gates.bad && (sm.gates.marks >> int(lo - t0)) & 1) {
        // The first token drops the state, and the products below give zeros, but not from rows that are not finite: they
        // have done their part.
        __syncthreads();
        uint4* at[2] = {reinterpret_cast<uint4*>(sm.q[0]), reinterpret_cast<uint4*>(sm.k[0])};
#pragma unroll 1
        for (int j = tid; j < L * C * SP / 8; j += NW * 32) at[0][j] = at[1][j] = make_uint4(0, 0, 0, 0);
        if (tid < C) sm.gates.ak[tid] = sm.gates.aq[tid] = 0.0f;
        __syncthreads();
      }
      if (more) {
        float x[4][4];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const float2 ak = *reinterpret_cast<const float2*>(&sm.gates.ak[n * 8 + qj]);
          const float2 aq = *reinterpret_cast<const float2*>(&sm.gates.aq[n * 8 + qj]);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const float fk = c & 1 ? ak.y : ak.x, fq = c & 1 ? aq.y : aq.x;
            const int at = (n * 8 + qj + (c & 1)) * DP + c0 + gi + (c >> 1) * 8;
            float y = __half2float(sm.d_out[0][at]);
            if (L == 2) y += __half2float(sm.d_out[L - 1][at]);
            x[n][c] = fq == 0.0f ? 0.0f : y * (fq * u_out);
            e[n][c] = fk == 0.0f ? 0.0f : e[n][c] * -fk;
          }
        }
        state_update<DK, L>(rt, keep, x, sm.q[0], 2, lane);
        state_update<DK, L>(rt, 1.0f, e, sm.k[0], 2, lane);
        has_r = true;
      }
      __syncthreads();
      if (tid == 0) sm.gates.bad = 0, sm.gates.state_bad = 0, sm.r_bad = 0, sm.most_out = sm.most_state = sm.most_r = sm.most_w = sm.most_e = 0;
      __syncthreads();
      if (more) raise(&sm.most_r, sm.r_bad, most_of<DK / 8>(rt));
      hi = lo;
    }
  }
  if (r_to) for_state<DK>(rt, dk, dv, c0, lane, [&](float& x, int64_t at) { r_to[at] = x; });
}

// dq (grid y 0) and dk (1) of a key head: the sum over its value heads, in their order.  A warp a row.
template <class T>
__global__ void __launch_bounds__(256)
shared_heads_kernel(const float* part_q, const float* part_k, ZenoTensor d_q, ZenoTensor d_k, uint64_t rows, uint32_t tokens,
                    uint32_t key_heads, uint32_t group, uint32_t dk) {
  const float* part = blockIdx.y ? part_k : part_q;
  const ZenoTensor& out = blockIdx.y ? d_k : d_q;
  const uint32_t lane = threadIdx.x & 31;
  for (uint64_t row = blockIdx.x * 8ull + (threadIdx.x >> 5); row < rows; row += uint64_t(gridDim.x) * 8) {  // (b, t, key head)
    const uint64_t bt = row / key_heads;
    const uint32_t kh = uint32_t(row - bt * key_heads);
    const uint64_t b = bt / tokens;
    T* at = static_cast<T*>(out.data) + int64_t(b) * out.stride[0] + int64_t(bt - b * tokens) * out.stride[1] + int64_t(kh) * out.stride[2];
    const float* in = part + row * group * dk;
#pragma unroll 4
    for (uint32_t c = lane; c < dk; c += 32) {
      float sum = 0.0f;
      for (uint32_t g = 0; g < group; ++g) sum += in[g * dk + c];
      if constexpr (sizeof(T) == 2) at[c] = __float2bfloat16_rn(sum);
      else at[c] = sum;
    }
  }
}

// Segments of a call: as many as fill the SMs with blocks, each of at least 4 chunks.
// (8 environments x 8 heads of 128 x 128, 1000 tokens, with the forward pass: 961 us in 2 segments, 1161 whole.)
inline uint32_t back_segments(const ZenoDeltaRule& p) {
  const uint64_t chunks = (uint64_t(p.tokens) + C - 1) / C, blocks = uint64_t(p.batch) * p.value_heads;
  const int warps = value_groups(p), width = key_width(p);
  const uint64_t slots = uint64_t(kSms) * ((width == 32 || (width == 64 && warps > 2) ? 12 : 8) / warps);
  uint64_t n = blocks ? slots / blocks : 1;
  if (n > chunks / 4) n = chunks / 4;
  return n < 2 ? 1 : uint32_t(n);
}

template <int DK, int NW, class T, class OUT>
cudaError_t launch(const ZenoDeltaRule& p, const ZenoDeltaRuleGrads& d, char* workspace, cudaStream_t stream) {
  const auto kernel = delta_backward_kernel<DK, NW, T, OUT>;
  constexpr int smem = int(sizeof(BackwardSmem<DK, NW, T>));
  static_assert(smem <= 227 * 1024, "shared memory of a block");
  static std::atomic<uint64_t> allowed{0};
  cudaError_t e = allow_smem(kernel, smem, allowed);
  if (e != cudaSuccess) return e;
  const uint32_t rows = p.batch * p.value_heads, segments = back_segments(p);
  BackSplit sp{};
  sp.segments = 1, sp.chunks = (p.tokens + C - 1) / C;
  if (segments > 1) {
    const DeltaSplitLayout lay(p, segments);
    float* m = reinterpret_cast<float*>(workspace);
    float* state = reinterpret_cast<float*>(workspace + lay.m + lay.n);
    int* cleared = reinterpret_cast<int*>(workspace + lay.m + 2 * lay.n);
    sp.n = reinterpret_cast<float*>(workspace + lay.m);
    sp.chunks = (sp.chunks + segments - 1) / segments;
    sp.segments = ((p.tokens + C - 1) / C + sp.chunks - 1) / sp.chunks;  // none of them empty
    if (sp.segments > 2) e = launch_delta_transitions(p, m, cleared, sp.segments, sp.chunks, stream);
    if (e != cudaSuccess) return e;
    sp.r_only = true;
    kernel<<<dim3(rows, 1, sp.segments), NW * 32, smem, stream>>>(p, d, sp);
    e = cudaGetLastError();
    if (e == cudaSuccess)
      e = launch_delta_walk(DeltaWalk{m, sp.n, state, cleared, d.d_final, sp.segments, p.key_dim, p.value_dim, true}, rows, stream);
    if (e != cudaSuccess) return e;
    sp.r_only = false, sp.state = state;
  }
  kernel<<<dim3(rows, 1, sp.segments), NW * 32, smem, stream>>>(p, d, sp);
  return cudaGetLastError();
}

template <int DK, class T, class OUT>
cudaError_t by_width(const ZenoDeltaRule& p, const ZenoDeltaRuleGrads& d, char* workspace, cudaStream_t stream) {
  switch (value_groups(p)) {
    case 2:
      if constexpr (DK < 128) return launch<DK, 2, T, OUT>(p, d, workspace, stream);
    case 4: return launch<DK, 4, T, OUT>(p, d, workspace, stream);
    default: return launch<DK, 8, T, OUT>(p, d, workspace, stream);
  }
}

template <class T, class OUT>
cudaError_t by_rows(const ZenoDeltaRule& p, const ZenoDeltaRuleGrads& d, char* workspace, cudaStream_t stream) {
  switch (key_width(p)) {
    case 32: return by_width<32, T, OUT>(p, d, workspace, stream);
    case 64: return by_width<64, T, OUT>(p, d, workspace, stream);
    default: return by_width<128, T, OUT>(p, d, workspace, stream);
  }
}

inline uint64_t split_bytes(const ZenoDeltaRule& p) {
  const uint32_t segments = back_segments(p);
  return segments > 1 ? DeltaSplitLayout(p, segments).total : 0;
}

// Rows of a gradient of their own: dq and dk of the call's type, written by the kernel itself.
template <class T>
cudaError_t own_heads(const ZenoDeltaRule& p, const ZenoDeltaRuleGrads& d, void* workspace, cudaStream_t stream) {
  return by_rows<T, T>(p, d, static_cast<char*>(workspace), stream);
}

// Shared key heads: 32-bit rows for each value head, then their sums.
template <class T>
cudaError_t shared_heads(const ZenoDeltaRule& p, const ZenoDeltaRuleGrads& d, void* workspace, cudaStream_t stream) {
  const uint64_t rows = uint64_t(p.batch) * p.tokens * p.key_heads;
  const uint32_t group = p.value_heads / p.key_heads;
  char* at = static_cast<char*>(workspace);  // the segments' part, then the rows'
  float* part_q = reinterpret_cast<float*>(at + split_bytes(p));
  float* part_k = part_q + rows * group * p.key_dim;
  ZenoDeltaRuleGrads x = d;
  const int64_t width = p.key_dim;
  for (ZenoTensor* t : {&x.d_q, &x.d_k})
    t->stride[2] = width, t->stride[1] = width * p.value_heads, t->stride[0] = width * p.value_heads * int64_t(p.tokens);
  x.d_q.data = part_q, x.d_k.data = part_k;
  cudaError_t e = by_rows<T, float>(p, x, at, stream);
  if (e != cudaSuccess || rows == 0) return e;
  const uint64_t blocks = (rows + 7) / 8;
  shared_heads_kernel<T><<<dim3(unsigned(blocks < kSms * 8 ? blocks : kSms * 8), 2), 256, 0, stream>>>(part_q, part_k, d.d_q, d.d_k, rows,
                                                                                                   p.tokens, p.key_heads, group, p.key_dim);
  return cudaGetLastError();
}

}  // namespace
}  // namespace delta
}  // namespace zb
