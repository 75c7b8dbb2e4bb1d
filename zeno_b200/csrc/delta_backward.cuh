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
#pragma once
#include "delta_mma.cuh"

namespace zb {
namespace delta {
namespace {

template <int DK, int NW, class T>
struct BackwardSmem {
  static constexpr int L = In<T>::limbs;
  static constexpr int VC = 16 * NW;
  Gates gates;
  Pairs pairs;
  Gram gram;
  __align__(16) __half q[L][C * (DK + 8)];
  __align__(16) __half k[L][C * (DK + 8)];
  __align__(16) __half d_out[L][C * (VC + 8)];
  __align__(16) T v[C * (VC + 16 / int(sizeof(T)))];
  __align__(16) __half w[2][VC * CP];         // W^T [channel][token]
  __align__(16) __half d_e[2][VC * CP];       // dE^T
  __align__(16) __half state[2][VC * (DK + 8)];  // S0^T, then R^T [channel][key channel]
  // M and X with k's factors, rows of the later token; M^T and X^T with q's and k's, rows of the earlier one
  __align__(16) __half mk[2][C * CP], xk[2][C * CP], mq[2][C * CP], xt[2][C * CP];
  float fmk[C], fxk[C], fmq[C], fxt[C], fk[C];
  float beta_part[8][C], beta_pairs[C];
  float dot_q[8][C], dot_row[8][C], dot_col[8][C];
  float end_part[8];
  unsigned most_out, most_state, most_r, most_w, most_e;  // largest finite magnitudes (float bits)
  int r_bad;
};

__device__ __forceinline__ void raise(unsigned* at, float x) {
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(kAll, x, d));
  if ((threadIdx.x & 31) == 0 && x < INFINITY) atomicMax(at, __float_as_uint(x));
}

template <int N>
__device__ __forceinline__ float most_of(const float (&t)[N][4]) {
  float m = 0.0f;
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int x = 0; x < 4; ++x) m = fmaxf(m, fabsf(t[n][x]));
  return m;
}

template <int N>
__device__ __forceinline__ bool finite(const float (&t)[N][4]) {
  bool ok = true;
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int x = 0; x < 4; ++x) ok &= fabsf(t[n][x]) < INFINITY;
  return ok;
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

// Rows of a token-by-token plane (pitch CP, two limbs) times rows of K or Q (limb planes), blocks
// [from, to) of 16, into 16 x 8 N tiles from column c0 on; the result times the row's factor.
template <int DK, int N, int L>
__device__ __forceinline__ void pairs_times_rows(float (&out)[N][4], const __half* plane, const float* factor, const __half* x,
                                                 int r, int from, int to, int c0, int lane) {
  constexpr int PITCH = DK + 8, PLANE = C * PITCH;
  float acc[N][4] = {};
  for (int j = from; j < to; ++j) {
    uint32_t ah[4], al[4];
    a_rows(ah, plane + r * 16 * CP + j * 16, CP, lane);
    a_rows(al, plane + C * CP + r * 16 * CP + j * 16, CP, lane);
#pragma unroll
    for (int n = 0; n < N; n += 2) {
      uint32_t bh[4], bl[4] = {};
      b_cols(bh, x + j * 16 * PITCH + c0 + n * 8, PITCH, lane);
      if (L == 2) b_cols(bl, x + PLANE + j * 16 * PITCH + c0 + n * 8, PITCH, lane);
      mma2<2, L>(acc[n], acc[n + 1], ah, al, bh, bl);
    }
  }
  const float f0 = factor[r * 16 + (lane >> 2)], f1 = factor[r * 16 + (lane >> 2) + 8];
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int c = 0; c < 4; ++c) out[n][c] = fmaf(acc[n][c], c < 2 ? f0 : f1, out[n][c]);
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

// OUT: type of the dq and dk rows (float: the workspace of shared heads, reduced afterwards).
template <int DK, int NW, class T, class OUT>
__global__ void __launch_bounds__(NW * 32)
delta_backward_kernel(const __grid_constant__ ZenoDeltaRule p, const __grid_constant__ ZenoDeltaRuleGrads d) {
  extern __shared__ __align__(16) unsigned char raw[];
  using Smem = BackwardSmem<DK, NW, T>;
  constexpr int L = In<T>::limbs, VC = 16 * NW, VP = VC + 16 / int(sizeof(T)), DP = VC + 8, SP = DK + 8;
  Smem& sm = *reinterpret_cast<Smem*>(raw);
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

  float rt[DK / 8][4];  // R^T
#pragma unroll
  for (int n = 0; n < DK / 8; ++n)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int c = c0 + gi + (x >> 1) * 8, r = n * 8 + qj + (x & 1);
      rt[n][x] = d.d_final && c < dv && r < dk ? d.d_final[state_at + int64_t(r) * dv + c] : 0.0f;
    }
  if (tid == 0) sm.gates.bad = 0, sm.gates.state_bad = 0, sm.r_bad = 0, sm.most_out = sm.most_state = sm.most_r = sm.most_w = sm.most_e = 0;
  __syncthreads();
  raise(&sm.most_r, most_of<DK / 8>(rt));
  if (!finite<DK / 8>(rt)) sm.r_bad = 1;

  const int64_t T_ = p.tokens;
  const int64_t chunks = (T_ + C - 1) / C;
  for (int64_t chunk = chunks - 1; chunk >= 0; --chunk) {
    const int64_t t0 = chunk * C, t1 = min(t0 + C, T_);
    for (int64_t hi = t1; hi > t0;) {
      int64_t lo = t0;
      // ---- loads
      float st[DK / 8][4];  // S0^T
      if (chunk > 0) {
        const float4* from = reinterpret_cast<const float4*>(p.saved + ((int64_t(blockIdx.x) * (chunks - 1) + chunk - 1) * VC + c0) * DK);
#pragma unroll
        for (int n = 0; n < DK / 8; ++n) {
          const float4 x = __ldcs(from + n * 32 + lane);
          st[n][0] = x.x, st[n][1] = x.y, st[n][2] = x.z, st[n][3] = x.w;
        }
      } else {
#pragma unroll
        for (int n = 0; n < DK / 8; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int c = c0 + gi + (x >> 1) * 8, r = n * 8 + qj + (x & 1);
            st[n][x] = p.initial_state && c < dv && r < dk ? p.initial_state[state_at + int64_t(r) * dv + c] : 0.0f;
          }
      }
      float go[2][8];
      const auto load_out = [&](int64_t from, int64_t to) {
        bool bad = false;
        float most = 0.0f;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int j = tid + u * NW * 32, row = j / (VC / 8), at = (j % (VC / 8)) * 8;
          const int64_t t = t0 + row;
          if (t >= from && t < to && at < dv) {
            unpack8<T>(go[u], fetch8(d_out + t * d.d_out.stride[1] + at, dv - at, vec_do));
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) go[u][i] = 0.0f;
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            bad |= !(fabsf(go[u][i]) < INFINITY);
            most = fmaxf(most, fabsf(go[u][i]));
          }
        }
        raise(&sm.most_out, most);
        if (bad) sm.gates.bad = 1;
      };
      if (warp == 0) scan_gates(sm.gates, p, rows.g, rows.beta, rows.reset, t0, lo, hi, lane);
      load_rows<DK, NW, T>(sm.gates, p, rows, sm.q[0], sm.k[0], sm.v, 0, t0, lo, hi, tid);
      load_out(lo, hi);
      if (!finite<DK / 8>(st)) sm.gates.state_bad = 1;
      raise(&sm.most_state, most_of<DK / 8>(st));
      __syncthreads();
      // A value that is not finite must not reach another episode through a product with
      // zero: such a chunk is taken episode by episode.
      if ((sm.gates.bad || sm.gates.state_bad || sm.r_bad) && (sm.gates.marks >> 1) != 0) {
        lo = t0 + 31 - __clz(int(sm.gates.marks));
        __syncthreads();
        if (tid == 0) sm.gates.bad = 0, sm.gates.state_bad = 0, sm.most_out = sm.most_state = 0;
        __syncthreads();
        if (warp == 0) scan_gates(sm.gates, p, rows.g, rows.beta, rows.reset, t0, lo, hi, lane);
        load_rows<DK, NW, T>(sm.gates, p, rows, sm.q[0], sm.k[0], sm.v, 0, t0, lo, hi, tid);
        load_out(lo, hi);
#pragma unroll
        for (int n = 0; n < DK / 8; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x) st[n][x] = 0.0f;  // the episode's first token drops the state
        __syncthreads();
      }
      const int e_out = pow2_exp(__uint_as_float(sm.most_out)), e_state = pow2_exp(__uint_as_float(sm.most_state));
      const float u_out = pow2_unscale(e_out) * p.scale, u_state = pow2_unscale(e_state);
      {
        const float sc = pow2_scale(e_out);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int j = tid + u * NW * 32, row = j / (VC / 8), at = (j % (VC / 8)) * 8;
          uint4 h4, l4;
          split(go[u][0] * sc, go[u][1] * sc, h4.x, l4.x);
          split(go[u][2] * sc, go[u][3] * sc, h4.y, l4.y);
          split(go[u][4] * sc, go[u][5] * sc, h4.z, l4.z);
          split(go[u][6] * sc, go[u][7] * sc, h4.w, l4.w);
          *reinterpret_cast<uint4*>(&sm.d_out[0][row * DP + at]) = h4;
          if (L == 2) *reinterpret_cast<uint4*>(&sm.d_out[L - 1][row * DP + at]) = l4;
        }
      }
      store_planes<DK / 8>(sm.state[0], sm.state[1], SP, st, pow2_scale(e_state), warp, lane);
      if (tid < C) sm.fk[tid] = sm.gates.token[tid].fk;
      pair_matrices<DK, NW, L, true>(sm.gates, sm.pairs, &sm.gram, sm.q[0], sm.k[0], warp, lane);
      __syncthreads();

      // ---- phase A: this warp's value channels
      float w[4][4] = {}, e[4][4] = {};
      const float keep = sm.gates.keep;
      {
        float end = 0.0f;  // of <S_C, R>
        if (keep != 0.0f) {
#pragma unroll
          for (int n = 0; n < DK / 8; ++n)
#pragma unroll
            for (int x = 0; x < 4; ++x) end = fmaf(st[n][x], rt[n][x], end);
          end *= keep;
        }
        int e0, e1, e2, e3;
        row_exps<DK / 8>(st, e0, e1);
        row_exps<DK / 8>(rt, e2, e3);
        const float s0 = pow2_scale(e0), s1 = pow2_scale(e1), s2 = pow2_scale(e2), s3 = pow2_scale(e3);
#pragma unroll
        for (int kk = 0; kk < DK; kk += 16) {
          uint32_t ah[4], al[4];
          split_a(ah, al, st[kk / 8], st[kk / 8 + 1], s0, s1);
          state_times_rows<DK, L>(w, ah, al, sm.k[0], kk, lane);
          split_a(ah, al, rt[kk / 8], rt[kk / 8 + 1], s2, s3);
          state_times_rows<DK, L>(e, ah, al, sm.k[0], kk, lane);
        }
        const float f0 = pow2_unscale(e0), f1 = pow2_unscale(e1), f2 = pow2_unscale(e2), f3 = pow2_unscale(e3);
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int i = n * 8 + qj + (x & 1);
            const float a = sm.gates.ak[i], z = sm.gates.zk[i];
            const float v = In<T>::up(sm.v[i * VP + c0 + gi + (x >> 1) * 8]);
            w[n][x] = a == 0.0f ? v : v - w[n][x] * ((x < 2 ? f0 : f1) * a);
            e[n][x] = z == 0.0f ? 0.0f : e[n][x] * ((x < 2 ? f2 : f3) * z);
          }
        solve_forward(w, sm.pairs, lane);
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x)
            end = fmaf(e[n][x], w[n][x] * sm.gates.beta[n * 8 + qj + (x & 1)], end);
#pragma unroll
        for (int m = 1; m < 32; m <<= 1) end += __shfl_xor_sync(kAll, end, m);
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
          b_rows(bh, sm.pairs.p[0] + r * 16 * CP + i * 16, CP, lane);
          b_rows(bl, sm.pairs.p[1] + r * 16 * CP + i * 16, CP, lane);
          mma2<L, 2>(acc[0], acc[1], ah, al, bh, bl);
        }
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x)
            e[2 * r + n][x] = fmaf(acc[n][x], u_out * sm.pairs.fp[r * 16 + n * 8 + qj + (x & 1)], e[2 * r + n][x]);
      }
      // dbeta: dU . w over this warp's channels; then dW = beta dU
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float s = fmaf(e[n][x], w[n][x], e[n][x + 2] * w[n][x + 2]);
          s += __shfl_xor_sync(kAll, s, 4);
          s += __shfl_xor_sync(kAll, s, 8);
          s += __shfl_xor_sync(kAll, s, 16);
          if (gi == 0) sm.beta_part[warp][n * 8 + qj + x] = s;
          const float be = sm.gates.beta[n * 8 + qj + x];
          e[n][x] *= be, e[n][x + 2] *= be;
        }
      solve_backward(e, sm.pairs, lane);  // now dE^T
      store_out(e, d_v, d.d_v.stride[1], t0, lo, hi, c0, dv, dv_pairs, lane);
      raise(&sm.most_w, most_of<4>(w));
      raise(&sm.most_e, most_of<4>(e));
      __syncthreads();
      const int e_w = pow2_exp(__uint_as_float(sm.most_w)), e_e = pow2_exp(__uint_as_float(sm.most_e));
      const float u_w = pow2_unscale(e_w), u_e = pow2_unscale(e_e);
      store_planes<4>(sm.w[0], sm.w[1], CP, w, pow2_scale(e_w), warp, lane);
      store_planes<4>(sm.d_e[0], sm.d_e[1], CP, e, pow2_scale(e_e), warp, lane);
      __syncthreads();

      // ---- token-by-token matrices of the gradients: jobs of 16 rows
      for (int job = warp; job < 8; job += NW) {
        const int kind = job >> 1, r = (job & 1) ^ (kind & 1);  // 0: M, 1: X, 2: M^T, 3: X^T; a warp gets long and short rows
        const bool later = kind < 2;                             // rows are the later token
        float acc[4][4] = {};
        const int from = later ? 0 : r, to = later ? r + 1 : 2;
#pragma unroll 1
        for (int kk = 0; kk < VC; kk += 16) {
          uint32_t ah[4], al[4] = {};
          if (kind == 0) {
            a_rows(ah, sm.d_out[0] + r * 16 * DP + kk, DP, lane);
            if (L == 2) a_rows(al, sm.d_out[L - 1] + r * 16 * DP + kk, DP, lane);
          } else {
            const __half* a = kind == 1 ? sm.d_e[0] : sm.w[0];
            a_cols(ah, a + kk * CP + r * 16, CP, lane);
            a_cols(al, a + VC * CP + kk * CP + r * 16, CP, lane);
          }
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            if (c < from || c >= to) continue;
            uint32_t bh[4], bl[4] = {};
            if (kind == 2) {
              b_rows(bh, sm.d_out[0] + c * 16 * DP + kk, DP, lane);
              if (L == 2) b_rows(bl, sm.d_out[L - 1] + c * 16 * DP + kk, DP, lane);
            } else {
              const __half* y = kind == 3 ? sm.d_e[0] : sm.w[0];
              b_cols(bh, y + kk * CP + c * 16, CP, lane);
              b_cols(bl, y + VC * CP + kk * CP + c * 16, CP, lane);
            }
            if (kind == 0 && L == 1) mma2<1, 2>(acc[2 * c], acc[2 * c + 1], ah, al, bh, bl);
            else if (kind == 2 && L == 1) mma2<2, 1>(acc[2 * c], acc[2 * c + 1], ah, al, bh, bl);
            else mma2<2, 2>(acc[2 * c], acc[2 * c + 1], ah, al, bh, bl);
          }
        }
        const float unit = (kind & 1) ? -u_e * u_w : u_out * u_w;
        __half* plane = kind == 0 ? sm.mk[0] : kind == 1 ? sm.xk[0] : kind == 2 ? sm.mq[0] : sm.xt[0];
        float* factor = kind == 0 ? sm.fmk : kind == 1 ? sm.fxk : kind == 2 ? sm.fmq : sm.fxt;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int row = r * 16 + gi + half * 8;
          float x[8], most = 0.0f, db = 0.0f;
#pragma unroll
          for (int n = 0; n < 8; ++n) {
            const int col = (n >> 1) * 8 + qj + (n & 1);
            const int i = later ? row : col, j = later ? col : row;
            const bool on = kind & 1 ? j < i : j <= i;
            float y = on ? acc[n >> 1][half * 2 + (n & 1)] * unit : 0.0f;
            if (kind == 3 && on) db = fmaf(y, sm.gram.at[i][j], db);
            if (on) y *= sm.gates.beta[j] * decay(sm.gates.token[i], sm.gates.token[j]) * (kind == 2 ? sm.gates.fq[i] : later ? sm.gates.token[j].fk : sm.gates.token[i].fk);
            x[n] = y;
            most = fmaxf(most, fabsf(y));
          }
          most = quad_max(most);
          const int ex = pow2_exp(most);
          const float sc = pow2_scale(ex);
#pragma unroll
          for (int n = 0; n < 4; ++n)
            store_split(plane, plane + C * CP, row * CP + n * 8 + qj, x[2 * n] * sc, x[2 * n + 1] * sc);
          if ((lane & 3) == 0) factor[row] = pow2_unscale(ex);
          if (kind == 3) {
            db += __shfl_xor_sync(kAll, db, 1);
            db += __shfl_xor_sync(kAll, db, 2);
            if ((lane & 3) == 0) sm.beta_pairs[row] = db;
          }
        }
      }
      __syncthreads();

      // ---- phase B: 16 tokens and a share of the key channels
      constexpr int DKW = 2 * DK / NW < 16 ? 16 : 2 * DK / NW, N = DKW / 8, GROUPS = DK / DKW;
      const int r = warp & 1, group = warp >> 1, k0 = group * DKW;
      const bool works = group < GROUPS;
      float gq[N][4] = {}, g_row[N][4] = {}, g_col[N][4] = {};
      if (works) {
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
        pairs_times_rows<DK, N, L>(gq, sm.mk[0], sm.fmk, sm.k[0], r, 0, r + 1, k0, lane);
        pairs_times_rows<DK, N, L>(g_row, sm.xk[0], sm.fxk, sm.k[0], r, 0, r + 1, k0, lane);
        pairs_times_rows<DK, N, L>(g_col, sm.mq[0], sm.fmq, sm.q[0], r, r, 2, k0, lane);
        pairs_times_rows<DK, N, L>(g_col, sm.xt[0], sm.fxt, sm.k[0], r, r, 2, k0, lane);
      }
      __syncthreads();
      const int e_r = pow2_exp(__uint_as_float(sm.most_r));
      store_planes<DK / 8>(sm.state[0], sm.state[1], SP, rt, pow2_scale(e_r), warp, lane);
      __syncthreads();
      if (works) {
        float acc[N][4] = {};
        rows_times_state<DK, NW, N, 2, true>(acc, sm.w[0], CP, VC * CP, sm.state[0], r, k0, lane);
        const float u = u_w * pow2_unscale(e_r);
        const int i0 = r * 16 + gi;
        const float z0 = sm.gates.to_end[i0] * sm.gates.beta[i0] * u, z1 = sm.gates.to_end[i0 + 8] * sm.gates.beta[i0 + 8] * u;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const float z = x < 2 ? z0 : z1;
            if (z != 0.0f) g_col[n][x] = fmaf(acc[n][x], z, g_col[n][x]);
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
        float dg = 0.0f, db = sm.beta_pairs[lane];
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
      // ---- R^T <- a_C R^T + (a dO)^T Q - (a dE)^T K
      {
        float x[4][4];
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int i = n * 8 + qj + (c & 1);
            const float ak = sm.gates.ak[i], aq = sm.gates.aq[i];
            const int at = i * DP + c0 + gi + (c >> 1) * 8;
            float y = __half2float(sm.d_out[0][at]);
            if (L == 2) y += __half2float(sm.d_out[L - 1][at]);
            x[n][c] = aq == 0.0f ? 0.0f : y * (aq * u_out);
            e[n][c] = ak == 0.0f ? 0.0f : e[n][c] * -ak;
          }
        state_update<DK, L>(rt, keep, x, sm.q[0], lane);
        state_update<DK, L>(rt, 1.0f, e, sm.k[0], lane);
      }
      __syncthreads();
      if (tid == 0) sm.gates.bad = 0, sm.gates.state_bad = 0, sm.r_bad = 0, sm.most_out = sm.most_state = sm.most_r = sm.most_w = sm.most_e = 0;
      __syncthreads();
      raise(&sm.most_r, most_of<DK / 8>(rt));
      if (!finite<DK / 8>(rt)) sm.r_bad = 1;
      hi = lo;
    }
  }
  if (d.d_initial) {
#pragma unroll
    for (int n = 0; n < DK / 8; ++n)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int c = c0 + gi + (x >> 1) * 8, r = n * 8 + qj + (x & 1);
        if (c < dv && r < dk) d.d_initial[state_at + int64_t(r) * dv + c] = rt[n][x];
      }
  }
}

// dq and dk of a key head: the sum over its value heads, in their order.
template <class T>
__global__ void __launch_bounds__(256)
shared_heads_kernel(const float* part, ZenoTensor out, uint64_t rows, uint32_t tokens, uint32_t key_heads, uint32_t group, uint32_t dk) {
  const uint64_t n = rows * dk;
  for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < n; i += uint64_t(gridDim.x) * 256) {
    const uint64_t row = i / dk;  // (b, t, key head)
    const uint32_t c = uint32_t(i % dk), kh = uint32_t(row % key_heads);
    const uint64_t bt = row / key_heads;
    float sum = 0.0f;
    for (uint32_t g = 0; g < group; ++g) sum += part[((bt * key_heads + kh) * group + g) * dk + c];
    T* at = static_cast<T*>(out.data) + int64_t(bt / tokens) * out.stride[0] + int64_t(bt % tokens) * out.stride[1] +
            int64_t(kh) * out.stride[2] + c;
    if constexpr (sizeof(T) == 2) *at = __float2bfloat16_rn(sum);
    else *at = sum;
  }
}

template <int DK, int NW, class T, class OUT>
cudaError_t launch(const ZenoDeltaRule& p, const ZenoDeltaRuleGrads& d, cudaStream_t stream) {
  const auto kernel = delta_backward_kernel<DK, NW, T, OUT>;
  constexpr int smem = int(sizeof(BackwardSmem<DK, NW, T>));
  static_assert(smem <= 227 * 1024, "shared memory of a block");
  static std::atomic<uint64_t> allowed{0};
  const cudaError_t e = allow_smem(kernel, smem, allowed);
  if (e != cudaSuccess) return e;
  kernel<<<p.batch * p.value_heads, NW * 32, smem, stream>>>(p, d);
  return cudaGetLastError();
}

template <int DK, class T, class OUT>
cudaError_t by_width(const ZenoDeltaRule& p, const ZenoDeltaRuleGrads& d, cudaStream_t stream) {
  switch (value_warps(p)) {
    case 2:
      if constexpr (DK < 128) return launch<DK, 2, T, OUT>(p, d, stream);
    case 4: return launch<DK, 4, T, OUT>(p, d, stream);
    default: return launch<DK, 8, T, OUT>(p, d, stream);
  }
}

template <class T, class OUT>
cudaError_t by_rows(const ZenoDeltaRule& p, const ZenoDeltaRuleGrads& d, cudaStream_t stream) {
  switch (key_width(p)) {
    case 32: return by_width<32, T, OUT>(p, d, stream);
    case 64: return by_width<64, T, OUT>(p, d, stream);
    default: return by_width<128, T, OUT>(p, d, stream);
  }
}

template <class T>
cudaError_t by_heads(const ZenoDeltaRule& p, const ZenoDeltaRuleGrads& d, void* workspace, cudaStream_t stream) {
  if (p.key_heads == p.value_heads) return by_rows<T, T>(p, d, stream);
  const uint64_t rows = uint64_t(p.batch) * p.tokens * p.key_heads;
  const uint32_t group = p.value_heads / p.key_heads;
  float* part_q = static_cast<float*>(workspace);
  float* part_k = part_q + rows * group * p.key_dim;
  ZenoDeltaRuleGrads x = d;
  const int64_t width = p.key_dim;
  for (ZenoTensor* t : {&x.d_q, &x.d_k})
    t->stride[2] = width, t->stride[1] = width * p.value_heads, t->stride[0] = width * p.value_heads * int64_t(p.tokens);
  x.d_q.data = part_q, x.d_k.data = part_k;
  cudaError_t e = by_rows<T, float>(p, x, stream);
  if (e != cudaSuccess || rows == 0) return e;
  const uint64_t blocks = (rows * p.key_dim + 255) / 256;
  const unsigned grid = unsigned(blocks < 148 * 8 ? blocks : 148 * 8);
  shared_heads_kernel<T><<<grid, 256, 0, stream>>>(part_q, d.d_q, rows, p.tokens, p.key_heads, group, p.key_dim);
  shared_heads_kernel<T><<<grid, 256, 0, stream>>>(part_k, d.d_k, rows, p.tokens, p.key_heads, group, p.key_dim);
  return cudaGetLastError();
}

}  // namespace
}  // namespace delta
}  // namespace zb
