// Rollouts of up to 32 tokens of many environments, bfloat16: one warp takes one (environment, value head).
//
// The formulas are those of the chunked kernels (linear_forward.cuh, linear_backward.cuh) for a single chunk.  With a warp to itself a
// head needs no barrier, and P and dP never leave the registers: the accumulators of a product are the left operand of the next one.  What
// four warps spent on addresses, gates and waiting for one another was half of their instructions (4096 x 32 tokens, 4 heads of 64 x 64: 5000
// instructions a head forward, 6000 backward; now 2860 and 2840).  A state is not kept: it passes through the registers 16 channels at a
// time, transposed, as the right operand of S^T q and the sum of the update at once.
//
// That rollout takes 116 us forward (167 with a state in front, where its bytes alone are 123) and 128 us backward.  Both are bound
// by the latency of instructions: registers and shared memory leave place for 12 and 11 warps an SM, 1.4 instructions a cycle.
//
// Values that are not finite are looked for in P, dP and V before anything is written; a head that has some is taken element by element.
#pragma once
#include "linear_backward.cuh"

namespace zb {
namespace linear {

template <int D_>
struct WarpShape {
  using T = bf16;
  static constexpr int D = D_, C = 32, THREADS = 32, L = 1, PL = 2;
  static constexpr int P = D + 8, PLANE = C * P, KT = D / 16;
};

struct WarpGates {
  Gates<32> gates;
  float pass[32], x[32];  // what passes a token; x_i
};

// (out of line: it would hold registers that the rows' loads are waiting in)
static __device__ __noinline__ void scan_gates_of(Gates<32>& s, GateIn<32> in, bool fixed, int n, int lane) { scan_gates<32>(s, in, fixed, n, lane); }

struct WarpAt {
  uint32_t row, b, h, kh;
};
__device__ __forceinline__ WarpAt warp_at(const ZenoLinearAttention& p) {
  WarpAt a;
  a.row = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  a.b = a.row / p.value_heads, a.h = a.row % p.value_heads;
  a.kh = p.value_heads == p.key_heads ? a.h : a.h / (p.value_heads / p.key_heads);
  return a;
}

// The limbs of a 16 x 16 accumulator as a left operand.
__device__ __forceinline__ void as_left(uint32_t (&to)[2][4], const float (&acc)[2][4]) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      uint32_t w[2];
      split<2>(acc[h][2 * r], acc[h][2 * r + 1], w);
      to[0][h * 2 + r] = w[0], to[1][h * 2 + r] = w[1];
    }
}
__device__ __forceinline__ void transposed(uint32_t (&to)[2][4], const uint32_t (&from)[2][4]) {
#pragma unroll
  for (int l = 0; l < 2; ++l) {
    to[l][0] = delta::movm(from[l][0]), to[l][1] = delta::movm(from[l][2]);
    to[l][2] = delta::movm(from[l][1]), to[l][3] = delta::movm(from[l][3]);
  }
}

// x's weighted columns [col, col + 16) as a left operand of 3 limbs: A[m][token] = x[token][col + m] weight[token] factor.
template <class S>
__device__ __forceinline__ void weighted_left(uint32_t (&a)[2][3][4], const plane_t* x, int col, const float* weight, float factor, int nt, int lane) {
#pragma unroll
  for (int kk = 0; kk < 2; ++kk) {
    if (kk >= nt) break;
    uint32_t raw[4];
    frag_a<true>(raw, x + kk * 16 * S::P + col, S::P, lane);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float2 w = *reinterpret_cast<const float2*>(weight + kk * 16 + (r >> 1) * 8 + (lane & 3) * 2);
      uint32_t limbs[3];
      split<3>(lower(raw[r]) * (w.x * factor), upper(raw[r]) * (w.y * factor), limbs);
      a[kk][0][r] = limbs[0], a[kk][1][r] = limbs[1], a[kk][2][r] = limbs[2];
    }
  }
}
// sum over the tokens of the left operand with y's columns [col, col + 16).
template <class S>
__device__ __forceinline__ void weighted_product(float (&acc)[2][4], const uint32_t (&a)[2][3][4], const plane_t* y, int col, int nt, int lane) {
  float low[2][4];
  uint32_t b[1][4];
  frag_b<true>(b[0], y + col, S::P, lane);
  mma_terms<3, 1, true>(acc, low, a[0], b);
  if (nt > 1) {
    frag_b<true>(b[0], y + 16 * S::P + col, S::P, lane);
    mma_terms<3, 1>(acc, low, a[1], b);
  }
#pragma unroll
  for (int x = 0; x < 8; ++x) acc[x >> 2][x & 3] += low[x >> 2][x & 3];
}

// Two row tiles of accumulators, rounded, into columns [col, col + 16) of rows in shared memory.
template <class S>
__device__ __forceinline__ void stage_columns(plane_t* to, const float (&acc)[2][2][4], int col, int nt, int lane) {
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    if (r >= nt) break;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int s = 0; s < 2; ++s)
        *reinterpret_cast<uint32_t*>(to + (r * 16 + (lane >> 2) + s * 8) * S::P + col + h * 8 + (lane & 3) * 2) =
            pack_round(acc[r][h][2 * s], acc[r][h][2 * s + 1]);
  }
}

// acc = sum_d x_i[d] y_lane[d], this lane's token against token i.
template <class S>
__device__ __forceinline__ float dot_rows(const plane_t* x, const plane_t* y, int width) {
  float sum = 0.0f;
  for (int d = 0; d < width; ++d) sum = fmaf(value<1>(x + d, 0), value<1>(y + d, 0), sum);
  return sum;
}

// ---------------------------------------------------------------- forward
template <class S>
__device__ __noinline__ void warp_forward_slow(const ZenoLinearAttention& p, const Gates<32>& s, const plane_t* q, const plane_t* k, const plane_t* v,
                                               bf16* out, const float* initial, float* final, int n, int lane) {
  const int dk = int(p.key_dim), dv = int(p.value_dim);
  for (int i = 0; i < n; ++i) {
    const bool meet = lane < n && meets(s.token[i], s.token[lane], i, lane);
    const float f = pair_decay(s.token[i], s.token[lane], meet) * p.scale;
    const float pair = meet ? dot_rows<S>(q + i * S::P, k + lane * S::P, dk) * f : 0.0f;
    const unsigned met = __ballot_sync(kAll, meet);
    for (int c0 = 0; c0 < dv; c0 += 32) {
      const int c = c0 + lane;
      float y = 0.0f;
      if (initial && c < dv && s.carried[i] != 0.0f) {
        for (int d = 0; d < dk; ++d) y = fmaf(value<1>(q + i * S::P + d, 0), initial[d * dv + c], y);
        y *= s.carried[i] * p.scale;
      }
      for (int j = 0; j <= i; ++j) {
        const float x = __shfl_sync(kAll, pair, j);
        if ((met >> j & 1) && c < dv) y = fmaf(x, value<1>(v + j * S::P + c, 0), y);
      }
      if (c < dv) out[int64_t(i) * p.out.stride[1] + c] = __float2bfloat16_rn(y);
    }
  }
  if (!final) return;
  for (int c = lane; c < dv; c += 32)
    for (int d = 0; d < dk; ++d) {
      float y = 0.0f;
      for (int j = 0; j < n; ++j)
        if (s.to_end[j] != 0.0f) y = fmaf(s.to_end[j] * value<1>(k + j * S::P + d, 0), value<1>(v + j * S::P + c, 0), y);
      if (initial && s.keep != 0.0f) y = fmaf(s.keep, initial[d * dv + c], y);
      final[d * dv + c] = y;
    }
}

// FULL: keys and values of D channels, so that offsets are known and nothing is past an end.
template <int D, bool FULL, int WARPS, int BLOCKS>
__global__ void __launch_bounds__(WARPS * 32, BLOCKS) linear_warp_forward_kernel(const __grid_constant__ ZenoLinearAttention p, const uint32_t vec) {
  using S = WarpShape<D>;
  constexpr int KT = S::KT;
  extern __shared__ __align__(16) char smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const WarpAt a = warp_at(p);
  if (a.row >= p.batch * p.value_heads) return;
  char* mine = smem + warp * (int(sizeof(Gates<32>)) + 3 * 2 * S::PLANE);
  Gates<32>& s = *reinterpret_cast<Gates<32>*>(mine);
  plane_t *q = reinterpret_cast<plane_t*>(mine + sizeof(Gates<32>)), *k = q + S::PLANE, *v = k + S::PLANE;
  const int dk = FULL ? D : int(p.key_dim), dv = FULL ? D : int(p.value_dim), n = int(p.tokens), nt = (n + 15) / 16;
  const Mover<S> mv(lane);
  const uint8_t* gr = p.reset.data ? static_cast<const uint8_t*>(p.reset.data) + int64_t(a.b) * p.reset.stride[0] : nullptr;
  load_rows<S>(q, place<bf16>(p.q, a.b, a.kh), p.q.stride[1], dk, vec & kVecQ, n, nt, mv);
  load_rows<S>(k, place<bf16>(p.k, a.b, a.kh), p.k.stride[1], dk, vec & kVecK, n, nt, mv);
  load_rows<S>(v, place<bf16>(p.v, a.b, a.h), p.v.stride[1], dv, vec & kVecV, n, nt, mv);
  const GateIn<32> gates = fetch_gates<32>(place<float>(p.g, a.b, a.h), p.g.stride[1], gr, p.reset.stride[1], 0, n, lane);
  scan_gates_of(s, gates, p.g.stride[1] == 0, n, lane);
  const int64_t state_size = int64_t(dk) * dv;
  const float* initial = p.initial_state ? p.initial_state + int64_t(a.row) * state_size : nullptr;
  if (initial)  // (to L2; it is read 16 channels at a time)
    for (int x = lane * 32; x < state_size; x += 1024) delta::prefetch(initial + x);
  float* final = p.final_state ? p.final_state + int64_t(a.row) * state_size : nullptr;
  bf16* out = place<bf16>(p.out, a.b, a.h);
  copies_landed();
  __syncwarp();

  const int g = lane >> 2, c2 = (lane & 3) * 2;
  uint32_t pf[3][2][4];  // P of the tiles (0, 0), (1, 0), (1, 1)
  float odd = 0.0f;      // not a number where something is not finite
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    if (r >= nt) break;
    float sc[2][2][4] = {};
#pragma unroll
    for (int kk = 0; kk < KT; ++kk) {
      if (kk * 16 >= dk) break;
      uint32_t fa[4], fb[4];
      frag_a<false>(fa, q + r * 16 * S::P + kk * 16, S::P, lane);
#pragma unroll
      for (int c = 0; c <= r; ++c) {
        frag_b<false>(fb, k + c * 16 * S::P + kk * 16, S::P, lane);
        mma(sc[c][0], fa, fb[0], fb[1]);
        mma(sc[c][1], fa, fb[2], fb[3]);
      }
    }
    const int i0 = r * 16 + g;
    const Token ti[2] = {s.token[i0], s.token[i0 + 8]};
#pragma unroll
    for (int c = 0; c <= r; ++c) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int j = c * 16 + h * 8 + c2 + e;
          const Token tj = s.token[j];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const bool meet = meets(ti[u], tj, i0 + u * 8, j);
            float& x = sc[c][h][2 * u + e];
            x = meet ? x * (pair_decay(ti[u], tj, meet) * p.scale) : 0.0f;
            odd = fmaf(x, 0.0f, odd);
          }
        }
      as_left(pf[r + c], sc[c]);
    }
  }
  if (__any_sync(kAll, odd != odd || rows_odd<S>(v, dv, nt, mv))) {
    warp_forward_slow<S>(p, s, q, k, v, out, initial, final, n, lane);
    return;
  }

  const float keep = s.keep;
#pragma unroll 1
  for (int vt = 0; vt * 16 < dv; ++vt) {
    float o[2][2][4] = {};
    // S^T: [k tile][k half][2 (channel half) + (k & 1)]: k = 16 kk + 8 h + c2 + e, channel 16 vt + 8 t + g
    float s0[KT][2][4];
    const int left = dv - vt * 16 - g;  // channels from this lane's first on
    if (initial) {
#pragma unroll
      for (int kk = 0; kk < KT; ++kk) {
        if (kk * 16 >= dk) break;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int row = kk * 16 + h * 8 + c2 + e;
            const float* from = initial + row * dv + vt * 16 + g;
            s0[kk][h][e] = FULL || (row < dk && left > 0) ? from[0] : 0.0f;
            s0[kk][h][2 + e] = FULL || (row < dk && left > 8) ? from[8] : 0.0f;
          }
      }
#pragma unroll
      for (int kk = 0; kk < KT; ++kk) {
        if (kk * 16 >= dk) break;
        uint32_t b[2][2][2];  // [channel half][k half][limb]
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int h = 0; h < 2; ++h) split<2>(s0[kk][h][2 * t], s0[kk][h][2 * t + 1], b[t][h]);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          if (r >= nt) break;
          uint32_t fa[4];
          frag_a<false>(fa, q + r * 16 * S::P + kk * 16, S::P, lane);
#pragma unroll
          for (int l = 1; l >= 0; --l)
#pragma unroll
            for (int t = 0; t < 2; ++t) mma(o[r][t], fa, b[t][0][l], b[t][1][l]);
        }
      }
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float f = s.carried[r * 16 + g + u * 8];
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float& y = o[r][t][2 * u + e];
              y = f == 0.0f ? 0.0f : y * (f * p.scale);
            }
        }
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      if (c >= nt) break;
      uint32_t fv[4];
      frag_b<true>(fv, v + c * 16 * S::P + vt * 16, S::P, lane);
#pragma unroll
      for (int r = c; r < 2; ++r) {
        if (r >= nt) break;
#pragma unroll
        for (int l = 1; l >= 0; --l)
#pragma unroll
          for (int t = 0; t < 2; ++t) mma(o[r][t], pf[r + c][l], fv[2 * t], fv[2 * t + 1]);
      }
    }
    if (final) {
      uint32_t w[2][3][4];
      weighted_left<S>(w, v, vt * 16, s.to_end, 1.0f, nt, lane);
#pragma unroll
      for (int kk = 0; kk < KT; ++kk) {
        if (kk * 16 >= dk) break;
        float add[2][4];
        weighted_product<S>(add, w, k, kk * 16, nt, lane);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int row = kk * 16 + h * 8 + c2 + e;
            float* to = final + row * dv + vt * 16 + g;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              float y = add[h][2 * t + e];
              if (initial && keep != 0.0f) y = fmaf(keep, s0[kk][h][2 * t + e], y);
              if (FULL || (row < dk && left > 8 * t)) to[8 * t] = y;
            }
          }
      }
    }
    __syncwarp();  // these columns of V have been read
    stage_columns<S>(v, o, vt * 16, nt, lane);
  }
  __syncwarp();
  store_rows<S>(out, p.out.stride[1], v, dv, vec & kVecOut, n, mv);
}

// ---------------------------------------------------------------- backward
// Where a head's results go: rows of bfloat16, or of 32 bits where value heads share a key head.
struct WarpResults {
  bf16 *q, *k, *v;
  float *shared_q, *shared_k;
  int64_t shared_stride;
};

// dg of each token from what passes it and from the state in front; returns that of the lane's.
__device__ __forceinline__ float warp_decays(const ZenoLinearAttentionGrads& d, const WarpAt& a, float pass, float x, int n, int lane) {
#pragma unroll
  for (int y = 1; y < 32; y <<= 1) {
    const float z = __shfl_down_sync(kAll, x, y);
    if (lane + y < 32) x += z;
  }
  if (lane >= n) return 0.0f;
  place<float>(d.d_g, a.b, a.h)[lane * d.d_g.stride[1]] = pass + x;
  return pass + x;
}
// Their sum over the head, from the lanes' parts.
__device__ __forceinline__ void sum_decays(const BackwardOut& extra, const WarpAt& a, uint32_t batch, double part, int lane) {
  if (!extra.decay) return;
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) part += __shfl_xor_sync(kAll, part, x);
  if (lane == 0) extra.decay[uint64_t(a.h) * batch + a.b] = part;
}

template <class S>
__device__ __noinline__ double warp_backward_slow(const ZenoLinearAttention& p, const ZenoLinearAttentionGrads& d, const WarpAt& a, const WarpResults& to,
                                                  const Gates<32>& s, const plane_t* q, const plane_t* k, const plane_t* v, const plane_t* o,
                                                  const float* initial, int n, int lane) {
  const int dk = int(p.key_dim), dv = int(p.value_dim);
  float passes = 0.0f, mine_x = 0.0f;
  double decays = 0.0;
  for (int i = 0; i < n; ++i) {  // dQ, and the decays
    const bool meet = lane < n && meets(s.token[i], s.token[lane], i, lane);
    const float f = pair_decay(s.token[i], s.token[lane], meet) * p.scale;
    const float raw = meet ? dot_rows<S>(o + i * S::P, v + lane * S::P, dv) : 0.0f;
    const float dp = meet ? raw * f : 0.0f;
    const float pass = meet ? dot_rows<S>(q + i * S::P, k + lane * S::P, dk) * f * raw : 0.0f;
    if (lane < i) decays += double(pass) * (i - lane);
    float front = pass;
    for (int y = 1; y < 32; y <<= 1) {
      const float z = __shfl_up_sync(kAll, front, y);
      if (lane >= y) front += z;
    }
    front = __shfl_up_sync(kAll, front, 1);
    if (lane > 0 && lane <= i) passes += front;
    const unsigned met = __ballot_sync(kAll, meet);
    float x = 0.0f;
    for (int c0 = 0; c0 < dk; c0 += 32) {
      const int c = c0 + lane;
      float y = 0.0f;
      if (initial && c < dk && s.carried[i] != 0.0f) {
        for (int e = 0; e < dv; ++e) y = fmaf(value<1>(o + i * S::P + e, 0), initial[c * dv + e], y);
        y *= s.carried[i] * p.scale;
        x = fmaf(y, value<1>(q + i * S::P + c, 0), x);
      }
      for (int j = 0; j <= i; ++j) {
        const float z = __shfl_sync(kAll, dp, j);
        if ((met >> j & 1) && c < dk) y = fmaf(z, value<1>(k + j * S::P + c, 0), y);
      }
      if (c < dk) {
        if (to.shared_q) to.shared_q[i * to.shared_stride + c] = y;
        else to.q[int64_t(i) * d.d_q.stride[1] + c] = __float2bfloat16_rn(y);
      }
    }
    for (int y = 1; y < 32; y <<= 1) x += __shfl_xor_sync(kAll, x, y);
    if (lane == i) mine_x = x;
    if (lane == 0) decays += double(x) * (i + 1);
  }
  for (int j = 0; j < n; ++j) {  // dK and dV
    const bool meet = lane < n && meets(s.token[lane], s.token[j], lane, j);
    const float f = pair_decay(s.token[lane], s.token[j], meet) * p.scale;
    const float dp = meet ? dot_rows<S>(o + lane * S::P, v + j * S::P, dv) * f : 0.0f;
    const float pr = meet ? dot_rows<S>(q + lane * S::P, k + j * S::P, dk) * f : 0.0f;
    const unsigned met = __ballot_sync(kAll, meet);
    for (int c0 = 0; c0 < max(dk, dv); c0 += 32) {
      const int c = c0 + lane;
      float y = 0.0f, z = 0.0f;
      for (int i = j; i < n; ++i) {
        const float x0 = __shfl_sync(kAll, dp, i), x1 = __shfl_sync(kAll, pr, i);
        if (!(met >> i & 1)) continue;
        if (c < dk) y = fmaf(x0, value<1>(q + i * S::P + c, 0), y);
        if (c < dv) z = fmaf(x1, value<1>(o + i * S::P + c, 0), z);
      }
      if (c < dk) {
        if (to.shared_k) to.shared_k[j * to.shared_stride + c] = y;
        else to.k[int64_t(j) * d.d_k.stride[1] + c] = __float2bfloat16_rn(y);
      }
      if (c < dv) to.v[int64_t(j) * d.d_v.stride[1] + c] = __float2bfloat16_rn(z);
    }
  }
  if (d.d_initial) {
    float* state = d.d_initial + int64_t(a.row) * dk * dv;
    for (int c = lane; c < dv; c += 32)
      for (int e = 0; e < dk; ++e) {
        float y = 0.0f;
        for (int i = 0; i < n; ++i)
          if (s.carried[i] != 0.0f) y = fmaf(s.carried[i] * p.scale * value<1>(q + i * S::P + e, 0), value<1>(o + i * S::P + c, 0), y);
        state[e * dv + c] = y;
      }
  }
  return d.d_g.data ? double(warp_decays(d, a, passes, mine_x, n, lane)) : decays;
}

// Without a gradient of the final state.
template <int D, bool FULL, int WARPS, int BLOCKS>
__global__ void __launch_bounds__(WARPS * 32, BLOCKS)
linear_warp_backward_kernel(const __grid_constant__ ZenoLinearAttention p, const __grid_constant__ ZenoLinearAttentionGrads d, const uint32_t vec,
                            const BackwardOut extra) {
  using S = WarpShape<D>;
  constexpr int KT = S::KT;
  extern __shared__ __align__(16) char smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  early::let_next_start();
  const WarpAt a = warp_at(p);
  if (a.row >= p.batch * p.value_heads) return;
  char* mine = smem + warp * (int(sizeof(WarpGates)) + 4 * 2 * S::PLANE);
  WarpGates& all = *reinterpret_cast<WarpGates*>(mine);
  Gates<32>& s = all.gates;
  plane_t *q = reinterpret_cast<plane_t*>(mine + sizeof(WarpGates)), *k = q + S::PLANE, *v = k + S::PLANE, *o = v + S::PLANE;
  const int dk = FULL ? D : int(p.key_dim), dv = FULL ? D : int(p.value_dim), n = int(p.tokens), nt = (n + 15) / 16;
  const Mover<S> mv(lane);
  const uint8_t* gr = p.reset.data ? static_cast<const uint8_t*>(p.reset.data) + int64_t(a.b) * p.reset.stride[0] : nullptr;
  load_rows<S>(q, place<bf16>(p.q, a.b, a.kh), p.q.stride[1], dk, vec & kVecQ, n, nt, mv);
  load_rows<S>(k, place<bf16>(p.k, a.b, a.kh), p.k.stride[1], dk, vec & kVecK, n, nt, mv);
  load_rows<S>(v, place<bf16>(p.v, a.b, a.h), p.v.stride[1], dv, vec & kVecV, n, nt, mv);
  load_rows<S>(o, place<bf16>(d.d_out, a.b, a.h), d.d_out.stride[1], dv, vec & kVecOut, n, nt, mv);
  const GateIn<32> gates = fetch_gates<32>(place<float>(p.g, a.b, a.h), p.g.stride[1], gr, p.reset.stride[1], 0, n, lane);
  scan_gates_of(s, gates, p.g.stride[1] == 0, n, lane);
  const int64_t state_size = int64_t(dk) * dv;
  const float* initial = p.initial_state ? p.initial_state + int64_t(a.row) * state_size : nullptr;
  if (initial)  // (to L2; it is read 16 channels at a time)
    for (int x = lane * 32; x < state_size; x += 1024) delta::prefetch(initial + x);
  WarpResults to{place<bf16>(d.d_q, a.b, a.kh), place<bf16>(d.d_k, a.b, a.kh), place<bf16>(d.d_v, a.b, a.h), nullptr, nullptr, 0};
  if (extra.shared_q) {
    to.shared_stride = int64_t(p.value_heads) * dk;
    const int64_t at = int64_t(a.b) * p.tokens * to.shared_stride + int64_t(a.h) * dk;
    to.shared_q = extra.shared_q + at, to.shared_k = extra.shared_k + at;
  }
  const bool each = d.d_g.data != nullptr;
  copies_landed();
  __syncwarp();

  const int g = lane >> 2, c2 = (lane & 3) * 2;
  uint32_t pf[3][2][4], df[3][2][4];  // P and D of the tiles (0, 0), (1, 0), (1, 1)
  float odd = 0.0f, decays = 0.0f;
  float passes[2][2][2] = {};  // [tile][half][e] of the columns: what passes their tokens, over the lane's rows
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    if (r >= nt) break;
    float sp[2][2][4] = {}, so[2][2][4] = {};
#pragma unroll
    for (int kk = 0; kk < KT; ++kk) {
      if (kk * 16 >= dk) break;
      uint32_t fa[4], fb[4];
      frag_a<false>(fa, q + r * 16 * S::P + kk * 16, S::P, lane);
#pragma unroll
      for (int c = 0; c <= r; ++c) {
        frag_b<false>(fb, k + c * 16 * S::P + kk * 16, S::P, lane);
        mma(sp[c][0], fa, fb[0], fb[1]);
        mma(sp[c][1], fa, fb[2], fb[3]);
      }
    }
#pragma unroll
    for (int kk = 0; kk < KT; ++kk) {
      if (kk * 16 >= dv) break;
      uint32_t fa[4], fb[4];
      frag_a<false>(fa, o + r * 16 * S::P + kk * 16, S::P, lane);
#pragma unroll
      for (int c = 0; c <= r; ++c) {
        frag_b<false>(fb, v + c * 16 * S::P + kk * 16, S::P, lane);
        mma(so[c][0], fa, fb[0], fb[1]);
        mma(so[c][1], fa, fb[2], fb[3]);
      }
    }
    const int i0 = r * 16 + g;
    const Token ti[2] = {s.token[i0], s.token[i0 + 8]};
    float before[2] = {0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c <= r; ++c) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float pass[2][2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int j = c * 16 + h * 8 + c2 + e;
          const Token tj = s.token[j];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const bool meet = meets(ti[u], tj, i0 + u * 8, j);
            const float f = pair_decay(ti[u], tj, meet) * p.scale;
            float &x = sp[c][h][2 * u + e], &y = so[c][h][2 * u + e];
            x = meet ? x * f : 0.0f;
            pass[u][e] = meet ? x * y : 0.0f;
            y = meet ? y * f : 0.0f;
            odd = fmaf(pass[u][e], 0.0f, odd);  // (x and y are finite if their product is)
          }
        }
        if (!each) {  // a pair passes i - j tokens
          const float far = float(i0 - c * 16 - h * 8 - c2);
          decays = fmaf(pass[0][0], far, fmaf(pass[0][1], far - 1.0f, fmaf(pass[1][0], far + 8.0f, fmaf(pass[1][1], far + 7.0f, decays))));
          continue;
        }
        const int cc = c * 16 + h * 8 + c2;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float sum = pass[u][0] + pass[u][1];
          const float x1 = __shfl_up_sync(kAll, sum, 1, 4);
          if ((lane & 3) >= 1) sum += x1;
          const float x2 = __shfl_up_sync(kAll, sum, 2, 4);
          if ((lane & 3) >= 2) sum += x2;
          float left = __shfl_up_sync(kAll, sum, 1, 4);
          left = (lane & 3) ? before[u] + left : before[u];
          before[u] += __shfl_sync(kAll, sum, 3, 4);
          if (i0 + u * 8 >= cc) passes[c][h][0] += left;
          if (i0 + u * 8 >= cc + 1) passes[c][h][1] += left + pass[u][0];
        }
      }
      as_left(pf[r + c], sp[c]);
      as_left(df[r + c], so[c]);
    }
  }
  if (__any_sync(kAll, odd != odd)) {
    sum_decays(extra, a, p.batch, warp_backward_slow<S>(p, d, a, to, s, q, k, v, o, initial, n, lane), lane);
    return;
  }

  float x_rows[2][2] = {};  // x_i of the lane's rows, over its columns
  uint32_t dt[3][2][4];
#pragma unroll
  for (int t = 0; t < 3; ++t)
    if (t == 0 || nt > 1) transposed(dt[t], df[t]);
#pragma unroll 1
  for (int kt = 0; kt * 16 < dk; ++kt) {
    float dq[2][2][4] = {};
    if (initial) {
      float low[2][2][4] = {};
      const int row = kt * 16 + g;  // of the state: n of the product
#pragma unroll
      for (int kk = 0; kk < KT; ++kk) {
        if (kk * 16 >= dv) break;
        uint32_t b[2][2][3];  // [n half][channel half][limb]
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int c = kk * 16 + h * 8 + c2;
            const float* from = initial + (row + 8 * t) * dv + c;
            const bool there = row + 8 * t < dk;
            split<3>(FULL || (there && c < dv) ? from[0] : 0.0f, FULL || (there && c + 1 < dv) ? from[1] : 0.0f, b[t][h]);
          }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          if (r >= nt) break;
          uint32_t fa[4];
          frag_a<false>(fa, o + r * 16 * S::P + kk * 16, S::P, lane);
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            mma(low[r][t], fa, b[t][0][2], b[t][1][2]);
            mma(low[r][t], fa, b[t][0][1], b[t][1][1]);
            mma(dq[r][t], fa, b[t][0][0], b[t][1][0]);
          }
        }
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        if (r >= nt) break;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float f = s.carried[r * 16 + g + u * 8];
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const float2 x = values<1>(q + (r * 16 + g + u * 8) * S::P + kt * 16 + t * 8 + c2, 0);
            float &y0 = dq[r][t][2 * u], &y1 = dq[r][t][2 * u + 1];
            y0 = f == 0.0f ? 0.0f : (y0 + low[r][t][2 * u]) * (f * p.scale);
            y1 = f == 0.0f ? 0.0f : (y1 + low[r][t][2 * u + 1]) * (f * p.scale);
            x_rows[r][u] = fmaf(x.x, y0, fmaf(x.y, y1, x_rows[r][u]));
          }
        }
      }
    }
    float dk_[2][2][4] = {};
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      if (c >= nt) break;
      uint32_t fk[4], fq[4];
      frag_b<true>(fk, k + c * 16 * S::P + kt * 16, S::P, lane);
      frag_b<true>(fq, q + c * 16 * S::P + kt * 16, S::P, lane);
#pragma unroll
      for (int r = c; r < 2; ++r) {  // row tile r of dQ takes the keys of tiles c <= r
        if (r >= nt) break;
#pragma unroll
        for (int l = 1; l >= 0; --l)
#pragma unroll
          for (int t = 0; t < 2; ++t) mma(dq[r][t], df[r + c][l], fk[2 * t], fk[2 * t + 1]);
      }
#pragma unroll
      for (int r = 0; r <= c; ++r)  // row tile r of dK takes the queries of tiles c >= r
#pragma unroll
        for (int l = 1; l >= 0; --l)
#pragma unroll
          for (int t = 0; t < 2; ++t) mma(dk_[r][t], dt[r + c][l], fq[2 * t], fq[2 * t + 1]);
    }
    if (d.d_initial) {
      uint32_t w[2][3][4];
      weighted_left<S>(w, q, kt * 16, s.carried, p.scale, nt, lane);
      float* state = d.d_initial + int64_t(a.row) * state_size;
#pragma unroll
      for (int vt = 0; vt < KT; ++vt) {
        if (vt * 16 >= dv) break;
        float add[2][4];
        weighted_product<S>(add, w, o, vt * 16, nt, lane);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int row = kt * 16 + g + u * 8, c = vt * 16 + h * 8 + c2;
            if (FULL || (row < dk && c < dv)) {
              float* at = state + row * dv + c;
              write_pair(at, c, dv, dv % 2 == 0 && reinterpret_cast<uintptr_t>(at) % 8 == 0, add[h][2 * u], add[h][2 * u + 1]);
            }
          }
      }
    }
    if (to.shared_q) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float x[1][2][4], y[1][2][4];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[0][e >> 2][e & 3] = dq[r][e >> 2][e & 3], y[0][e >> 2][e & 3] = dk_[r][e >> 2][e & 3];
        store_float(to.shared_q, to.shared_stride, x, r * 16, kt * 16, n, dk, lane);
        store_float(to.shared_k, to.shared_stride, y, r * 16, kt * 16, n, dk, lane);
      }
    } else {
      __syncwarp();  // these columns of Q and K have been read
      stage_columns<S>(k, dq, kt * 16, nt, lane);
      stage_columns<S>(q, dk_, kt * 16, nt, lane);
    }
  }
#pragma unroll
  for (int t = 0; t < 3; ++t)
    if (t == 0 || nt > 1) transposed(dt[t], pf[t]);
#pragma unroll 1
  for (int vt = 0; vt * 16 < dv; ++vt) {
    float dv_[2][2][4] = {};
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      if (c >= nt) break;
      uint32_t fo[4];
      frag_b<true>(fo, o + c * 16 * S::P + vt * 16, S::P, lane);
#pragma unroll
      for (int r = 0; r <= c; ++r)
#pragma unroll
        for (int l = 1; l >= 0; --l)
#pragma unroll
          for (int t = 0; t < 2; ++t) mma(dv_[r][t], dt[r + c][l], fo[2 * t], fo[2 * t + 1]);
    }
    __syncwarp();
    stage_columns<S>(o, dv_, vt * 16, nt, lane);
  }
  // the decays
  if (each) {
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float y = passes[c][h][e];
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) y += __shfl_xor_sync(kAll, y, x);
          if (lane < 4) all.pass[c * 16 + h * 8 + c2 + e] = y;
        }
#pragma unroll
    for (int r = 0; r < 2; ++r) keep_rows(all.x, make_float2(x_rows[r][0], x_rows[r][1]), r, lane);
    __syncwarp();
    sum_decays(extra, a, p.batch, double(warp_decays(d, a, all.pass[lane], lane < n ? all.x[lane] : 0.0f, n, lane)), lane);
  } else {
#pragma unroll
    for (int r = 0; r < 2; ++r)  // the state in front passes every token up to a row's own
      decays = fmaf(x_rows[r][0], float(r * 16 + g + 1), fmaf(x_rows[r][1], float(r * 16 + g + 9), decays));
    sum_decays(extra, a, p.batch, double(decays), lane);
  }
  __syncwarp();
  if (!to.shared_q) {
    store_rows<S>(to.q, d.d_q.stride[1], k, dk, vec & kVecDq, n, mv);
    store_rows<S>(to.k, d.d_k.stride[1], q, dk, vec & kVecDk, n, mv);
  }
  store_rows<S>(to.v, d.d_v.stride[1], o, dv, vec & kVecDv, n, mv);
}

}  // namespace linear
}  // namespace zb
