// Gradients of the linear attention with decays.  With R the gradient of the state behind a chunk, S the state in front of
// it, f_ij = scale a_ij, P_ij = f_ij (q_i . k_j) and D_ij = f_ij (dO_i . v_j):
//   dq_i = scale c_i S dO_i + sum_{j <= i} D_ij k_j        dk_j = e_j R v_j   + sum_{i >= j} D_ij q_i
//   R   <- keep R + scale sum_i c_i q_i dO_i^T             dv_j = e_j R^T k_j + sum_{i >= j} P_ij dO_i
// The gradient of a log decay is the sum of all that passes its token, term by term: with A_ij = P_ij (dO_i . v_j),
// x_i = scale c_i q_i . S dO_i and y_j = e_j k_j . R v_j,
//   dg_t = sum_{i >= t > j} A_ij + sum_{i >= t} x_i + sum_{j < t} y_j + keep <S, R>
// so no difference of long sums is taken.  A block walks over its chunks from the last one back, R in the warps'
// accumulators; S comes from where the forward pass kept it.
//
// Bound as the forward pass is.  1024 x 64 tokens of 4 heads of 64 x 64: 32-bit 433 us (122 registers, 1.5 instructions a cycle and SM), bfloat16 at 2048 x 64 441 us.
#pragma once
#include "linear_forward.cuh"

namespace zb {
namespace linear {

template <class S>
struct BackwardSmem {
  struct Sums {
    float x[S::NH][S::C], y[S::NH][S::C];  // x_i and y_j over each group of columns
    float pairs[S::RT][S::C];              // sum over the rows of a tile i >= t of the A_ij in front of t in t's group of columns
    float row[S::NHS][S::C];               // sum of A_ij over each group of columns
    float state[S::NW];                    // <S, R> over each warp's part
  };
  static constexpr int row = S::L * S::PLANE, pairs = S::PL * S::CPLANE, state = 3 * S::SPLANE;
  static constexpr int front = int(sizeof(Gates<S::C>)) + (int(sizeof(Sums)) + 15) / 16 * 16;
  static int bytes(bool with_state) { return front + 2 * (4 * row + 2 * pairs + (with_state ? state : 0)); }
};

struct BackwardOut {
  float *shared_q, *shared_k;  // [batch][tokens][value heads][dk], where value heads share a key head
  double* decay;               // [value heads][batch][segments], where all tokens of a head have one decay
};

// acc's rows by f[i] (what f is zero for is left out).  Returns the products of the lane's two rows with those of X over its columns:
// summed over the 4 lanes of a row and the groups of columns they are x_i.
template <class S>
__device__ __forceinline__ float2 scale_and_dot(float (&acc)[S::NO][2][4], const float* f, float scale, const plane_t* x, int rt, int ct, int pairs,
                                                int lane) {
  const int i0 = rt * 16 + (lane >> 2);
  const float f0 = f[i0], f1 = f[i0 + 8];
  const float s0 = f0 * scale, s1 = f1 * scale;
  float d0 = 0.0f, d1 = 0.0f;
#pragma unroll
  for (int j = 0; j < S::NO; ++j) {
    if (j >= pairs) break;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float(&y)[4] = acc[j][h];
      const plane_t* at = x + i0 * S::P + (ct * S::NO + j) * 16 + h * 8 + (lane & 3) * 2;
      const float2 x0 = values<S::L>(at, S::PLANE), x1 = values<S::L>(at + 8 * S::P, S::PLANE);
      y[0] = f0 == 0.0f ? 0.0f : y[0] * s0, y[1] = f0 == 0.0f ? 0.0f : y[1] * s0;
      y[2] = f1 == 0.0f ? 0.0f : y[2] * s1, y[3] = f1 == 0.0f ? 0.0f : y[3] * s1;
      d0 = fmaf(x0.x, y[0], fmaf(x0.y, y[1], d0)), d1 = fmaf(x1.x, y[2], fmaf(x1.y, y[3], d1));
    }
  }
  // f == 0: the row of x may hold anything
  return make_float2(f0 == 0.0f ? 0.0f : d0, f1 == 0.0f ? 0.0f : d1);
}
__device__ __forceinline__ void keep_rows(float* to, float2 x, int rt, int lane) {
  x.x += __shfl_xor_sync(kAll, x.x, 1), x.y += __shfl_xor_sync(kAll, x.y, 1);
  x.x += __shfl_xor_sync(kAll, x.x, 2), x.y += __shfl_xor_sync(kAll, x.y, 2);
  if ((lane & 3) == 0) to[rt * 16 + (lane >> 2)] = x.x, to[rt * 16 + (lane >> 2) + 8] = x.y;
}

// One element of a gradient over the pairs that the mask leaves: factor (state row . x) + sum over the pairs.
//   state: f * sum_w st[.][w] x[w], the state's element stride `ss`; pairs (i, j) of P or D with y.
template <class S, bool ROWS>
__device__ __noinline__ float masked_element(const Gates<S::C>& s, float f, const plane_t* x, const plane_t* st, int ss, int width, const plane_t* pairs,
                                             const plane_t* y, int at, int n) {
  float sum = 0.0f;
  if (f != 0.0f) {
    for (int w = 0; w < width; ++w) sum = fmaf(value<S::L>(x + w, S::PLANE), value<3>(st + w * ss, S::SPLANE), sum);
    sum *= f;
  }
  for (int o = ROWS ? 0 : at; o < (ROWS ? at + 1 : n); ++o) {
    const int i = ROWS ? at : o, j = ROWS ? o : at;
    if (pair_decay(s.token[i], s.token[j], meets(s.token[i], s.token[j], i, j)) != 0.0f) sum = fmaf(value<S::PL>(pairs + i * S::CP + j, S::CPLANE), value<S::L>(y + o * S::P, S::PLANE), sum);
  }
  return sum;
}

template <class S, class F>
__device__ __forceinline__ void again(float (&acc)[S::NO][2][4], int rt, int col, int n, int width, int lane, F&& element) {
#pragma unroll 1
  for (int x = 0; x < S::NO * 8; ++x) {
    const int i = rt * 16 + (lane >> 2) + ((x >> 1) & 1) * 8, c = col + (x >> 3) * 16 + ((x >> 2) & 1) * 8 + (lane & 3) * 2 + (x & 1);
    if (i >= n || c >= width) continue;
    const float y = element(i, c);
#pragma unroll
    for (int z = 0; z < S::NO * 8; ++z)
      if (z == x) acc[z >> 3][(z >> 2) & 1][z & 3] = y;
  }
}

template <class S, int BLOCKS>
__global__ void __launch_bounds__(S::THREADS, BLOCKS)
linear_backward_kernel(const __grid_constant__ ZenoLinearAttention p, const __grid_constant__ ZenoLinearAttentionGrads d, const Segments sg,
                       const BackwardOut extra) {
  using T = typename S::T;
  using M = BackwardSmem<S>;
  extern __shared__ __align__(16) char smem[];
  Gates<S::C>& s = *reinterpret_cast<Gates<S::C>*>(smem);
  typename M::Sums& sums = *reinterpret_cast<typename M::Sums*>(smem + sizeof(Gates<S::C>));
  plane_t* q = reinterpret_cast<plane_t*>(smem + M::front);
  plane_t *k = q + M::row, *v = k + M::row, *o = v + M::row, *pr = o + M::row, *dp = pr + M::pairs, *st = dp + M::pairs;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rt = warp % S::RT, ct = warp / S::RT;
  const int dk = S::FULL ? S::D : int(p.key_dim), dv = S::FULL ? S::D : int(p.value_dim), nk = (dk + 15) / 16, nv = (dv + 15) / 16;
  const At a = block_at(p, sg, 0, S::C);
  if (a.b >= p.batch) return;
  const Mover<S> mv(tid);
  const int64_t state_size = int64_t(dk) * dv;
  const bool shared = extra.shared_q != nullptr;
  const T *gq = place<T>(p.q, a.b, a.kh), *gk = place<T>(p.k, a.b, a.kh), *gv = place<T>(p.v, a.b, a.h), *go = place<T>(d.d_out, a.b, a.h);
  const float* gg = place<float>(p.g, a.b, a.h);
  const uint8_t* gr = p.reset.data ? static_cast<const uint8_t*>(p.reset.data) + int64_t(a.b) * p.reset.stride[0] : nullptr;
  T *wq = place<T>(d.d_q, a.b, a.kh), *wk = place<T>(d.d_k, a.b, a.kh), *wv = place<T>(d.d_v, a.b, a.h);
  const int64_t shared_stride = int64_t(p.value_heads) * dk;

  const Part<S> part(warp, dk, dv);
  float m[S::NM][2][4];
  const bool last_segment = a.c1 == a.chunks;
  const float* behind = !last_segment ? sg.state + (int64_t(a.row) * sg.count + a.seg) * state_size
                                      : d.d_final ? d.d_final + int64_t(a.row) * state_size : nullptr;
  early::wait_for_previous();
  if (behind) read_state<S>(m, behind, part, dk, dv, lane);
  else clear<S>(m);
  const bool each = d.d_g.data != nullptr;  // every token's decay has a gradient of its own
  double decay_sum = 0.0;
  const int col = ct * S::NO * 16;

  for (int c = a.c1 - 1; c >= a.c0; --c) {
    const int64_t t0 = int64_t(c) * S::C;
    const int n = int(min(int64_t(S::C), int64_t(p.tokens) - t0)), nt = (n + 15) / 16;
    const float* front = c > 0 ? p.saved + (int64_t(a.row) * (a.chunks - 1) + c - 1) * state_size
                               : p.initial_state ? p.initial_state + int64_t(a.row) * state_size : nullptr;
    const bool have_r = c + 1 < a.c1 || behind;
    __syncthreads();  // the last chunk's results have left
    GateIn<S::C> gates{};
    if (warp == S::NW - 1) gates = fetch_gates<S::C>(gg, p.g.stride[1], gr, p.reset.stride[1], t0, n, lane);
    load_rows<S>(q, gq + t0 * p.q.stride[1], p.q.stride[1], dk, sg.vec & kVecQ, n, nt, mv);
    load_rows<S>(k, gk + t0 * p.k.stride[1], p.k.stride[1], dk, sg.vec & kVecK, n, nt, mv);
    load_rows<S>(v, gv + t0 * p.v.stride[1], p.v.stride[1], dv, sg.vec & kVecV, n, nt, mv);
    load_rows<S>(o, go + t0 * d.d_out.stride[1], d.d_out.stride[1], dv, sg.vec & kVecOut, n, nt, mv);
    if (warp == S::NW - 1) scan_gates<S::C>(s, gates, p.g.stride[1] == 0, n, lane);
    float state_dot = 0.0f;  // <S, R> over this thread's elements
    if (front) {
      float x[S::NM][2][4];
      read_state<S>(x, front, part, dk, dv, lane);
      float dot = 0.0f;
#pragma unroll
      for (int j = 0; j < S::NM; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) dot = fmaf(x[j][e >> 2][e & 3], m[j][e >> 2][e & 3], dot);
      dump_state<S, 3>(x, st, part, lane);
      state_dot = have_r ? dot : 0.0f;
      if (each) {
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) dot += __shfl_xor_sync(kAll, dot, x);
        if (lane == 0) sums.state[warp] = dot;
      }
    }
    copies_landed();
    __syncthreads();

    // P, D, and what the pairs give the decays
    // this thread's part of their gradient, where all tokens of the head have one
    float decays = each || s.keep == 0.0f ? 0.0f : state_dot * s.keep * float(n);
    if (ct < S::NHS) {
      float sp[S::SP][2][4] = {}, so[S::SP][2][4] = {};
      const int pairs = rt < nt ? min(S::SP, rt - ct * S::SP + 1) : 0;
      if (pairs > 0) {
        product<S::L, S::L, false, false>(sp, q + rt * 16 * S::P, S::P, S::PLANE, k + ct * S::SP * 16 * S::P, S::P, S::PLANE, 0, nk, pairs, lane);
        product<S::L, S::L, false, false>(so, o + rt * 16 * S::P, S::P, S::PLANE, v + ct * S::SP * 16 * S::P, S::P, S::PLANE, 0, nv, pairs, lane);
      }
      const int i0 = rt * 16 + (lane >> 2);
      const Token ti[2] = {s.token[i0], s.token[i0 + 8]};
      float before[2] = {0.0f, 0.0f};  // of the group's columns so far, for each of the lane's two rows
#pragma unroll
      for (int j = 0; j < S::SP; ++j) {
        const int c0 = (ct * S::SP + j) * 16;
        if (j >= pairs) {
          // nothing lies in front of these columns' tokens but what lies to the left
          if (each && lane < 16) sums.pairs[rt][c0 + lane] = 0.0f;
          continue;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int cc = c0 + h * 8 + (lane & 3) * 2;
          const Token t0 = s.token[cc], t1 = s.token[cc + 1];
          float pass[2][2];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int i = i0 + r * 8;
            const bool m0 = meets(ti[r], t0, i, cc), m1 = meets(ti[r], t1, i, cc + 1);
            const float f0 = pair_decay(ti[r], t0, m0) * p.scale, f1 = pair_decay(ti[r], t1, m1) * p.scale;
            const float o0 = so[j][h][2 * r], o1 = so[j][h][2 * r + 1];
            const float p0 = m0 ? sp[j][h][2 * r] * f0 : 0.0f, p1 = m1 ? sp[j][h][2 * r + 1] * f1 : 0.0f;
            uint32_t w[S::PL];
            split<S::PL>(p0, p1, w);
#pragma unroll
            for (int l = 0; l < S::PL; ++l) *reinterpret_cast<uint32_t*>(pr + l * S::CPLANE + i * S::CP + cc) = w[l];
            split<S::PL>(m0 ? o0 * f0 : 0.0f, m1 ? o1 * f1 : 0.0f, w);
#pragma unroll
            for (int l = 0; l < S::PL; ++l) *reinterpret_cast<uint32_t*>(dp + l * S::CPLANE + i * S::CP + cc) = w[l];
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
            // the sum of A in front of each column, over the 4 lanes of the row
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
      }
      if (each && (lane & 3) == 0) {
        sums.row[ct][i0] = before[0];
        sums.row[ct][i0 + 8] = before[1];
      }
    }
    __syncthreads();

    // dQ
    const int pk = rt >= nt ? 0 : S::FULL ? S::NO : min(S::NO, (dk - col + 15) / 16), pv = rt >= nt ? 0 : S::FULL ? S::NO : min(S::NO, (dv - col + 15) / 16);  // column tiles of this warp
    float dq[S::NO][2][4] = {};
    bool bad = false;
    if (pk > 0) {
      if (front) {
        product<S::L, 3, false, false>(dq, o + rt * 16 * S::P, S::P, S::PLANE, st + col * S::P, S::P, S::SPLANE, 0, nv, pk, lane);
        const float2 x = scale_and_dot<S>(dq, s.carried, p.scale, q, rt, ct, pk, lane);
        const float i = float(rt * 16 + (lane >> 2));
        if (each) keep_rows(sums.x[ct], x, rt, lane);
        else decays = fmaf(x.x, i + 1.0f, fmaf(x.y, i + 9.0f, decays));  // the state in front passes every token up to this one
      }
      product<S::PL, S::L, false, true>(dq, dp + rt * 16 * S::CP, S::CP, S::CPLANE, k + col, S::P, S::PLANE, 0, rt + 1, pk, lane);
      bad = not_finite(dq);
    }
    if (__syncthreads_or(bad)) {
      if (pk > 0)
        again<S>(dq, rt, col, n, dk, lane, [&](int i, int cc) {
          return masked_element<S, true>(s, front ? s.carried[i] * p.scale : 0.0f, o + i * S::P, st + cc * S::P, 1, dv, dp, k + cc, i, n);
        });
      __syncthreads();
    }
    if (have_r) {
      dump_state<S, 3>(m, st, part, lane);
      __syncthreads();
    }

    // dK, dV
    float dk_[S::NO][2][4] = {}, dv_[S::NO][2][4] = {};
    bad = false;
    if (pk > 0) {
      if (have_r) {
        product<S::L, 3, false, false>(dk_, v + rt * 16 * S::P, S::P, S::PLANE, st + col * S::P, S::P, S::SPLANE, 0, nv, pk, lane);
        const float2 y = scale_and_dot<S>(dk_, s.to_end, 1.0f, k, rt, ct, pk, lane);
        const float rest = float(n - 1 - rt * 16 - (lane >> 2));
        if (each) keep_rows(sums.y[ct], y, rt, lane);
        else decays += (rest == 0.0f ? 0.0f : y.x * rest) + (rest == 8.0f ? 0.0f : y.y * (rest - 8.0f));  // what begins here passes the tokens behind it
      }
      product<S::PL, S::L, true, true>(dk_, dp + rt * 16, S::CP, S::CPLANE, q + col, S::P, S::PLANE, rt, nt, pk, lane);
      bad = not_finite(dk_);
    }
    if (pv > 0) {
      if (have_r) {
        product<S::L, S::PL, false, true>(dv_, k + rt * 16 * S::P, S::P, S::PLANE, st + col, S::P, S::SPLANE, 0, nk, pv, lane);
        const float e0 = s.to_end[rt * 16 + (lane >> 2)], e1 = s.to_end[rt * 16 + (lane >> 2) + 8];
#pragma unroll
        for (int j = 0; j < S::NO; ++j)
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            float& y = dv_[j][x >> 2][x & 3];
            const float e = x & 2 ? e1 : e0;
            y = e == 0.0f ? 0.0f : y * e;
          }
      }
      product<S::PL, S::L, true, true>(dv_, pr + rt * 16, S::CP, S::CPLANE, o + col, S::P, S::PLANE, rt, nt, pv, lane);
      bad |= not_finite(dv_);
    }
    bad = __syncthreads_or(bad);
    if (bad) {
      if (pk > 0)
        again<S>(dk_, rt, col, n, dk, lane, [&](int j, int cc) {
          return masked_element<S, false>(s, have_r ? s.to_end[j] : 0.0f, v + j * S::P, st + cc * S::P, 1, dv, dp, q + cc, j, n);
        });
      if (pv > 0)
        again<S>(dv_, rt, col, n, dv, lane, [&](int j, int cc) {
          return masked_element<S, false>(s, have_r ? s.to_end[j] : 0.0f, k + j * S::P, st + cc, S::P, dk, pr, o + cc, j, n);
        });
      __syncthreads();
    }
    // results, bfloat16 by way of rows that are not needed any more (Q and dO still are)
    if constexpr (sizeof(T) == 2) {
      if (!shared) {
        stage<S>(k, dq, rt * 16, col, pk, lane);
        stage<S>(v, dk_, rt * 16, col, pk, lane);
      }
      stage<S>(pr, dv_, rt * 16, col, pv, lane);
    } else {
      if (!shared) {
        store_float(reinterpret_cast<float*>(wq + t0 * d.d_q.stride[1]), d.d_q.stride[1], dq, rt * 16, col, n, dk, lane);
        store_float(reinterpret_cast<float*>(wk + t0 * d.d_k.stride[1]), d.d_k.stride[1], dk_, rt * 16, col, n, dk, lane);
      }
      store_float(reinterpret_cast<float*>(wv + t0 * d.d_v.stride[1]), d.d_v.stride[1], dv_, rt * 16, col, n, dv, lane);
    }
    if (shared) {
      const int64_t at = (int64_t(a.b) * p.tokens + t0) * shared_stride + int64_t(a.h) * dk;
      store_float(extra.shared_q + at, shared_stride, dq, rt * 16, col, n, dk, lane);
      store_float(extra.shared_k + at, shared_stride, dk_, rt * 16, col, n, dk, lane);
    }
    // the decays: a warp, C / 32 neighbouring tokens a lane
    decay_sum += double(decays);
    if (each && warp == S::NW - 1) {
      constexpr int U = S::C / 32;
      float z = 0.0f;
      if (front && have_r && s.keep != 0.0f) {
#pragma unroll 1
        for (int w = 0; w < S::NW; ++w) z += sums.state[w];
        z *= s.keep;
      }
      float dg[U];
      // behind: what ends at this token or after it; ahead: what begins in front of it
      float behind_[U], ahead[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int t = lane * U + u;
        behind_[u] = ahead[u] = 0.0f;
        if (t < n) {
#pragma unroll
          for (int x = 0; x < S::NH; ++x) {
            if (x * S::NO * 16 >= dk) break;
            if (front) behind_[u] += sums.x[x][t];
            if (have_r) ahead[u] += sums.y[x][t];
          }
        }
        dg[u] = z;
#pragma unroll
        for (int r = 0; r < S::RT; ++r)
          if (t < n && r < nt && r * 16 + 15 >= t) dg[u] += sums.pairs[r][t];
      }
      // sums over the tokens in front (exclusive) and from this one on
      float in_front = 0.0f, from_here = 0.0f;
#pragma unroll
      for (int u = 0; u < U; ++u) in_front += ahead[u], from_here += behind_[u];
#pragma unroll
      for (int x = 1; x < 32; x <<= 1) {
        const float y0 = __shfl_up_sync(kAll, in_front, x), y1 = __shfl_down_sync(kAll, from_here, x);
        if (lane >= x) in_front += y0;
        if (lane + x < 32) from_here += y1;
      }
      in_front = __shfl_up_sync(kAll, in_front, 1), from_here = __shfl_down_sync(kAll, from_here, 1);
      if (lane == 0) in_front = 0.0f;
      if (lane == 31) from_here = 0.0f;
#pragma unroll
      for (int u = 0; u < U; ++u) dg[u] += in_front, in_front += ahead[u];
#pragma unroll
      for (int u = U - 1; u >= 0; --u) from_here += behind_[u], dg[u] += from_here;
      // pairs whose first token lies in an earlier group of columns
#pragma unroll
      for (int x = 0; x + 1 < S::NHS; ++x) {
        float rest[U], sum = 0.0f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int t = lane * U + u;
          rest[u] = t < n ? sums.row[x][t] : 0.0f;
          sum += rest[u];
        }
#pragma unroll
        for (int y = 1; y < 32; y <<= 1) {
          const float w = __shfl_down_sync(kAll, sum, y);
          if (lane + y < 32) sum += w;
        }
        float here = __shfl_down_sync(kAll, sum, 1);
        if (lane == 31) here = 0.0f;
#pragma unroll
        for (int u = U - 1; u >= 0; --u) {
          here += rest[u];
          if (lane * U + u >= (x + 1) * S::SP * 16) dg[u] += here;
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int t = lane * U + u;
        if (t < n) {
          decay_sum += double(dg[u]);
          place<float>(d.d_g, a.b, a.h)[(t0 + t) * d.d_g.stride[1]] = dg[u];
        }
      }
    }
    if (c > a.c0 || (c == 0 && d.d_initial)) {
      if (bad) update_masked<S>(m, q, o, s.carried, p.scale, s.keep, n, part, dk, dv, lane);
      else update<S>(m, q, o, s.carried, p.scale, s.keep, nt, part, lane);
    }
    if constexpr (sizeof(T) == 2) {
      __syncthreads();
      if (!shared) {
        store_rows<S>(wq + t0 * d.d_q.stride[1], d.d_q.stride[1], k, dk, sg.vec & kVecDq, n, mv);
        store_rows<S>(wk + t0 * d.d_k.stride[1], d.d_k.stride[1], v, dk, sg.vec & kVecDk, n, mv);
      }
      store_rows<S>(wv + t0 * d.d_v.stride[1], d.d_v.stride[1], pr, dv, sg.vec & kVecDv, n, mv);
    }
  }
  if (a.c0 == 0 && d.d_initial) write_state<S>(m, d.d_initial + int64_t(a.row) * state_size, part, dk, dv, lane);
  if (extra.decay) {
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) decay_sum += __shfl_xor_sync(kAll, decay_sum, x);
    double* part_sum = reinterpret_cast<double*>(smem);  // (where the gates were)
    __syncthreads();
    if (lane == 0) part_sum[warp] = decay_sum;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < S::NW; ++w) decay_sum += part_sum[w];
      extra.decay[(uint64_t(a.h) * p.batch + a.b) * sg.count + a.seg] = decay_sum;
    }
  }
}

}  // namespace linear
}  // namespace zb
