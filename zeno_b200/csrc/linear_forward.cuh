// Linear attention with decays over a rollout, forward.  With c_i, e_j and a_ij the decays from the state in front of a
// chunk to token i, from token j to the chunk's end, and from j to i (0 across a reset):
//   o_i = scale (c_i S^T q_i + sum_{j <= i} a_ij (q_i . k_j) v_j),   S <- keep S + sum_j e_j k_j v_j^T
// One block takes one (environment, value head) and walks over its chunks, the state in the warps'
// accumulators.  Few long rollouts are cut into segments: one kernel sums what each segment adds to the state, one walks
// over the segments, and then every segment is a block of its own.
//
// What bounds it is neither bytes nor products: addresses, limbs and fragments are most of the instructions, and a chunk's steps wait
// for one another (1.5 instructions a cycle and SM, two blocks of 8 warps).  1024 x 64 tokens of 4 heads of 64 x 64: 32-bit 230 us (six products
// for one), bfloat16 at 2048 x 64 223 us.  Having the next chunk's rows on their way to L2 was worth 3 % and not kept.
#pragma once
#include "linear_mma.cuh"

namespace zb {
namespace linear {

// Rows and head of a block: the grid is [batch / kBatchAxis][batch][segments of a head][heads], the last the fastest, so that neighbouring
// blocks read neighbouring rows.
constexpr uint32_t kBatchAxis = 32768;
struct At {
  uint32_t row, b, h, kh, seg;
  int c0, c1, chunks;
};
__device__ __forceinline__ At block_at(const ZenoLinearAttention& p, const Segments& sg, uint32_t first, int C) {
  At a;
  a.b = blockIdx.z * kBatchAxis + blockIdx.y;
  a.h = blockIdx.x, a.seg = first;
  if (sg.count > 1) a.seg += blockIdx.x / p.value_heads, a.h = blockIdx.x % p.value_heads;
  a.row = a.b * p.value_heads + a.h;
  a.kh = p.value_heads == p.key_heads ? a.h : a.h / (p.value_heads / p.key_heads);
  a.chunks = (int(p.tokens) + C - 1) / C;
  a.c0 = int(a.seg * sg.chunks);
  a.c1 = a.seg + 1 == sg.count ? a.chunks : a.c0 + int(sg.chunks);
  return a;
}
inline dim3 grid_of(const ZenoLinearAttention& p, uint32_t segments) {
  return dim3(p.value_heads * segments, p.batch < kBatchAxis ? p.batch : kBatchAxis, (p.batch + kBatchAxis - 1) / kBatchAxis);
}

template <class S>
struct ForwardSmem {
  static constexpr int rows = 3 * S::L * S::PLANE, pairs = S::PL * S::CPLANE, state = S::PL * S::SPLANE;
  static constexpr int gates = int(sizeof(Gates<S::C>));
  static int bytes(bool with_state) { return gates + 2 * (rows + pairs + (with_state ? state : 0)); }
};

template <class S, int BLOCKS>
__global__ void __launch_bounds__(S::THREADS, BLOCKS) linear_forward_kernel(const __grid_constant__ ZenoLinearAttention p, const Segments sg) {
  using T = typename S::T;
  using M = ForwardSmem<S>;
  extern __shared__ __align__(16) char smem[];
  Gates<S::C>& s = *reinterpret_cast<Gates<S::C>*>(smem);
  plane_t* q = reinterpret_cast<plane_t*>(smem + M::gates);
  plane_t *k = q + S::L * S::PLANE, *v = k + S::L * S::PLANE, *pr = v + S::L * S::PLANE, *st = pr + M::pairs;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rt = warp % S::RT, ct = warp / S::RT;
  const int dk = S::FULL ? S::D : int(p.key_dim), dv = S::FULL ? S::D : int(p.value_dim), nk = (dk + 15) / 16;
  const At a = block_at(p, sg, 0, S::C);
  if (a.b >= p.batch) return;
  const Mover<S> mv(tid);
  const int64_t state_size = int64_t(dk) * dv;
  const T *gq = place<T>(p.q, a.b, a.kh), *gk = place<T>(p.k, a.b, a.kh), *gv = place<T>(p.v, a.b, a.h);
  const float* gg = place<float>(p.g, a.b, a.h);
  const uint8_t* gr = p.reset.data ? static_cast<const uint8_t*>(p.reset.data) + int64_t(a.b) * p.reset.stride[0] : nullptr;
  T* go = place<T>(p.out, a.b, a.h);

  const Part<S> part(warp, dk, dv);
  float m[S::NM][2][4];
  // (of several segments the first one's is a copy too: the last one may be writing over the initial state by now)
  const float* first = a.seg || (sg.count > 1 && p.initial_state) ? sg.state + (int64_t(a.row) * sg.count + a.seg) * state_size
                       : p.initial_state                          ? p.initial_state + int64_t(a.row) * state_size
                                                                  : nullptr;
  early::wait_for_previous();
  if (first) read_state<S>(m, first, part, dk, dv, lane);
  else clear<S>(m);

  for (int c = a.c0; c < a.c1; ++c) {
    const int64_t t0 = int64_t(c) * S::C;
    const int n = int(min(int64_t(S::C), int64_t(p.tokens) - t0)), nt = (n + 15) / 16;
    const bool have = c > a.c0 || first;
    __syncthreads();  // the last chunk's results have left
    GateIn<S::C> gates{};
    if (warp == S::NW - 1) gates = fetch_gates<S::C>(gg, p.g.stride[1], gr, p.reset.stride[1], t0, n, lane);
    load_rows<S>(q, gq + t0 * p.q.stride[1], p.q.stride[1], dk, sg.vec & kVecQ, n, nt, mv);
    load_rows<S>(k, gk + t0 * p.k.stride[1], p.k.stride[1], dk, sg.vec & kVecK, n, nt, mv);
    load_rows<S>(v, gv + t0 * p.v.stride[1], p.v.stride[1], dv, sg.vec & kVecV, n, nt, mv);
    if (warp == S::NW - 1) scan_gates<S::C>(s, gates, p.g.stride[1] == 0, n, lane);
    if (have) dump_state<S, S::PL>(m, st, part, lane);
    if (p.saved && c > 0) write_state<S>(m, p.saved + (int64_t(a.row) * (a.chunks - 1) + c - 1) * state_size, part, dk, dv, lane);
    copies_landed();
    __syncthreads();

    if (ct < S::NHS && rt < nt) {
      float acc[S::SP][2][4] = {};
      const int pairs = min(S::SP, rt - ct * S::SP + 1);  // up to the diagonal
      if (pairs > 0)
        product<S::L, S::L, false, false>(acc, q + rt * 16 * S::P, S::P, S::PLANE, k + ct * S::SP * 16 * S::P, S::P, S::PLANE, 0, nk, pairs, lane);
      const int i0 = rt * 16 + (lane >> 2);
      const Token ti[2] = {s.token[i0], s.token[i0 + 8]};
#pragma unroll
      for (int j = 0; j < S::SP; ++j) {
        if (j >= pairs) break;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int col = (ct * S::SP + j) * 16 + h * 8 + (lane & 3) * 2;
          const Token t0 = s.token[col], t1 = s.token[col + 1];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int i = i0 + r * 8;
            const bool m0 = meets(ti[r], t0, i, col), m1 = meets(ti[r], t1, i, col + 1);
            const float f0 = pair_decay(ti[r], t0, m0) * p.scale, f1 = pair_decay(ti[r], t1, m1) * p.scale;
            uint32_t w[S::PL];
            split<S::PL>(m0 ? acc[j][h][2 * r] * f0 : 0.0f, m1 ? acc[j][h][2 * r + 1] * f1 : 0.0f, w);
#pragma unroll
            for (int l = 0; l < S::PL; ++l) *reinterpret_cast<uint32_t*>(pr + l * S::CPLANE + i * S::CP + col) = w[l];
          }
        }
      }
    }
    __syncthreads();

    const int col = ct * S::NO * 16, pairs = rt >= nt ? 0 : S::FULL ? S::NO : min(S::NO, (dv - col + 15) / 16);
    float acc[S::NO][2][4] = {};
    bool bad = false;
    if (pairs > 0) {
      if (have) {
        product<S::L, S::PL, false, true>(acc, q + rt * 16 * S::P, S::P, S::PLANE, st + col, S::P, S::SPLANE, 0, nk, pairs, lane);
        const float c0 = s.carried[rt * 16 + (lane >> 2)], c1 = s.carried[rt * 16 + (lane >> 2) + 8];
#pragma unroll
        for (int j = 0; j < S::NO; ++j)
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            float& y = acc[j][x >> 2][x & 3];
            const float f = x & 2 ? c1 : c0;
            y = f == 0.0f ? 0.0f : y * (f * p.scale);
          }
      }
      product<S::PL, S::L, false, true>(acc, pr + rt * 16 * S::CP, S::CP, S::CPLANE, v + col, S::P, S::PLANE, 0, rt + 1, pairs, lane);
      bad = not_finite(acc);
    }
    bad = __syncthreads_or(bad);
    if (bad) {
      if (pairs > 0) {
#pragma unroll 1
        for (int x = 0; x < S::NO * 8; ++x) {
          const int i = rt * 16 + (lane >> 2) + ((x >> 1) & 1) * 8, cc = col + (x >> 3) * 16 + ((x >> 2) & 1) * 8 + (lane & 3) * 2 + (x & 1);
          if (i >= n || cc >= dv) continue;
          float y = 0.0f;
          if (have && s.carried[i] != 0.0f) {
            for (int d = 0; d < dk; ++d) y = fmaf(value<S::L>(q + i * S::P + d, S::PLANE), value<S::PL>(st + d * S::P + cc, S::SPLANE), y);
            y *= s.carried[i] * p.scale;
          }
          for (int j = 0; j <= i; ++j)
            if (pair_decay(s.token[i], s.token[j], meets(s.token[i], s.token[j], i, j)) != 0.0f)
              y = fmaf(value<S::PL>(pr + i * S::CP + j, S::CPLANE), value<S::L>(v + j * S::P + cc, S::PLANE), y);
#pragma unroll
          for (int z = 0; z < S::NO * 8; ++z)
            if (z == x) acc[z >> 3][(z >> 2) & 1][z & 3] = y;
        }
      }
      __syncthreads();
    }
    if constexpr (sizeof(T) == 2) stage<S>(q, acc, rt * 16, col, pairs, lane);
    else store_float(reinterpret_cast<float*>(go + t0 * p.out.stride[1]), p.out.stride[1], acc, rt * 16, col, n, pairs > 0 ? dv : 0, lane);
    if (c + 1 < a.c1 || (c + 1 == a.chunks && p.final_state)) {
      if (bad) update_masked<S>(m, k, v, s.to_end, 1.0f, s.keep, n, part, dk, dv, lane);
      else update<S>(m, k, v, s.to_end, 1.0f, s.keep, nt, part, lane);
    }
    if constexpr (sizeof(T) == 2) {
      __syncthreads();
      store_rows<S>(go + t0 * p.out.stride[1], p.out.stride[1], q, dv, sg.vec & kVecOut, n, mv);
    }
  }
  if (a.c1 == a.chunks && p.final_state) write_state<S>(m, p.final_state + int64_t(a.row) * state_size, part, dk, dv, lane);
}

// What each segment adds to the state behind it: X, Y and weights are K, V and e; in reverse (the gradient of the
// state) Q, dO and scale c, from the last chunk to the first.
template <class S, int BLOCKS>
__global__ void __launch_bounds__(S::THREADS, BLOCKS) linear_segment_kernel(const __grid_constant__ ZenoLinearAttention p, const ZenoTensor tx, const ZenoTensor ty,
                                                                    const Segments sg, const bool reverse) {  // (at most a few hundred rows)
  using T = typename S::T;
  extern __shared__ __align__(16) char smem[];
  Gates<S::C>& s = *reinterpret_cast<Gates<S::C>*>(smem);
  plane_t* x = reinterpret_cast<plane_t*>(smem + ForwardSmem<S>::gates);
  plane_t* y = x + S::L * S::PLANE;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int dk = S::FULL ? S::D : int(p.key_dim), dv = S::FULL ? S::D : int(p.value_dim);
  const At a = block_at(p, sg, reverse ? 1 : 0, S::C);
  const Mover<S> mv(tid);
  const T *gx = place<T>(tx, a.b, a.kh), *gy = place<T>(ty, a.b, a.h);
  const float* gg = place<float>(p.g, a.b, a.h);
  const uint8_t* gr = p.reset.data ? static_cast<const uint8_t*>(p.reset.data) + int64_t(a.b) * p.reset.stride[0] : nullptr;
  const bool vx = sg.vec & (reverse ? kVecQ : kVecK), vy = sg.vec & (reverse ? kVecOut : kVecV);
  const Part<S> part(warp, dk, dv);
  float m[S::NM][2][4];
  clear<S>(m);
  float kept = 1.0f;
  early::let_next_start();
  for (int step = 0; step < a.c1 - a.c0; ++step) {
    const int64_t t0 = int64_t(reverse ? a.c1 - 1 - step : a.c0 + step) * S::C;
    const int n = int(min(int64_t(S::C), int64_t(p.tokens) - t0)), nt = (n + 15) / 16;
    __syncthreads();
    GateIn<S::C> gates{};
    if (warp == S::NW - 1) gates = fetch_gates<S::C>(gg, p.g.stride[1], gr, p.reset.stride[1], t0, n, lane);
    load_rows<S>(x, gx + t0 * tx.stride[1], tx.stride[1], dk, vx, n, nt, mv);
    load_rows<S>(y, gy + t0 * ty.stride[1], ty.stride[1], dv, vy, n, nt, mv);
    if (warp == S::NW - 1) scan_gates<S::C>(s, gates, p.g.stride[1] == 0, n, lane);
    copies_landed();
    const bool bad = __syncthreads_or(rows_odd<S>(x, dk, nt, mv) || rows_odd<S>(y, dv, nt, mv));
    const float* weight = reverse ? s.carried : s.to_end;
    const float factor = reverse ? p.scale : 1.0f, keep = step ? s.keep : 0.0f;
    kept = both_keep(kept, s.keep);
    if (bad) update_masked<S>(m, x, y, weight, factor, keep, n, part, dk, dv, lane);
    else update<S>(m, x, y, weight, factor, keep, nt, part, lane);
  }
  const int64_t at = int64_t(a.row) * sg.count + a.seg;
  write_state<S>(m, sg.state + at * dk * dv, part, dk, dv, lane);
  if (tid == 0) sg.keep[at] = kept;
}

}  // namespace linear
}  // namespace zb
