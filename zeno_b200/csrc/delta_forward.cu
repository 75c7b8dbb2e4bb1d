// Gated delta rule over a rollout, chunked: 32 tokens at a time meet the state in matrix
// products instead of one by one.
//
// With S0 the state in front of a chunk, G the running sum of its log decays,
// D_ij = exp(G_i - G_j) (0 across an episode's begin) and a_i = exp(G_i) (0 behind one):
//   N_ij = D_ij (k_i . k_j) beta_j  (j < i),   (I + N) W = V - a K S0,   U = beta W
//   O = a Q S0 + P U,  P_ij = D_ij (q_i . k_j)  (j <= i),   S <- a_C S0 + K^T (D_C U)
//
// A block has one (environment, head).  Each of its warps owns 16 value channels and holds
// their columns of the state, transposed, as the accumulators of 16-bit matrix
// instructions for the whole rollout.  Written with everything transposed
// (W^T = E^T (I + N)^-T, O^T = S^T Q^T + U^T P^T, S^T <- S^T + U^T K) each product's left
// operand is the previous one's accumulators, so state, errors and outputs never leave the
// registers, and warps meet only where the token-by-token matrices are made.
#include "delta_mma.cuh"

namespace zb {
namespace delta {
namespace {

template <int DK, int NW, class T>
struct ForwardSmem {
  static constexpr int L = In<T>::limbs;
  Gates gates;
  Pairs pairs;
  Squares squares;
  __align__(16) __half q[L][C * (DK + 8)];
  __align__(16) __half k[L][C * (DK + 8)];
  __align__(16) T v[C * (16 * NW + 16 / int(sizeof(T)))];
};

template <int DK, int NW, class T>
// Threads of an SM: 512 where the state is 32 registers a thread (4096 x 32 tokens, 64 x 64: 461 us against 544 with
// 384 and 714 with 256), 384 where it is 64 (2 x 4096 tokens, 128 x 128: 1250 us against 1405 with 512).
__global__ void __launch_bounds__(NW * 32, (DK <= 64 ? 512 : 384) / (NW * 32)) delta_forward_kernel(const __grid_constant__ ZenoDeltaRule p) {
  extern __shared__ __align__(16) unsigned char raw[];
  using Smem = ForwardSmem<DK, NW, T>;
  constexpr int L = In<T>::limbs;
  Smem& sm = *reinterpret_cast<Smem*>(raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int qj = (lane & 3) * 2;
  const uint32_t h = blockIdx.x % p.value_heads, b = blockIdx.x / p.value_heads;
  const int dk = int(p.key_dim), dv = int(p.value_dim);
  const int v0 = int(blockIdx.y) * 16 * NW;
  const int c0 = v0 + warp * 16;  // the warp's first channel
  const Rows<T> rows = rows_of<T>(p, b, h);
  T* out = static_cast<T*>(p.out.data) + int64_t(b) * p.out.stride[0] + int64_t(h) * p.out.stride[2];
  const bool pairs_ok = sizeof(T) == 2 && dv % 2 == 0 && reinterpret_cast<uintptr_t>(p.out.data) % 4 == 0 &&
                        ((p.out.stride[0] | p.out.stride[1] | p.out.stride[2]) & 1) == 0;
  const int64_t state_at = int64_t(blockIdx.x) * dk * dv;

  float st[DK / 8][4] = {};
  if (p.initial_state)
    for_state<DK, 16 * NW>(st, dk, dv, c0, lane, [&](float& x, int64_t at) { x = p.initial_state[state_at + at]; });
  bool has_state = p.initial_state != nullptr;  // there is a state in front of the chunk
  if (tid == 0) sm.gates.bad = 0, sm.gates.state_bad = 0;
  __syncthreads();

  const int64_t T_ = p.tokens;
  const int64_t chunks = (T_ + C - 1) / C;
  for (int64_t chunk = 0; chunk < chunks; ++chunk) {
    const int64_t t0 = chunk * C, t1 = min(t0 + C, T_);
    if (p.saved && chunk > 0) {
      const int64_t width = int64_t(gridDim.y) * 16 * NW;
      float4* to = reinterpret_cast<float4*>(p.saved + ((int64_t(blockIdx.x) * (chunks - 1) + chunk - 1) * width + c0) * DK);
#pragma unroll
      for (int n = 0; n < DK / 8; ++n) __stcs(to + n * 32 + lane, make_float4(st[n][0], st[n][1], st[n][2], st[n][3]));
    }
    for (int64_t lo = t0; lo < t1;) {
      int64_t hi = t1;
      int e0, e1;
      if (!row_exps_finite<DK / 8>(st, e0, e1)) sm.gates.state_bad = 1;
#pragma unroll 1
      for (;;) {
        GateIn gates{};
        if (warp == 0) gates = fetch_gates(p, rows.g, rows.beta, rows.reset, t0, lo, hi, lane);
        load_rows<DK, NW, T, false>(sm.gates, p, rows, sm.q[0], sm.k[0], sm.v, v0, t0, lo, hi, tid);
        if (warp == 0) scan_gates(sm.gates, gates, lane);
        __syncthreads();
        // A value that is not finite must not reach another episode, nor an earlier token,
        // through a product with zero: such a chunk is taken token by token.
        if (hi - lo == 1 || !(sm.gates.bad || (sm.gates.state_bad && sm.gates.marks != 0))) break;
        hi = lo + 1;
        __syncthreads();
      }
      if (t1 < T_) prefetch_rows<NW>(p, rows, t1, v0, tid);
      pair_matrices<DK, NW, L, false>(sm.gates, sm.pairs, sm.squares, nullptr, sm.q[0], sm.k[0], warp, lane);
      __syncthreads();

      // E^T = V^T - a (S0^T K^T), O^T = a (S0^T Q^T)
      float e[4][4] = {}, o[4][4] = {};
      if (has_state) {
        const float s0 = pow2_scale(e0), s1 = pow2_scale(e1);
#pragma unroll
        for (int kk = 0; kk < DK; kk += 16) {
          uint32_t ah[4], al[4];
          split_a(ah, al, st[kk / 8], st[kk / 8 + 1], s0, s1);
          state_times_rows<DK, L>(e, ah, al, sm.k[0], kk, lane);
          state_times_rows<DK, L>(o, ah, al, sm.q[0], kk, lane);
        }
      }
      const float f0 = pow2_unscale(e0), f1 = pow2_unscale(e1);
      float v[4][4];
      load_values(v, sm.v + warp * 16, 16 * NW + 16 / int(sizeof(T)), lane);
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const float2 ak = *reinterpret_cast<const float2*>(&sm.gates.ak[n * 8 + qj]);
        const float2 aq = *reinterpret_cast<const float2*>(&sm.gates.aq[n * 8 + qj]);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float a = x & 1 ? ak.y : ak.x, b = (x & 1 ? aq.y : aq.x) * p.scale, f = x < 2 ? f0 : f1;
          // a dropped state contributes nothing, whatever it held
          e[n][x] = a == 0.0f ? v[n][x] : fmaf(-e[n][x], f * a, v[n][x]);
          o[n][x] = a == 0.0f ? 0.0f : o[n][x] * (f * b);
        }
      }
      solve_forward(e, sm.pairs, lane);  // now W^T
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const float2 be = *reinterpret_cast<const float2*>(&sm.gates.beta[n * 8 + qj]);
#pragma unroll
        for (int x = 0; x < 4; ++x) e[n][x] *= x & 1 ? be.y : be.x;  // U^T
      }
      {  // O^T += U^T P^T
        row_exps<4>(e, e0, e1);
        const float s0 = pow2_scale(e0), s1 = pow2_scale(e1), g0 = pow2_unscale(e0), g1 = pow2_unscale(e1);
        uint32_t uh[2][4], ul[2][4];
#pragma unroll
        for (int r = 0; r < 2; ++r) split_a(uh[r], ul[r], e[2 * r], e[2 * r + 1], s0, s1);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float acc[2][4] = {};
#pragma unroll
          for (int r = 0; r <= i; ++r) {
            uint32_t bh[4], bl[4];
            b_rows(bh, sm.pairs.p[0] + i * 16 * CP + r * 16, CP, lane);
            b_rows(bl, sm.pairs.p[1] + i * 16 * CP + r * 16, CP, lane);
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              mma(acc[n], uh[r], bh[2 * n], bh[2 * n + 1]);
              mma(acc[n], ul[r], bh[2 * n], bh[2 * n + 1]);
              mma(acc[n], uh[r], bl[2 * n], bl[2 * n + 1]);
            }
          }
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const float2 fp = *reinterpret_cast<const float2*>(&sm.pairs.fp[i * 16 + n * 8 + qj]);
#pragma unroll
            for (int x = 0; x < 4; ++x)
              o[2 * i + n][x] = fmaf(acc[n][x], (x < 2 ? g0 : g1) * p.scale * (x & 1 ? fp.y : fp.x), o[2 * i + n][x]);
          }
        }
      }
      store_out(o, out, p.out.stride[1], t0, lo, hi, c0, dv, pairs_ok, lane);
      // S^T <- a_C S^T + (D_C U)^T K
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const float2 zk = *reinterpret_cast<const float2*>(&sm.gates.zk[n * 8 + qj]);
#pragma unroll
        for (int x = 0; x < 4; ++x) e[n][x] *= x & 1 ? zk.y : zk.x;
      }
      state_update<DK, L>(st, sm.gates.keep, e, sm.k[0], lane);
      has_state = true;
      __syncthreads();
      if (tid == 0) sm.gates.bad = 0, sm.gates.state_bad = 0;
      __syncthreads();
      lo = hi;
    }
  }
  if (p.final_state)
    for_state<DK, 16 * NW>(st, dk, dv, c0, lane, [&](float& x, int64_t at) { p.final_state[state_at + at] = x; });
}

template <int DK, int NW, class T>
cudaError_t launch(const ZenoDeltaRule& p, cudaStream_t stream) {
  const auto kernel = delta_forward_kernel<DK, NW, T>;
  constexpr int smem = int(sizeof(ForwardSmem<DK, NW, T>));
  static std::atomic<uint64_t> allowed{0};
  const cudaError_t e = allow_smem(kernel, smem, allowed);
  if (e != cudaSuccess) return e;
  const dim3 grid(p.batch * p.value_heads, (p.value_dim + 16 * NW - 1) / (16 * NW));
  kernel<<<grid, NW * 32, smem, stream>>>(p);
  return cudaGetLastError();
}

template <int DK, class T>
cudaError_t by_width(const ZenoDeltaRule& p, cudaStream_t stream) {
  switch (value_warps(p)) {
    case 2:
      if constexpr (DK < 128) return launch<DK, 2, T>(p, stream);
    case 4: return launch<DK, 4, T>(p, stream);
    default: return launch<DK, 8, T>(p, stream);
  }
}

template <class T>
cudaError_t by_type(const ZenoDeltaRule& p, cudaStream_t stream) {
  switch (key_width(p)) {
    case 32: return by_width<32, T>(p, stream);
    case 64: return by_width<64, T>(p, stream);
    default: return by_width<128, T>(p, stream);
  }
}

}  // namespace
}  // namespace delta

// The states in front of every chunk but the first (that one is initial_state), in the
// accumulators' order: [batch * heads][chunks - 1][channels / 16][DK / 8][32 lanes][4].
uint64_t delta_saved_bytes(const ZenoDeltaRule& p) {
  const uint64_t chunks = (uint64_t(p.tokens) + kDeltaChunk - 1) / kDeltaChunk;
  const uint64_t rows = delta::key_width(p), channels = 16 * delta::value_warps(p);
  return chunks > 1 ? uint64_t(p.batch) * p.value_heads * (chunks - 1) * rows * channels * 4 : 0;
}

cudaError_t launch_delta_forward(const ZenoDeltaRule& p, cudaStream_t stream) {
  return p.dtype == ZENO_DTYPE_BF16 ? delta::by_type<__nv_bfloat16>(p, stream) : delta::by_type<float>(p, stream);
}

}  // namespace zb
