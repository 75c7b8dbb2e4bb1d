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
//
// Few long rollouts.  A stretch of tokens takes the state in front of it to M S + N.  Where the
// environments and heads alone do not fill the GPU, the tokens are cut into segments; one launch
// runs every segment from the identity with V = 0 (its M) and from zero (its N), one walks over the
// segments' states, and one runs all segments again, each from its own state, for the outputs:
// about 2.5 times the work on the SMs that would have stood idle.
#include "delta_mma.cuh"

namespace zb {
namespace delta {
namespace {

enum Mode { kWhole, kTransitions, kOutputs };
struct Split {
  Mode mode;
  uint32_t segments, chunks;  // chunks of a segment
  float* m;        // [batch * heads][segments][dk][dk]
  bool m_transposed;
  float* n;        // ... [dk][dv]: what a segment leaves of nothing (the first one: of initial_state)
  float* state;    // ... [dk][dv]: the state in front of a segment
  int* cleared;    // ... whether the segment drops the state in front of it
  uint32_t value_blocks;  // kTransitions: blocks of N in the grid's second dimension, those of M behind them
};

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
// Threads of an SM: 512 where the state is 32 registers a thread (4096 x 32 tokens, 64 x 64, when first measured: 461 us against 544 with
// 384 and 714 with 256), 384 where it is 64 (2 x 4096 tokens, 128 x 128: 1250 us against 1405 with 512).
__global__ void __launch_bounds__(NW * 32, (DK <= 64 ? 512 : 384) / (NW * 32)) delta_forward_kernel(const __grid_constant__ ZenoDeltaRule p, const __grid_constant__ Split sp) {
  extern __shared__ __align__(16) unsigned char raw[];
  using Smem = ForwardSmem<DK, NW, T>;
  constexpr int L = In<T>::limbs;
  Smem& sm = *reinterpret_cast<Smem*>(raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int qj = (lane & 3) * 2;
  const uint32_t h = blockIdx.x % p.value_heads, b = blockIdx.x / p.value_heads;
  const int dk = int(p.key_dim);
  const uint32_t segment = blockIdx.z;
  const bool outputs = sp.mode != kTransitions, is_m = !outputs && blockIdx.y >= sp.value_blocks;
  if (is_m && segment == 0) return;
  const int dv = is_m ? dk : int(p.value_dim);  // columns of this block's state
  const int v0 = int(blockIdx.y - (is_m ? sp.value_blocks : 0)) * 16 * NW;
  const int c0 = v0 + warp * 16;  // the warp's first channel
  const Rows<T> rows = rows_of<T>(p, b, h);
  T* out = static_cast<T*>(p.out.data) + int64_t(b) * p.out.stride[0] + int64_t(h) * p.out.stride[2];
  const bool pairs_ok = sizeof(T) == 2 && dv % 2 == 0 && reinterpret_cast<uintptr_t>(p.out.data) % 4 == 0 &&
                        ((p.out.stride[0] | p.out.stride[1] | p.out.stride[2]) & 1) == 0;
  const int64_t state_size = int64_t(dk) * dv, row_at = int64_t(blockIdx.x) * state_size;
  const int64_t segment_at = (int64_t(blockIdx.x) * sp.segments + segment) * state_size;
  const float* initial = sp.mode == kOutputs                                     ? sp.state + segment_at
                         : p.initial_state && !is_m && segment == 0 ? p.initial_state + row_at
                                                                    : nullptr;
  float* final_state = sp.mode == kTransitions     ? (is_m ? sp.m : sp.n) + segment_at
                       : p.final_state && segment + 1 == sp.segments ? p.final_state + row_at
                                                                     : nullptr;

  float st[DK / 8][4] = {};
  if (initial) {
    for_state<DK>(st, dk, dv, c0, lane, [&](float& x, int64_t at) { x = initial[at]; });
  } else if (is_m) {
    const int gi = lane >> 2;
#pragma unroll
    for (int n = 0; n < DK / 8; ++n)
#pragma unroll
      for (int x = 0; x < 4; ++x) st[n][x] = c0 + gi + (x >> 1) * 8 == n * 8 + qj + (x & 1) ? 1.0f : 0.0f;
  }
  bool has_state = initial || is_m;  // there is a state in front of the chunk
  bool cleared = false;              // (M) some token has dropped it
  if (tid == 0) sm.gates.bad = 0, sm.gates.state_bad = 0;
  __syncthreads();

  const int64_t T_ = p.tokens;
  const int64_t chunks = (T_ + C - 1) / C;
  const int64_t last = min(chunks, (int64_t(segment) + 1) * sp.chunks);
  for (int64_t chunk = int64_t(segment) * sp.chunks; chunk < last; ++chunk) {
    const int64_t t0 = chunk * C, t1 = min(t0 + C, T_);
    if (p.saved && outputs && chunk > 0) {
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
        load_rows<DK, NW, T, false>(sm.gates, p, rows, sm.q[0], sm.k[0], sm.v, v0, is_m ? 0 : dv, t0, lo, hi, tid);
        if (warp == 0) scan_gates(sm.gates, gates, lane);
        __syncthreads();
        if (sm.gates.bad && p.normalize) {
          mend_norms<NW, T>(sm.gates, p, rows, t0, lo, hi, tid);
          __syncthreads();
        }
        // A value that is not finite must not reach another episode, nor an earlier token,
        // through a product with zero: such a chunk is taken token by token.
        if (hi - lo == 1 || !(sm.gates.bad || (sm.gates.state_bad && sm.gates.marks != 0))) break;
        hi = lo + 1;
        __syncthreads();
      }
      const int halves = hi - t0 <= 16 ? 1 : 2;
      if (t1 < T_) prefetch_rows<NW>(p, rows, t1, v0, tid);
      pair_matrices<DK, NW, L, false>(sm.gates, sm.pairs, sm.squares, nullptr, sm.q[0], sm.k[0], outputs, halves, warp, lane);
      cleared |= sm.gates.marks != 0;
      __syncthreads();

      // E^T = V^T - a (S0^T K^T), O^T = a (S0^T Q^T)
      float e[4][4] = {}, o[4][4] = {};
      if (has_state) {
        const float s0 = pow2_scale(e0), s1 = pow2_scale(e1);
#pragma unroll
        for (int kk = 0; kk < DK; kk += 16) {
          uint32_t ah[4], al[4];
          split_a(ah, al, st[kk / 8], st[kk / 8 + 1], s0, s1);
          state_times_rows<DK, L>(e, ah, al, sm.k[0], kk, halves, lane);
          if (outputs) state_times_rows<DK, L>(o, ah, al, sm.q[0], kk, halves, lane);
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
      solve_forward(e, sm.pairs, halves, lane);  // now W^T
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const float2 be = *reinterpret_cast<const float2*>(&sm.gates.beta[n * 8 + qj]);
#pragma unroll
        for (int x = 0; x < 4; ++x) e[n][x] *= x & 1 ? be.y : be.x;  // U^T
      }
      if (outputs) {  // O^T += U^T P^T
        row_exps<4>(e, e0, e1);
        const float s0 = pow2_scale(e0), s1 = pow2_scale(e1), g0 = pow2_unscale(e0), g1 = pow2_unscale(e1);
        uint32_t uh[2][4], ul[2][4];
#pragma unroll
        for (int r = 0; r < 2; ++r) split_a(uh[r], ul[r], e[2 * r], e[2 * r + 1], s0, s1);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (i == 1 && halves == 1) break;
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
      if (outputs) store_out(o, out, p.out.stride[1], t0, lo, hi, c0, dv, pairs_ok, lane);
      // S^T <- a_C S^T + (D_C U)^T K
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const float2 zk = *reinterpret_cast<const float2*>(&sm.gates.zk[n * 8 + qj]);
#pragma unroll
        for (int x = 0; x < 4; ++x) e[n][x] *= x & 1 ? zk.y : zk.x;
      }
      state_update<DK, L>(st, sm.gates.keep, e, sm.k[0], halves, lane);
      has_state = true;
      __syncthreads();
      if (tid == 0) sm.gates.bad = 0, sm.gates.state_bad = 0;
      __syncthreads();
      lo = hi;
    }
  }
  if (final_state && is_m && sp.m_transposed)
    for_state<DK>(st, dk, dv, c0, lane, [&](float& x, int64_t at) { final_state[int(at) % dk * dk + int(at) / dk] = x; });
  else if (final_state)
    for_state<DK>(st, dk, dv, c0, lane, [&](float& x, int64_t at) { final_state[at] = x; });
  if (is_m && v0 == 0 && tid == 0) sp.cleared[int64_t(blockIdx.x) * sp.segments + segment] = cleared;
}

// Segments of a call: enough to give every SM three blocks of 128 threads, each of at least 4 chunks;
// 1 (not split) below 4 of them.  (2 environments x 8 heads of 128 x 128, 4096 tokens: 375 us in 13 segments, 963 whole.)
inline uint32_t segments_of(const ZenoDeltaRule& p) {
  const uint64_t chunks = (uint64_t(p.tokens) + C - 1) / C;
  const int groups = value_groups(p), warps = groups < 4 ? groups : 4;
  const uint64_t blocks = uint64_t(p.batch) * p.value_heads * (groups / warps);
  uint64_t n = blocks ? uint64_t(kSms) * 12 / (blocks * warps) : 1;
  if (n > chunks / 4) n = chunks / 4;
  return n < 4 ? 1 : uint32_t(n);
}

template <int DK, int NW, class T>
cudaError_t launch(const ZenoDeltaRule& p, const Split& sp, dim3 grid, cudaStream_t stream) {
  const auto kernel = delta_forward_kernel<DK, NW, T>;
  constexpr int smem = int(sizeof(ForwardSmem<DK, NW, T>));
  static std::atomic<uint64_t> allowed{0};
  const cudaError_t e = allow_smem(kernel, smem, allowed);
  if (e != cudaSuccess) return e;
  kernel<<<grid, NW * 32, smem, stream>>>(p, sp);
  return cudaGetLastError();
}

template <int DK, int NW, class T>
cudaError_t launch(const ZenoDeltaRule& p, void* workspace, cudaStream_t stream) {
  const uint32_t rows = p.batch * p.value_heads, segments = segments_of(p), blocks = uint32_t(value_groups(p) / NW);
  Split sp{};
  sp.segments = 1, sp.chunks = (p.tokens + C - 1) / C;
  if (segments == 1) return launch<DK, NW, T>(p, sp, dim3(rows, blocks), stream);
  const DeltaSplitLayout lay(p, segments);
  char* at = static_cast<char*>(workspace);
  sp.m = reinterpret_cast<float*>(at), sp.n = reinterpret_cast<float*>(at + lay.m), sp.state = reinterpret_cast<float*>(at + lay.m + lay.n);
  sp.cleared = reinterpret_cast<int*>(at + lay.m + 2 * lay.n);
  sp.mode = kTransitions, sp.chunks = (sp.chunks + segments - 1) / segments;
  sp.segments = ((p.tokens + C - 1) / C + sp.chunks - 1) / sp.chunks;  // none of them empty
  sp.value_blocks = blocks, sp.m_transposed = true;
  // nothing is asked of the last segment's transition
  cudaError_t e = launch<DK, NW, T>(p, sp, dim3(rows, blocks + (DK + 16 * NW - 1) / (16 * NW), sp.segments - 1), stream);
  if (e != cudaSuccess) return e;
  e = launch_delta_walk(DeltaWalk{sp.m, sp.n, sp.state, sp.cleared, p.initial_state, sp.segments, p.key_dim, p.value_dim, false}, rows, stream);
  if (e != cudaSuccess) return e;
  sp.mode = kOutputs;
  return launch<DK, NW, T>(p, sp, dim3(rows, blocks, sp.segments), stream);
}

template <int DK, class T>
cudaError_t by_width(const ZenoDeltaRule& p, void* workspace, cudaStream_t stream) {
  const int groups = value_groups(p);
  switch (groups == 8 && segments_of(p) > 1 ? 4 : groups) {
    case 2:
      if constexpr (DK < 128) return launch<DK, 2, T>(p, workspace, stream);
    case 4: return launch<DK, 4, T>(p, workspace, stream);
    default: return launch<DK, 8, T>(p, workspace, stream);
  }
}

// The M of the segments of a backward pass.
template <int DK, class T>
cudaError_t transitions(const ZenoDeltaRule& p, const Split& sp, cudaStream_t stream) {
  constexpr int NW = DK == 32 ? 2 : 4;
  return launch<DK, NW, T>(p, sp, dim3(p.batch * p.value_heads, (DK + 16 * NW - 1) / (16 * NW), sp.segments - 1), stream);
}
template <class T>
cudaError_t transitions_by_width(const ZenoDeltaRule& p, const Split& sp, cudaStream_t stream) {
  switch (key_width(p)) {
    case 32: return transitions<32, T>(p, sp, stream);
    case 64: return transitions<64, T>(p, sp, stream);
    default: return transitions<128, T>(p, sp, stream);
  }
}

template <class T>
cudaError_t by_type(const ZenoDeltaRule& p, void* workspace, cudaStream_t stream) {
  switch (key_width(p)) {
    case 32: return by_width<32, T>(p, workspace, stream);
    case 64: return by_width<64, T>(p, workspace, stream);
    default: return by_width<128, T>(p, workspace, stream);
  }
}

}  // namespace
}  // namespace delta

// The states in front of every chunk but the first (that one is initial_state), in the
// accumulators' order: [batch * heads][chunks - 1][channels / 16][DK / 8][32 lanes][4].
uint64_t delta_saved_bytes(const ZenoDeltaRule& p) {
  const uint64_t chunks = (uint64_t(p.tokens) + kDeltaChunk - 1) / kDeltaChunk;
  const uint64_t rows = delta::key_width(p), channels = 16 * delta::value_groups(p);
  return chunks > 1 ? uint64_t(p.batch) * p.value_heads * (chunks - 1) * rows * channels * 4 : 0;
}

cudaError_t launch_delta_transitions(const ZenoDeltaRule& p, float* m, int* cleared, uint32_t segments, uint32_t chunks,
                                     cudaStream_t stream) {
  delta::Split sp{};
  sp.mode = delta::kTransitions, sp.segments = segments, sp.chunks = chunks, sp.m = m, sp.cleared = cleared;
  ZenoDeltaRule q = p;
  q.saved = nullptr;
  return p.dtype == ZENO_DTYPE_BF16 ? delta::transitions_by_width<__nv_bfloat16>(q, sp, stream)
                                    : delta::transitions_by_width<float>(q, sp, stream);
}

uint64_t delta_forward_workspace(const ZenoDeltaRule& p) {
  const uint32_t segments = delta::segments_of(p);
  return segments == 1 ? 0 : DeltaSplitLayout(p, segments).total;
}

cudaError_t launch_delta_forward(const ZenoDeltaRule& p, void* workspace, cudaStream_t stream) {
  return p.dtype == ZENO_DTYPE_BF16 ? delta::by_type<__nv_bfloat16>(p, workspace, stream) : delta::by_type<float>(p, workspace, stream);
}

}  // namespace zb
