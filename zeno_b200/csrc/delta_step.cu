// Gated delta rule, recurrent form: the state of one (environment, head) stays in the
// registers of a few warps while they walk over its tokens.
//
//   S <- exp(g) S           (S <- 0 where an episode begins)
//   u  = beta (v - S^T k),  S <- S + k u^T,  o = scale S^T q
//
// A column of S (one value channel) never meets another, so a warp owns a group of
// columns and needs no other warp: lane (r, c) holds rows [16 r, 16 r + 16) of 4 adjacent
// columns, S^T k and S^T q are 16 products a lane and log2(RG) shuffles, and each state
// element is read once and written once.  For one token the time is that traffic.
#include <cuda_bf16.h>

#include "policy_ops.h"

namespace zb {
namespace {

template <class T>
__device__ __forceinline__ float to_f(T x) { return float(x); }
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T>
__device__ __forceinline__ T from_f(float x) { return T(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f(float x) { return __float2bfloat16_rn(x); }

constexpr int kStepWarps = 4;

// RG: row groups in a warp; 16 RG >= key_dim, and a warp holds 4 (32 / RG) columns.
// Four blocks an SM; the compiler by itself takes registers for three of some (4096 x 4 states of 128 x 128: 351 us
// against 391 in bfloat16, 376 against 423 in 32 bits).
template <int RG, class T, bool VEC>
__global__ void __launch_bounds__(kStepWarps * 32, 4)
delta_recurrent_kernel(const __grid_constant__ ZenoDeltaRule p, uint32_t slices, uint64_t jobs) {
  constexpr int DK = 16 * RG, CG = 32 / RG;
  __shared__ __align__(16) float sk[kStepWarps][DK], sq[kStepWarps][DK];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rg = lane / CG, cg = lane % CG;
  const uint64_t job = uint64_t(blockIdx.x) * kStepWarps + warp;
  if (job >= jobs) return;
  const uint32_t slice = uint32_t(job % slices);
  const uint64_t bh = job / slices;
  const uint32_t h = uint32_t(bh % p.value_heads);
  const uint64_t b = bh / p.value_heads;
  const uint32_t kh = h / (p.value_heads / p.key_heads);
  const int dk = int(p.key_dim), dv = int(p.value_dim);
  const int col = int(slice) * CG * 4 + cg * 4;
  const int cols = min(4, dv - col);  // may be <= 0

  const T* q = static_cast<const T*>(p.q.data) + int64_t(b) * p.q.stride[0] + int64_t(kh) * p.q.stride[2];
  const T* k = static_cast<const T*>(p.k.data) + int64_t(b) * p.k.stride[0] + int64_t(kh) * p.k.stride[2];
  const T* v = static_cast<const T*>(p.v.data) + int64_t(b) * p.v.stride[0] + int64_t(h) * p.v.stride[2];
  T* o = static_cast<T*>(p.out.data) + int64_t(b) * p.out.stride[0] + int64_t(h) * p.out.stride[2];
  const float* g = static_cast<const float*>(p.g.data) + int64_t(b) * p.g.stride[0] + int64_t(h) * p.g.stride[2];
  const float* be = static_cast<const float*>(p.beta.data) + int64_t(b) * p.beta.stride[0] + int64_t(h) * p.beta.stride[2];
  const uint8_t* rs = p.reset.data ? static_cast<const uint8_t*>(p.reset.data) + int64_t(b) * p.reset.stride[0] : nullptr;
  const int64_t state_at = int64_t(bh) * dk * dv;

  float s[16][4];
#pragma unroll
  for (int i = 0; i < 16; ++i)
#pragma unroll
    for (int c = 0; c < 4; ++c) s[i][c] = 0.0f;
  // a first token that clears the state needs no read of it
  const bool cleared = rs && rs[0];
  if (p.initial_state && !cleared) {
    const float* in = p.initial_state + state_at;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int r = rg * 16 + i;
      if (r < dk) {
        if (VEC) {
          if (cols > 0) {
            const float4 x = __ldcs(reinterpret_cast<const float4*>(in + int64_t(r) * dv + col));
            s[i][0] = x.x, s[i][1] = x.y, s[i][2] = x.z, s[i][3] = x.w;
          }
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (c < cols) s[i][c] = in[int64_t(r) * dv + col + c];
        }
      }
    }
  }
  for (uint32_t t = 0; t < p.tokens; ++t) {
    float nq = 0.0f, nk = 0.0f;
    __syncwarp();
    float xq[(DK + 31) / 32], xk[(DK + 31) / 32];
    bool big_q = false, big_k = false;
#pragma unroll
    for (int i = 0; i < (DK + 31) / 32; ++i) {
      const int r = i * 32 + lane;
      xq[i] = r < dk ? to_f(q[int64_t(t) * p.q.stride[1] + r]) : 0.0f;
      xk[i] = r < dk ? to_f(k[int64_t(t) * p.k.stride[1] + r]) : 0.0f;
      big_q |= fabsf(xq[i]) >= 0x1p60f, big_k |= fabsf(xk[i]) >= 0x1p60f;
    }
    // rows whose squares could leave 32 bits are normalised from a 2^80th of themselves
    const float lq = p.normalize && __any_sync(0xffffffffu, big_q) ? 0x1p-80f : 1.0f;
    const float lk = p.normalize && __any_sync(0xffffffffu, big_k) ? 0x1p-80f : 1.0f;
#pragma unroll
    for (int i = 0; i < (DK + 31) / 32; ++i) {
      const int r = i * 32 + lane;
      xq[i] *= lq, xk[i] *= lk;
      if (r < DK) sq[warp][r] = xq[i], sk[warp][r] = xk[i];
      nq = fmaf(xq[i], xq[i], nq), nk = fmaf(xk[i], xk[i], nk);
    }
    float fq = p.scale, fk = 1.0f;
    if (p.normalize) {
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) {
        nq += __shfl_xor_sync(0xffffffffu, nq, d);
        nk += __shfl_xor_sync(0xffffffffu, nk, d);
      }
      fq = p.scale / sqrtf(nq + kNormEps * lq * lq), fk = 1.0f / sqrtf(nk + kNormEps * lk * lk);
    }
    __syncwarp();
    const bool clear = rs && rs[int64_t(t) * p.reset.stride[1]];
    const float alpha = clear ? 0.0f : expf(g[int64_t(t) * p.g.stride[1]]);
    const float beta = be[int64_t(t) * p.beta.stride[1]];
    float kk[16], qq[16];
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const float4 x = *reinterpret_cast<const float4*>(&sk[warp][rg * 16 + i]);
      const float4 y = *reinterpret_cast<const float4*>(&sq[warp][rg * 16 + i]);
      kk[i] = x.x * fk, kk[i + 1] = x.y * fk, kk[i + 2] = x.z * fk, kk[i + 3] = x.w * fk;
      qq[i] = y.x * fq, qq[i + 1] = y.y * fq, qq[i + 2] = y.z * fq, qq[i + 3] = y.w * fq;
    }
    float u[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        s[i][c] = alpha == 0.0f ? 0.0f : s[i][c] * alpha;  // a cleared state is zero whatever it held
        u[c] = fmaf(s[i][c], kk[i], u[c]);
      }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
#pragma unroll
      for (int d = CG; d < 32; d <<= 1) u[c] += __shfl_xor_sync(0xffffffffu, u[c], d);
      const float x = c < cols ? to_f(v[int64_t(t) * p.v.stride[1] + col + c]) : 0.0f;
      u[c] = beta * (x - u[c]);
    }
    float y[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        s[i][c] = fmaf(kk[i], u[c], s[i][c]);
        y[c] = fmaf(s[i][c], qq[i], y[c]);
      }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
#pragma unroll
      for (int d = CG; d < 32; d <<= 1) y[c] += __shfl_xor_sync(0xffffffffu, y[c], d);
      if (rg == 0 && c < cols) o[int64_t(t) * p.out.stride[1] + col + c] = from_f<T>(y[c]);
    }
  }
  if (p.final_state) {
    float* out = p.final_state + state_at;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int r = rg * 16 + i;
      if (r < dk) {
        if (VEC) {
          if (cols > 0)
            __stcs(reinterpret_cast<float4*>(out + int64_t(r) * dv + col), make_float4(s[i][0], s[i][1], s[i][2], s[i][3]));
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (c < cols) out[int64_t(r) * dv + col + c] = s[i][c];
        }
      }
    }
  }
}

template <int RG, class T>
cudaError_t launch(const ZenoDeltaRule& p, cudaStream_t stream) {
  const uint32_t slices = (p.value_dim + 128 / RG - 1) / (128 / RG);
  const uint64_t jobs = uint64_t(p.batch) * p.value_heads * slices;
  const uint64_t blocks = (jobs + kStepWarps - 1) / kStepWarps;
  const bool vec = p.value_dim % 4 == 0 &&
                   ((reinterpret_cast<uintptr_t>(p.initial_state) | reinterpret_cast<uintptr_t>(p.final_state)) & 15) == 0;
  if (vec)
    delta_recurrent_kernel<RG, T, true><<<unsigned(blocks), kStepWarps * 32, 0, stream>>>(p, slices, jobs);
  else
    delta_recurrent_kernel<RG, T, false><<<unsigned(blocks), kStepWarps * 32, 0, stream>>>(p, slices, jobs);
  return cudaGetLastError();
}

template <class T>
cudaError_t by_rows(const ZenoDeltaRule& p, cudaStream_t stream) {
  if (p.key_dim <= 16) return launch<1, T>(p, stream);
  if (p.key_dim <= 32) return launch<2, T>(p, stream);
  if (p.key_dim <= 64) return launch<4, T>(p, stream);
  return launch<8, T>(p, stream);
}

}  // namespace

cudaError_t launch_delta_recurrent(const ZenoDeltaRule& p, cudaStream_t stream) {
  if (p.tokens == 0 && p.reset.data) {  // the kernel looks at the first token's flag before it walks: there is none
    ZenoDeltaRule q = p;
    q.reset.data = nullptr;
    return launch_delta_recurrent(q, stream);
  }
  return p.dtype == ZENO_DTYPE_BF16 ? by_rows<__nv_bfloat16>(p, stream) : by_rows<float>(p, stream);
}

}  // namespace zb
