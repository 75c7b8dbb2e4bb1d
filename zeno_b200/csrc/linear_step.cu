// Linear attention with decays, recurrent form, one token:
//   S <- exp(g) S + k v^T  (without the first term where an episode begins),  o = scale S^T q
// The time is the state's bytes, once in and once out.  A warp takes a slice of value channels of one (environment, head):
// lane (r, c) has 4 neighbouring channels c of the rows r, r + RG, ...; the rows of a slice are whole 16-byte
// vectors side by side, eight of them under way at once, and nothing but S^T q crosses lanes.
// 16384 environments of 4 heads of 64 x 64, bfloat16: 336 us, 6.4 TB/s.  One environment: 3 us, the latency of
// two loads one behind the other (k and q, then up to 64 rows of the state at once).  777 environments, 3 heads of 40 x 56 on one key head, 32-bit: 10.6 us (6.6 us of
// bytes); four slices of 16 channels a state, of which the last is half empty, and each fetches its own k and q.
#include <cuda_bf16.h>

#include "policy_ops.h"

namespace zb {
namespace {

constexpr int kWarps = 4;
constexpr int kBatch = 8;  // vectors of a lane under way

__device__ __forceinline__ float up(float x) { return x; }
__device__ __forceinline__ float up(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void down(float* to, float x) { *to = x; }
__device__ __forceinline__ void down(__nv_bfloat16* to, float x) { *to = __float2bfloat16_rn(x); }

// CG: lanes over a slice's channels.
template <int CG, class T, bool VEC>
__global__ void __launch_bounds__(kWarps * 32) linear_step_kernel(const __grid_constant__ ZenoLinearAttention p, const uint32_t slices,
                                                                  const uint64_t jobs) {
  constexpr int RG = 32 / CG;
  __shared__ float2 kq[kWarps][kDeltaMaxDim];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rg = lane / CG, cg = lane % CG;
  const uint64_t job = uint64_t(blockIdx.x) * kWarps + warp;
  if (job >= jobs) return;
  const uint64_t row = job / slices;
  const uint32_t h = uint32_t(row % p.value_heads);
  const int64_t b = int64_t(row / p.value_heads);
  const uint32_t kh = h / (p.value_heads / p.key_heads);
  const int dk = int(p.key_dim), dv = int(p.value_dim);
  const int col = int(job % slices) * CG * 4 + cg * 4;
  const int cols = min(4, dv - col);  // may be <= 0

  const uint8_t* rs = static_cast<const uint8_t*>(p.reset.data);
  const float g = static_cast<const float*>(p.g.data)[b * p.g.stride[0] + int64_t(h) * p.g.stride[2]];
  const float alpha = rs && rs[b * p.reset.stride[0]] ? 0.0f : expf(g);
  const T* q = static_cast<const T*>(p.q.data) + b * p.q.stride[0] + int64_t(kh) * p.q.stride[2];
  const T* k = static_cast<const T*>(p.k.data) + b * p.k.stride[0] + int64_t(kh) * p.k.stride[2];
  const T* v = static_cast<const T*>(p.v.data) + b * p.v.stride[0] + int64_t(h) * p.v.stride[2] + col;
  T* o = static_cast<T*>(p.out.data) + b * p.out.stride[0] + int64_t(h) * p.out.stride[2] + col;
  const int64_t at = int64_t(row) * dk * dv + col;
  // a state that is dropped is not read
  const float* in = p.initial_state && alpha != 0.0f ? p.initial_state + at : nullptr;
  float* out = p.final_state ? p.final_state + at : nullptr;

  for (int i = lane; i < dk; i += 32) kq[warp][i] = make_float2(up(k[i]), up(q[i]) * p.scale);
  float x[4], y[4] = {0, 0, 0, 0};
#pragma unroll
  for (int c = 0; c < 4; ++c) x[c] = c < cols ? up(v[c]) : 0.0f;
  __syncwarp();
#pragma unroll 1
  for (int first = 0; first < dk; first += RG * kBatch) {
    float4 s[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int r = first + u * RG + rg;
      s[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (in && r < dk && cols > 0) {
        const float* from = in + int64_t(r) * dv;
        if (VEC) {
          s[u] = __ldcs(reinterpret_cast<const float4*>(from));
        } else {
          s[u].x = from[0];
          if (cols > 1) s[u].y = from[1];
          if (cols > 2) s[u].z = from[2];
          if (cols > 3) s[u].w = from[3];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int r = first + u * RG + rg;
      if (r >= dk) break;
      const float2 f = kq[warp][r];
      s[u].x = fmaf(alpha, s[u].x, f.x * x[0]), s[u].y = fmaf(alpha, s[u].y, f.x * x[1]);
      s[u].z = fmaf(alpha, s[u].z, f.x * x[2]), s[u].w = fmaf(alpha, s[u].w, f.x * x[3]);
      y[0] = fmaf(s[u].x, f.y, y[0]), y[1] = fmaf(s[u].y, f.y, y[1]);
      y[2] = fmaf(s[u].z, f.y, y[2]), y[3] = fmaf(s[u].w, f.y, y[3]);
      if (out && cols > 0) {
        float* to = out + int64_t(r) * dv;
        if (VEC) {
          __stcs(reinterpret_cast<float4*>(to), s[u]);
        } else {
          to[0] = s[u].x;
          if (cols > 1) to[1] = s[u].y;
          if (cols > 2) to[2] = s[u].z;
          if (cols > 3) to[3] = s[u].w;
        }
      }
    }
  }
#pragma unroll
  for (int c = 0; c < 4; ++c) {
#pragma unroll
    for (int d = CG; d < 32; d <<= 1) y[c] += __shfl_xor_sync(0xffffffffu, y[c], d);
    if (rg == 0 && c < cols) down(o + c, y[c]);
  }
}

template <int CG, class T>
cudaError_t launch(const ZenoLinearAttention& p, cudaStream_t stream) {
  const uint32_t slices = (p.value_dim + 4 * CG - 1) / (4 * CG);
  const uint64_t jobs = uint64_t(p.batch) * p.value_heads * slices;
  const unsigned blocks = unsigned((jobs + kWarps - 1) / kWarps);
  const bool vec = p.value_dim % 4 == 0 &&
                   ((reinterpret_cast<uintptr_t>(p.initial_state) | reinterpret_cast<uintptr_t>(p.final_state)) & 15) == 0;
  if (vec) linear_step_kernel<CG, T, true><<<blocks, kWarps * 32, 0, stream>>>(p, slices, jobs);
  else linear_step_kernel<CG, T, false><<<blocks, kWarps * 32, 0, stream>>>(p, slices, jobs);
  return cudaGetLastError();
}

template <class T>
cudaError_t by_columns(const ZenoLinearAttention& p, cudaStream_t stream) {
  // Few states: slices of 16 channels, all of a lane's rows under way at once.  Many: rows of 64 channels and more together.
  if (uint64_t(p.batch) * p.value_heads < 16 * kSms || p.value_dim <= 16) return launch<4, T>(p, stream);
  if (p.value_dim <= 32) return launch<8, T>(p, stream);
  return launch<16, T>(p, stream);
}

}  // namespace

cudaError_t launch_linear_step(const ZenoLinearAttention& p, cudaStream_t stream) {
  return p.dtype == ZENO_DTYPE_BF16 ? by_columns<__nv_bfloat16>(p, stream) : by_columns<float>(p, stream);
}

}  // namespace zb
