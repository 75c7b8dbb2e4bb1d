// Which instance of the chunked linear attention serves a call, and how a rollout is cut into segments.
#pragma once
#include "linear_tensor.cuh"
#include "linear_warp.cuh"

namespace zb {
namespace linear {

inline int width_of(const ZenoLinearAttention& p) {
  const uint32_t w = p.key_dim > p.value_dim ? p.key_dim : p.value_dim;
  return w <= 32 ? 32 : w <= 64 ? 64 : 128;
}

// Chunks of 64 tokens in bfloat16 heads of more than 32 channels, so that what a chunk costs whatever its length (the state's limbs, its traffic in
// training) comes half as often (64 x 512 tokens, 4 heads of 48 x 56, with gradients: 178 us against 232); rollouts of up to 32
// tokens, heads of up to 32 channels (2048 x 128: 578 us against 644) and 32-bit calls (three limbs of everything in shared memory) take 32.
inline int chunk_of(const ZenoLinearAttention& p) { return p.dtype == ZENO_DTYPE_BF16 && p.tokens > 32 && width_of(p) > 32 ? 64 : 32; }

struct Cut {
  uint32_t count, chunks;  // segments, and chunks of each
  uint64_t state, keep, total;  // bytes
};
// How many segments: the least of the rounds of blocks that the main kernel takes, in chunks, and of what the segments cost besides: their sums,
// the walk over them, the start of a block.  The four weights are from bfloat16 heads of 128 channels (64 rollouts of 16 chunks are best in 2 segments, 322 us
// with gradients against 346 in 4; 16 of 64 chunks in 8) and serve all widths and both types, forward and backward, though a chunk's cost differs
// between them: only ratios to it count, and those of the others were not fitted.
inline Cut cut_of(const ZenoLinearAttention& p) {
  const uint32_t C = uint32_t(chunk_of(p)), chunks = (p.tokens + C - 1) / C;
  const uint64_t rows = uint64_t(p.batch) * p.value_heads;
  Cut c{1, chunks, 0, 0, 0};
  const uint64_t slots = kSms * (width_of(p) == 128 ? 1 : 2);
  if (rows == 0 || rows >= slots || chunks < 2) return c;
  float least = 0.0f;
  for (uint32_t want = 1; want <= chunks && want <= 256; ++want) {
    const uint32_t per = (chunks + want - 1) / want, count = (chunks + per - 1) / per;
    if (count != want) continue;
    float cost = float((rows * count + slots - 1) / slots) * (float(per) + 0.6f);
    if (count > 1) cost += 0.45f * float(per) * float((rows * (count - 1) + slots - 1) / slots) + 0.005f * float(rows * count) + 0.4f;
    if (count > 1 && cost >= least) continue;
    least = cost;
    c.count = count, c.chunks = per;
  }
  if (c.count == 1) return c;
  c.state = (rows * c.count * p.key_dim * p.value_dim * 4 + 15) / 16 * 16;
  c.keep = (rows * c.count * 4 + 15) / 16 * 16;
  c.total = c.state + c.keep;
  return c;
}

inline uint32_t vec_of(const ZenoTensor& t, uint32_t width, uint32_t dtype, uint32_t flag) {
  const int64_t n = dtype == ZENO_DTYPE_BF16 ? 8 : 4;
  const bool vec = width % 8 == 0 && reinterpret_cast<uintptr_t>(t.data) % 16 == 0 && t.stride[0] % n == 0 && t.stride[1] % n == 0 && t.stride[2] % n == 0;
  return vec ? flag : 0;
}
inline uint32_t vec_of(const ZenoLinearAttention& p, const ZenoTensor& out) {
  return vec_of(p.q, p.key_dim, p.dtype, kVecQ) | vec_of(p.k, p.key_dim, p.dtype, kVecK) | vec_of(p.v, p.value_dim, p.dtype, kVecV) |
         vec_of(out, p.value_dim, p.dtype, kVecOut);
}

// f(shape) of the call's instance, for one element type.  Heads of 128 channels are one block an SM: 16 warps for 32-bit calls (244 x 139 tokens, 2
// heads of 40 x 128, with gradients: 464 us against 530 with 8; 2183 x 4, 128 x 64: 393 against 421) and where widths are not whole (bfloat16, 777 x 20, 4 heads
// of 100 x 128, backward: 356 against 393); 8 for whole bfloat16 ones (1024 x 32, 4 of 128 x 128: 458 against 472).
template <class T, bool FULL, class F>
cudaError_t with_shape_of(const ZenoLinearAttention& p, int w, F&& f) {
  if constexpr (sizeof(T) == 2) {
    if (chunk_of(p) == 32) {
      if (w == 32) return f(Shape<T, 32, 32, 4, FULL>{});
      if (w == 64) return f(Shape<T, 64, 32, 4, FULL>{});
      return f(Shape<T, 128, 32, FULL ? 8 : 16, FULL>{});
    }
    if (w == 64) return f(Shape<T, 64, 64, 8, FULL>{});
    return f(Shape<T, 128, 64, 16, FULL>{});
  } else {
    if (w == 32) return f(Shape<T, 32, 32, 4, FULL>{});
    if (w == 64) return f(Shape<T, 64, 32, 8, FULL>{});
    return f(Shape<T, 128, 32, 16, FULL>{});
  }
}
inline bool full_width(const ZenoLinearAttention& p) { return int(p.key_dim) == width_of(p) && int(p.value_dim) == width_of(p); }
template <class T, class F>
cudaError_t with_shape(const ZenoLinearAttention& p, F&& f) {
  return full_width(p) ? with_shape_of<T, true>(p, width_of(p), f) : with_shape_of<T, false>(p, width_of(p), f);
}

// Short rollouts of many environments: a warp a head.  Few of them finish earlier with a block each.
inline bool warp_a_head(const ZenoLinearAttention& p) {
  return p.dtype == ZENO_DTYPE_BF16 && p.tokens >= 1 && p.tokens <= 32 && uint64_t(p.batch) * p.value_heads >= 4 * kSms;
}
template <class F>
cudaError_t with_warp_shape(const ZenoLinearAttention& p, F&& f) {
  const int w = width_of(p);
  const bool full = full_width(p);
  if (w == 32) return full ? f(WarpShape<32>{}, std::true_type{}) : f(WarpShape<32>{}, std::false_type{});
  if (w == 64) return full ? f(WarpShape<64>{}, std::true_type{}) : f(WarpShape<64>{}, std::false_type{});
  return full ? f(WarpShape<128>{}, std::true_type{}) : f(WarpShape<128>{}, std::false_type{});
}

template <class T>
cudaError_t forward(const ZenoLinearAttention& p, void* workspace, cudaStream_t stream);
template <class T>
cudaError_t backward(const ZenoLinearAttention& p, const ZenoLinearAttentionGrads& d, void* workspace, cudaStream_t stream);

// A main kernel, which may start while a walk over segments is under way.
template <class... Params, class... Args>
cudaError_t launch_main(void (*kernel)(Params...), dim3 grid, int threads, int smem, bool after_walk, cudaStream_t stream, Args... args) {
  if (after_walk) return launch_early(kernel, grid, threads, smem, stream, args...);
  kernel<<<grid, threads, smem, stream>>>(args...);
  return cudaGetLastError();
}

// What each segment adds, then the states in front of (behind) them.
// Wide heads in chunks of 64: on tcgen05.
template <class S>
constexpr bool kTensor = sizeof(typename S::T) == 2 && S::D == tensor::D && S::C == tensor::C;

template <class Full>
cudaError_t cut_states(const ZenoLinearAttention& p, const ZenoTensor& x, const ZenoTensor& y, const Segments& sg, const float* initial, bool reverse,
                       cudaStream_t stream) {
  const uint32_t rows = p.batch * p.value_heads;
  static std::atomic<uint64_t> devices{0};
  cudaError_t e;
  if constexpr (kTensor<Full>) {
    using S = tensor::SegmentShape<Full::FULL>;
    auto kernel = tensor::linear_tensor_segment_kernel<S>;
    e = allow_smem(kernel, tensor::kSegmentBytes, devices);
    if (e != cudaSuccess) return e;
    kernel<<<grid_of(p, sg.count - 1), S::THREADS, tensor::kSegmentBytes, stream>>>(p, x, y, sg, reverse, linear_patience());
  } else {
    constexpr int BLOCKS = 512 / Full::THREADS;
    auto kernel = linear_segment_kernel<Full, BLOCKS>;
    const int bytes = ForwardSmem<Full>::gates + 2 * 2 * Full::L * Full::PLANE;
    e = allow_smem(kernel, bytes, devices);
    if (e != cudaSuccess) return e;
    kernel<<<grid_of(p, sg.count - 1), Full::THREADS, bytes, stream>>>(p, x, y, sg, reverse);
  }
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  return launch_linear_walk(LinearWalk{sg.state, sg.keep, initial, sg.count, p.key_dim * p.value_dim, reverse}, rows, stream);
}

}  // namespace linear
}  // namespace zb
