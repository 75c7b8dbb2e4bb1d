// Launchers of the policy operators (gated delta rule, Newton-Schulz orthogonalisation),
// shared by the kernels' files and the C entries in policy_ops.cpp.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/zeno.h"

namespace zb {

constexpr int kDeltaMaxDim = 128;  // largest key or value width of a head
constexpr int kDeltaChunk = 32;    // tokens of one chunk (one lane each in the gate scan)
constexpr float kNormEps = 1e-6f;  // under the root of the norms of q and k

uint64_t delta_saved_bytes(const ZenoDeltaRule& p);
uint64_t delta_backward_workspace(const ZenoDeltaRule& p);
cudaError_t launch_delta_recurrent(const ZenoDeltaRule& p, cudaStream_t stream);
cudaError_t launch_delta_forward(const ZenoDeltaRule& p, cudaStream_t stream);
cudaError_t launch_delta_backward(const ZenoDeltaRule& p, const ZenoDeltaRuleGrads& d, void* workspace, cudaStream_t stream);

uint64_t orthogonalize_workspace(uint32_t count, uint32_t rows, uint32_t cols, uint32_t dtype);
cudaError_t launch_orthogonalize(const void* update, const int64_t* strides, void* out, uint32_t count, uint32_t rows, uint32_t cols,
                                 uint32_t dtype, uint32_t steps, void* workspace, cudaStream_t stream);

}  // namespace zb
