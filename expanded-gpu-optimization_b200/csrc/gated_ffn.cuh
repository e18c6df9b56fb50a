// The feed-forward block's path for a few tokens (gated_ffn_small.cu).
#pragma once

#include "blocks.cuh"

namespace fhb {

// Calls without gradients of up to so many tokens take it.
constexpr int kFfnSmallTokens = 8;
// Bytes of h, its workspace.
size_t ffn_small_bytes(const fhb_ffn_problem& p);
cudaError_t launch_ffn_small(const fhb_ffn_problem& p, void* y, void* h, const DeviceInfo& dev,
                             cudaStream_t stream);

}  // namespace fhb
