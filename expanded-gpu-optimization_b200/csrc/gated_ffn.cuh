// The feed-forward block's path for a few tokens (gated_ffn_small.cu).
#pragma once

#include "blocks.cuh"

namespace fhb {

// Calls without gradients of up to so many tokens take it: as many as it is faster for than the
// tensor-core products (1024 x 4096, us with either: bf16 13.3 and 16.2 for two tokens, 17.0 and
// 16.2 for four; fp32, whose weights the products have to split first, 30 and 50 for eight).
constexpr int64_t ffn_small_tokens(int dtype) { return dtype == FHB_DTYPE_F32 ? 8 : 2; }
// Bytes of h, its workspace.
size_t ffn_small_bytes(const fhb_ffn_problem& p);
cudaError_t launch_ffn_small(const fhb_ffn_problem& p, void* y, void* h, const DeviceInfo& dev,
                             cudaStream_t stream);

}  // namespace fhb
