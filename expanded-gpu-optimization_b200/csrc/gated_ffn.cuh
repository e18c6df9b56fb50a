// The feed-forward block's path for a few tokens (gated_ffn_small.cu).
#pragma once

#include "blocks.cuh"

namespace fhb {

// Whether a call without gradients takes it: where it is faster than the tensor-core products. FP32,
// whose weights the products have to split first: up to 8 tokens at any size (us, dots and products:
// 64 x 256 5.8 and 13.5, 1024 x 4096 30 and 51, 4096 x 11,008 229 and 421 for eight tokens; 102 and 417
// for one). bf16: up to 2 tokens, while tokens times weights are at most 72 Mi, since the dot products'
// rate falls with the tokens (one token 1024 x 4096 11.3 and 17.0, 2048 x 5632 21.9 and 25.3, 4096 x
// 11,008 61.9 and 55.2; two 13.4 and 17.2, 24.8 and 25.5, 72.2 and 56.3; four 17.0 and 16.2 at 1024 x 4096).
constexpr bool ffn_takes_small(const fhb_ffn_problem& p) {
  return p.dtype == FHB_DTYPE_F32
             ? p.tokens <= 8
             : p.tokens <= 2 && p.tokens * p.hidden * (2 * p.width + p.out_width) <= 72ll << 20;
}
// Bytes of h, its workspace.
size_t ffn_small_bytes(const fhb_ffn_problem& p);
cudaError_t launch_ffn_small(const fhb_ffn_problem& p, void* y, void* h, const DeviceInfo& dev,
                             cudaStream_t stream);

}  // namespace fhb
