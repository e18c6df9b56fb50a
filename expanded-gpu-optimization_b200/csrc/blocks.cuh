// Shared pieces of the gated residual trunk's kernels (feed-forward block, norms, AdamW):
// element types, and the launchers between the kernel files and the C ABI (capi_blocks.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/fused_hoad_b200.h"
#include "kernels.cuh"

namespace fhb {

using bf16 = __nv_bfloat16;

inline size_t dtype_bytes(int dtype) { return dtype == FHB_DTYPE_F32 ? 4 : 2; }

#ifdef __CUDACC__
__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(bf16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) {
  return x;
}
template <>
__device__ __forceinline__ bf16 from_float<bf16>(float x) {
  return __float2bfloat16_rn(x);
}

// The block's activation a and its derivative at g, on the special-function unit (ex2, rcp).
// silu: a = g s, a' = s (1 + g (1 - s)), s = 1 / (1 + e^-g). tanh: with r = 1 / (1 + e^2|g|) <= 1/2,
// |a| = 1 - 2 r and a' = 4 r (1 - r), which cancel nowhere on either side (with e^2g, r would go to 1
// for negative g, and 1 - r lose all its digits by g = -9); below 1/4, where 1 - 2 r loses digits, the
// Taylor series (next term below 2^-26 of a). An exponential e^x is off by about 1.5 |x| 2^-24, the
// rounding of its exponent, and a few ulp: so are the tails of a and a'.
__device__ __forceinline__ float reciprocal_of_one_plus_exp2(float x) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(e + 1.0f));
  return r;
}
template <bool Tanh>
__device__ __forceinline__ void block_activation(float g, float& a, float& slope) {
  if (Tanh) {
    const float r = reciprocal_of_one_plus_exp2(fabsf(g) * 2.8853900817779268f);  // 2 / ln 2
    const float q = g * g;
    float t = fmaf(q, 62.0f / 2835.0f, -17.0f / 315.0f);
    t = fmaf(q, t, 2.0f / 15.0f);
    t = fmaf(q, t, -1.0f / 3.0f);
    t = fmaf(g * q, t, g);
    a = fabsf(g) < 0.25f ? t : copysignf(fmaf(-2.0f, r, 1.0f), g);
    slope = 4.0f * r * (1.0f - r);
  } else {
    const float s = reciprocal_of_one_plus_exp2(g * -1.4426950408889634f);  // 1 / ln 2
    a = g * s;
    slope = fmaf(a, 1.0f - s, s);
  }
}
#endif

// ---- gated_ffn.cu ----
size_t ffn_saved_bytes(const fhb_ffn_problem& p);
size_t ffn_workspace_bytes(const fhb_ffn_problem& p, int pass, const DeviceInfo& dev);  // FHB_FFN_*
cudaError_t launch_ffn_forward(const fhb_ffn_problem& p, void* y, void* saved, void* workspace,
                               const DeviceInfo& dev, cudaStream_t stream);
cudaError_t launch_ffn_backward(const fhb_ffn_problem& p, const void* grad_y, int64_t grad_y_stride,
                                const void* saved, const fhb_ffn_grads& grads, void* workspace,
                                const DeviceInfo& dev, cudaStream_t stream);

// ---- residual_norm.cu ----
cudaError_t launch_residual_norm(const fhb_norm_problem& p, void* total, void* normed,
                                 float* stats, const DeviceInfo& dev, cudaStream_t stream);
cudaError_t launch_staged_wait_selftest(const float* rows, float* out, const DeviceInfo& dev,
                                        cudaStream_t stream);
size_t residual_norm_workspace_bytes(const fhb_norm_problem& p, const DeviceInfo& dev);
cudaError_t launch_residual_norm_backward(const fhb_norm_problem& p, const void* grad_total,
                                          int64_t grad_total_stride, const void* grad_normed,
                                          int64_t grad_normed_stride, const float* stats,
                                          const fhb_norm_grads& grads, void* workspace,
                                          const DeviceInfo& dev, cudaStream_t stream);

// ---- adamw.cu ----
cudaError_t launch_adamw(const fhb_adamw_tensor* tensors, int64_t n_tensors, int state_bits,
                         int64_t* step, double lr, double beta1, double beta2, double eps,
                         double weight_decay, const DeviceInfo& dev, cudaStream_t stream);

}  // namespace fhb
