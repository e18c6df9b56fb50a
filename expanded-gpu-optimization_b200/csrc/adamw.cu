// One AdamW step over many tensors, moments in FP32 or in 8 bits (e4m3 codes of m and sqrt(v)
// with one scale per block of 256 values). The arithmetic on the moments is the formula's,
// operation by operation (no contraction into fused multiply-adds), so the moments and codes
// are those of the same formula in any IEEE FP32 arithmetic.
#include <cuda_fp8.h>

#include <algorithm>

#include "blocks.cuh"

namespace fhb {
namespace {

constexpr int kBlock = FHB_ADAMW_BLOCK;
constexpr int kMaxTensors = 32;

struct AdamwConstants {
  double beta1, beta2, lr;  // for the bias corrections
  float b1, c1, b2, c2, decay, eps;  // beta, 1 - beta, 1 - lr weight_decay
};
struct AdamwBatch {
  fhb_adamw_tensor tensor[kMaxTensors];
  int64_t first_block[kMaxTensors + 1];  // running count of 256-value blocks
  int tensors;
};

// The maximum of two magnitudes; NaN wins.
__device__ __forceinline__ float max_or_nan(float a, float b) {
  return a != a ? a : (b != b ? b : fmaxf(a, b));
}
__device__ __forceinline__ float warp_max_or_nan(float v) {
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1) v = max_or_nan(v, __shfl_xor_sync(0xffffffffu, v, m));
  return v;
}
__device__ __forceinline__ float block_scale(float largest) {
  if (largest == INFINITY) return NAN;  // as a NaN in the block: all of it decodes to NaN
  const float s = __fmul_rn(largest, 1.0f / 448.0f);
  return s < 0x1p-126f ? 0x1p-126f : s;  // a NaN stays
}
__device__ __forceinline__ uint8_t encode(float x) {
  return __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float decode(uint8_t c) {
  __nv_fp8_e4m3 v;
  v.__x = c;
  return static_cast<float>(v);
}

// One warp per block of 256 values, eight per lane.
template <bool Eight>
__global__ void __launch_bounds__(256)
    adamw_kernel(const __grid_constant__ AdamwBatch batch, AdamwConstants k,
                 const int64_t* __restrict__ step) {
  const int64_t block = (blockIdx.x * 256ll + threadIdx.x) / 32;
  const int lane = threadIdx.x % 32;
  if (block >= batch.first_block[batch.tensors]) return;
  int at = 0;
  while (block >= batch.first_block[at + 1]) ++at;
  const fhb_adamw_tensor& t = batch.tensor[at];
  const int64_t own = block - batch.first_block[at], base = own * kBlock;
  const double now = static_cast<double>(*step + 1);
  const float step_size = static_cast<float>(k.lr / (1.0 - pow(k.beta1, now)));
  const float root = static_cast<float>(sqrt(1.0 - pow(k.beta2, now)));
  float sm = 0.0f, sv = 0.0f;
  if (Eight) {
    sm = t.exp_avg_scale[own];
    sv = t.exp_avg_sq_scale[own];
  }
  float m[8], v[8];
  float top_m = 0.0f, top_v = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t j = base + lane + 32 * i;
    m[i] = v[i] = 0.0f;
    if (j >= t.count) continue;
    const bool wide = t.dtype == FHB_DTYPE_F32;
    const float g = wide ? static_cast<const float*>(t.grad)[j]
                         : to_float(static_cast<const bf16*>(t.grad)[j]);
    const float p = wide ? static_cast<float*>(t.param)[j] : to_float(static_cast<bf16*>(t.param)[j]);
    float m0, v0;
    if (Eight) {
      m0 = __fmul_rn(decode(static_cast<uint8_t*>(t.exp_avg)[j]), sm);
      const float s = __fmul_rn(decode(static_cast<uint8_t*>(t.exp_avg_sq)[j]), sv);
      v0 = __fmul_rn(s, s);
    } else {
      m0 = static_cast<float*>(t.exp_avg)[j];
      v0 = static_cast<float*>(t.exp_avg_sq)[j];
    }
    m[i] = __fadd_rn(__fmul_rn(m0, k.b1), __fmul_rn(g, k.c1));
    v[i] = __fadd_rn(__fmul_rn(v0, k.b2), __fmul_rn(__fmul_rn(g, g), k.c2));
    const float denominator = sqrtf(v[i]) / root + k.eps;
    const float next = p * k.decay - step_size * (m[i] / denominator);
    if (wide) static_cast<float*>(t.param)[j] = next;
    else static_cast<bf16*>(t.param)[j] = from_float<bf16>(next);
    if (Eight) {
      v[i] = __fsqrt_rn(v[i]);
      top_m = max_or_nan(top_m, fabsf(m[i]));
      top_v = max_or_nan(top_v, v[i]);
    } else {
      static_cast<float*>(t.exp_avg)[j] = m[i];
      static_cast<float*>(t.exp_avg_sq)[j] = v[i];
    }
  }
  if (!Eight) return;
  const float new_sm = block_scale(warp_max_or_nan(top_m));
  const float new_sv = block_scale(warp_max_or_nan(top_v));
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t j = base + lane + 32 * i;
    if (j >= t.count) continue;
    float units = __fdiv_rn(v[i], new_sv);
    if (v[i] > 0.0f) units = units < 0x1p-9f ? 0x1p-9f : units;
    static_cast<uint8_t*>(t.exp_avg)[j] = encode(__fdiv_rn(m[i], new_sm));
    static_cast<uint8_t*>(t.exp_avg_sq)[j] = encode(units);
  }
  if (lane == 0) {
    t.exp_avg_scale[own] = new_sm;
    t.exp_avg_sq_scale[own] = new_sv;
  }
}

__global__ void advance_kernel(int64_t* step) { *step += 1; }

}  // namespace

cudaError_t launch_adamw(const fhb_adamw_tensor* tensors, int64_t n_tensors, int state_bits,
                         int64_t* step, double lr, double beta1, double beta2, double eps,
                         double weight_decay, cudaStream_t stream) {
  const AdamwConstants k{beta1, beta2, lr, static_cast<float>(beta1), static_cast<float>(1.0 - beta1),
                         static_cast<float>(beta2), static_cast<float>(1.0 - beta2),
                         static_cast<float>(1.0 - lr * weight_decay), static_cast<float>(eps)};
  for (int64_t first = 0; first < n_tensors; first += kMaxTensors) {
    AdamwBatch batch{};
    batch.tensors = static_cast<int>(std::min<int64_t>(kMaxTensors, n_tensors - first));
    for (int i = 0; i < batch.tensors; ++i) {
      batch.tensor[i] = tensors[first + i];
      batch.first_block[i + 1] = batch.first_block[i] + (tensors[first + i].count + kBlock - 1) / kBlock;
    }
    const int64_t blocks = batch.first_block[batch.tensors];
    if (blocks == 0) continue;
    const int64_t grid = (blocks + 7) / 8;
    if (grid > 0x7FFFFFFF) return cudaErrorInvalidValue;
    if (state_bits == 8)
      adamw_kernel<true><<<static_cast<unsigned>(grid), 256, 0, stream>>>(batch, k, step);
    else
      adamw_kernel<false><<<static_cast<unsigned>(grid), 256, 0, stream>>>(batch, k, step);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  advance_kernel<<<1, 1, 0, stream>>>(step);
  return cudaGetLastError();
}

}  // namespace fhb
