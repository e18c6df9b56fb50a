// One AdamW step over many tensors, moments in FP32 or in 8 bits (e4m3 codes of m and sqrt(v)
// with one scale per block of 256 values).
//
// Bound by memory: 28 bytes a value with FP32 parameters and states, 10 with bfloat16 parameters
// and 8-bit states. A warp takes a block of 256 values, 8 neighbours a lane, so every array is
// moved in whole sectors and an 8-bit block's largest value is one warp maximum away. The
// moments are the formula's, operation by operation (no contraction into fused multiply-adds;
// quotients and roots correctly rounded), so moments, codes and scales are those of the same
// formula in any IEEE FP32 arithmetic; the parameter's update uses approximate quotients (2^-22
// of the update). The tensors' addresses travel as kernel arguments: nothing is copied to the
// device before the launch, and the step counter is advanced by the last CTA to finish.
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>

#include "blocks.cuh"
#include "common.cuh"

namespace fhb {
namespace {

constexpr int kBlock = FHB_ADAMW_BLOCK;
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kResident = 3, kResidentEight = 3;  // CTAs an SM holds
// Tensors of one launch: its arguments hold 4 KB cheaply and 32 KB at most.
constexpr int kFewTensors = 40, kManyTensors = 400;
// The step counter's upper bits count the CTAs that are done (0 between launches).
constexpr int kStepBits = 40;
constexpr unsigned long long kStepMask = (1ull << kStepBits) - 1;

struct Constants {
  double beta1, beta2, lr;           // for the bias corrections
  float b1, c1, b2, c2, decay, eps;  // beta, 1 - beta, 1 - lr weight_decay
};
template <int Capacity>
struct Batch {
  fhb_adamw_tensor tensor[Capacity];
  int64_t first_block[Capacity + 1];  // running count of 256-value blocks
  unsigned char wide[Capacity];       // every array of the tensor is aligned for 8 values
  int tensors;
  int advances;  // the last launch of the step
};

// ---- 8 neighbours of an array ----
template <typename T>
__device__ __forceinline__ void load8(const T* p, int left, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = i < left ? to_float(p[i]) : 0.0f;
}
__device__ __forceinline__ void store8(float* p, bool full, int left, const float (&x)[8]) {
  if (full) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p),
                 "r"(__float_as_uint(x[0])), "r"(__float_as_uint(x[1])), "r"(__float_as_uint(x[2])),
                 "r"(__float_as_uint(x[3])), "r"(__float_as_uint(x[4])), "r"(__float_as_uint(x[5])),
                 "r"(__float_as_uint(x[6])), "r"(__float_as_uint(x[7]))
                 : "memory");
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < left) p[i] = x[i];
}
__device__ __forceinline__ void store8(bf16* p, bool full, int left, const float (&x)[8]) {
  if (full) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(u[i]) : "f"(x[2 * i + 1]), "f"(x[2 * i]));
    *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < left) p[i] = from_float<bf16>(x[i]);
}
__device__ __forceinline__ uint2 load_codes(const uint8_t* p, int left) {
  unsigned long long w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < left) w |= static_cast<unsigned long long>(p[i]) << (8 * i);
  return make_uint2(static_cast<uint32_t>(w), static_cast<uint32_t>(w >> 32));
}
__device__ __forceinline__ void decode8(uint2 codes, float scale, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t pair = ((i < 2 ? codes.x : codes.y) >> (16 * (i & 1))) & 0xFFFFu;
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(pair), __NV_E4M3);
    const float2 v = __half22float2(__half2(h));
    mul2o(x[2 * i], x[2 * i + 1], v.x, v.y, scale, scale);
  }
}
__device__ __forceinline__ void store_codes(uint8_t* p, bool full, int left, const float (&units)[8]) {
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i / 2] |= static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(units[2 * i], units[2 * i + 1]),
                                                               __NV_SATFINITE, __NV_E4M3))
                << (16 * (i & 1));
  if (full) {
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < left) p[i] = static_cast<uint8_t>(w[i / 4] >> (8 * (i & 3)));
}

// Largest of non-negative values over the warp; NaN (whatever its sign bit was) wins: as bit
// patterns, NaN > infinity > numbers in order.
__device__ __forceinline__ float warp_largest(const float (&x)[8]) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
  return __uint_as_float(__reduce_max_sync(0xffffffffu, top));
}
__device__ __forceinline__ float block_scale(float largest) {
  if (!(largest < INFINITY)) return NAN;  // a block with a NaN or infinity decodes to NaN
  const float s = __fmul_rn(largest, 1.0f / 448.0f);
  return s < 0x1p-126f ? 0x1p-126f : s;
}
// x[i] / scale, correctly rounded: one reciprocal for the block and Markstein's remainder step
// for each value. With r the correctly rounded 1 / s, q = x r is off by an ulp at most and
// q + (x - q s) r is the correctly rounded quotient, as long as the remainder does not
// underflow -- blocks whose largest value is that small divide.
__device__ __forceinline__ void divide8(float (&x)[8], float scale) {
  if (scale < 0x1p-90f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __fdiv_rn(x[i], scale);
    return;
  }
  const float r = __frcp_rn(scale);
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    float q0, q1, d0, d1;
    mul2o(q0, q1, x[i], x[i + 1], r, r);
    fma2o(d0, d1, q0, q1, -scale, -scale, x[i], x[i + 1]);
    fma2o(x[i], x[i + 1], d0, d1, r, r, q0, q1);
  }
}

// What a lane loads of its block, as it lies in memory: the next block's is on its way while
// this one's is worked on.
template <bool Eight, typename T>
struct Raw {
  uint32_t g[2 * sizeof(T)], p[2 * sizeof(T)], m[Eight ? 2 : 8], v[Eight ? 2 : 8];
  float sm, sv;
};
template <int Words>
__device__ __forceinline__ void load_words(const void* p, uint32_t (&w)[Words]) {
  if constexpr (Words == 8)
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]),
                   "=r"(w[6]), "=r"(w[7])
                 : "l"(p)
                 : "memory");
  else if constexpr (Words == 4)
    asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                 : "l"(p)
                 : "memory");
  else
    asm volatile("ld.global.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p) : "memory");
}
template <bool Eight, typename T>
__device__ __forceinline__ void load_raw(const fhb_adamw_tensor& t, int64_t own, int lane, Raw<Eight, T>& w) {
  const int64_t at = own * kBlock + lane * 8;
  load_words(static_cast<const T*>(t.grad) + at, w.g);
  load_words(static_cast<const T*>(t.param) + at, w.p);
  if constexpr (Eight) {
    load_words(static_cast<const uint8_t*>(t.exp_avg) + at, w.m);
    load_words(static_cast<const uint8_t*>(t.exp_avg_sq) + at, w.v);
    w.sm = t.exp_avg_scale[own];
    w.sv = t.exp_avg_sq_scale[own];
  } else {
    load_words(static_cast<const float*>(t.exp_avg) + at, w.m);
    load_words(static_cast<const float*>(t.exp_avg_sq) + at, w.v);
  }
}
template <int Words>
__device__ __forceinline__ void unpack(const uint32_t (&w)[Words], float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < Words; ++i) {
    if constexpr (Words == 8) {
      x[i] = __uint_as_float(w[i]);
    } else {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
}

// The values of a last block or an unaligned tensor, one by one.
template <bool Eight, typename T>
__device__ __forceinline__ void load_single(const fhb_adamw_tensor& t, int64_t own, int lane,
                                            float (&g)[8], float (&p)[8], float (&m)[8],
                                            float (&v)[8]) {
  const int64_t at = own * kBlock + lane * 8;
  const int left = static_cast<int>(min(t.count - at, int64_t{8}));  // may be negative
  load8(static_cast<const T*>(t.grad) + at, left, g);
  load8(static_cast<const T*>(t.param) + at, left, p);
  if constexpr (Eight) {
    decode8(load_codes(static_cast<const uint8_t*>(t.exp_avg) + at, left), t.exp_avg_scale[own], m);
    decode8(load_codes(static_cast<const uint8_t*>(t.exp_avg_sq) + at, left), t.exp_avg_sq_scale[own], v);
  } else {
    load8(static_cast<const float*>(t.exp_avg) + at, left, m);
    load8(static_cast<const float*>(t.exp_avg_sq) + at, left, v);
  }
}

// One block by one warp, from its gradient, parameter, m, and v (8 bits: sqrt(v)). Full: all
// 256 values exist and every array is aligned for 8 of them.
template <bool Eight, typename T, bool full>
__device__ __forceinline__ void update_block(const fhb_adamw_tensor& t, int64_t own, int lane,
                                             const Constants& k, float step_size,
                                             float inverse_root, const float (&g)[8], float (&p)[8],
                                             float (&m)[8], float (&v)[8]) {
  const int64_t at = own * kBlock + lane * 8;
  const int left = full ? 8 : static_cast<int>(min(t.count - at, int64_t{8}));
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    float a0, a1, c0, c1;
    if (Eight) mul2o(v[i], v[i + 1], v[i], v[i + 1], v[i], v[i + 1]);
    mul2o(a0, a1, m[i], m[i + 1], k.b1, k.b1);
    mul2o(c0, c1, g[i], g[i + 1], k.c1, k.c1);
    // single additions: a packed one would be contracted with the packed products before it
    m[i] = __fadd_rn(a0, c0);
    m[i + 1] = __fadd_rn(a1, c1);
    mul2o(a0, a1, v[i], v[i + 1], k.b2, k.b2);
    mul2o(c0, c1, g[i], g[i + 1], g[i], g[i + 1]);
    mul2o(c0, c1, c0, c1, k.c2, k.c2);
    v[i] = __fadd_rn(a0, c0);
    v[i + 1] = __fadd_rn(a1, c1);
  }
  if (!Eight) {
    store8(static_cast<float*>(t.exp_avg) + at, full, left, m);
    store8(static_cast<float*>(t.exp_avg_sq) + at, full, left, v);
  }
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    if (Eight) {
      v[i] = __fsqrt_rn(v[i]);
      v[i + 1] = __fsqrt_rn(v[i + 1]);
    } else {
      asm("sqrt.approx.f32 %0, %0;" : "+f"(v[i]));
      asm("sqrt.approx.f32 %0, %0;" : "+f"(v[i + 1]));
    }
    float d0, d1, w0, w1;
    fma2o(d0, d1, v[i], v[i + 1], inverse_root, inverse_root, k.eps, k.eps);
    mul2o(w0, w1, p[i], p[i + 1], k.decay, k.decay);
    // a denominator of 0 (eps 0): 0 / 0 and x / 0 as IEEE has them
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(d0));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(d1));
    mul2o(d0, d1, d0, d1, m[i], m[i + 1]);
    fma2o(p[i], p[i + 1], d0, d1, -step_size, -step_size, w0, w1);
  }
  store8(static_cast<T*>(t.param) + at, full, left, p);
  if (!Eight) return;
  const float scale_m = block_scale(warp_largest(m)), scale_v = block_scale(warp_largest(v));
  divide8(m, scale_m);
  float units[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) units[i] = v[i];
  divide8(units, scale_v);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    units[i] = fmaxf(units[i], v[i] > 0.0f ? 0x1p-9f : 0.0f);  // not zero stays not zero
  store_codes(static_cast<uint8_t*>(t.exp_avg) + at, full, left, m);
  store_codes(static_cast<uint8_t*>(t.exp_avg_sq) + at, full, left, units);
  if (lane == 0) {
    t.exp_avg_scale[own] = scale_m;
    t.exp_avg_sq_scale[own] = scale_v;
  }
}

// The rest: last blocks of a tensor and unaligned tensors, kept out of the others' registers.
template <bool Eight, typename T>
__device__ __noinline__ void update_partial(const fhb_adamw_tensor& t, int64_t own, int lane,
                                            const Constants& k, float step_size,
                                            float inverse_root) {
  float g[8], p[8], m[8], v[8];
  load_single<Eight, T>(t, own, lane, g, p, m, v);
  update_block<Eight, T, false>(t, own, lane, k, step_size, inverse_root, g, p, m, v);
}
template <bool Eight, typename T>
__device__ __forceinline__ int64_t update_tensor(const fhb_adamw_tensor& t, bool wide, int64_t block,
                                                 int64_t first, int64_t end, int64_t stride, int lane,
                                                 const Constants& k, float step_size,
                                                 float inverse_root) {
  // blocks before `whole` are full
  const int64_t whole = first + (wide ? t.count / kBlock : 0);
  if (block < whole) {
    Raw<Eight, T> w;
    load_raw(t, block - first, lane, w);
    while (true) {
      float g[8], p[8], m[8], v[8];
      unpack(w.g, g);
      unpack(w.p, p);
      if constexpr (Eight) {
        decode8(make_uint2(w.m[0], w.m[1]), w.sm, m);
        decode8(make_uint2(w.v[0], w.v[1]), w.sv, v);
      } else {
        unpack(w.m, m);
        unpack(w.v, v);
      }
      const int64_t own = block - first;
      block += stride;
      if (Eight && block < whole) load_raw(t, block - first, lane, w);
      update_block<Eight, T, true>(t, own, lane, k, step_size, inverse_root, g, p, m, v);
      if (block >= whole) break;
      if (!Eight) load_raw(t, block - first, lane, w);
    }
  }
  for (; block < end; block += stride)
    update_partial<Eight, T>(t, block - first, lane, k, step_size, inverse_root);
  return block;
}

template <bool Eight, int Capacity>
__global__ void __launch_bounds__(kThreads, Eight ? kResidentEight : kResident)
    adamw_kernel(const __grid_constant__ Batch<Capacity> batch, const __grid_constant__ Constants k,
                 unsigned long long* step) {
  __shared__ float corrections[2];
  __shared__ unsigned long long now;
  if (threadIdx.x == 0) {
    // volatile: other CTAs add to the upper bits
    now = (*const_cast<volatile unsigned long long*>(step) & kStepMask) + 1;
    const double t = static_cast<double>(now);
    corrections[0] = static_cast<float>(k.lr / (1.0 - pow(k.beta1, t)));
    corrections[1] = static_cast<float>(1.0 / sqrt(1.0 - pow(k.beta2, t)));
  }
  __syncthreads();
  const float step_size = corrections[0], inverse_root = corrections[1];
  const int lane = threadIdx.x % 32;
  const int64_t blocks = batch.first_block[batch.tensors];
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kWarps;
  int64_t block = blockIdx.x * static_cast<int64_t>(kWarps) + threadIdx.x / 32;
  int at = 0;
  while (block < blocks) {
    // the tensor: the last one whose first block is not past this (blocks only go up)
    int low = at, high = batch.tensors;
    while (high - low > 1) {
      const int mid = (low + high) / 2;
      if (batch.first_block[mid] <= block) low = mid;
      else high = mid;
    }
    at = low;
    const fhb_adamw_tensor& t = batch.tensor[at];
    const bool wide = batch.wide[at] != 0;
    const int64_t first = batch.first_block[at], end = batch.first_block[at + 1];
    block = t.dtype == FHB_DTYPE_F32
                ? update_tensor<Eight, float>(t, wide, block, first, end, stride, lane, k, step_size, inverse_root)
                : update_tensor<Eight, bf16>(t, wide, block, first, end, stride, lane, k, step_size, inverse_root);
  }
  if (!batch.advances) return;
  __syncthreads();
  if (threadIdx.x == 0 && atomicAdd(step, 1ull << kStepBits) >> kStepBits == gridDim.x - 1)
    *step = now;  // every CTA has read the counter
}

bool aligned(const void* p, uintptr_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

template <int Capacity>
cudaError_t launch(const fhb_adamw_tensor* tensors, int64_t count, bool eight, bool advances,
                   unsigned long long* step, const Constants& k, const DeviceInfo& dev,
                   cudaStream_t stream) {
  Batch<Capacity> batch{};
  batch.tensors = static_cast<int>(count);
  batch.advances = advances;
  for (int i = 0; i < batch.tensors; ++i) {
    const fhb_adamw_tensor& t = tensors[i];
    batch.tensor[i] = t;
    batch.first_block[i + 1] = batch.first_block[i] + (t.count + kBlock - 1) / kBlock;
    const uintptr_t of_param = 8 * dtype_bytes(t.dtype), of_state = eight ? 8 : 32;
    batch.wide[i] = aligned(t.param, of_param) && aligned(t.grad, of_param) &&
                    aligned(t.exp_avg, of_state) && aligned(t.exp_avg_sq, of_state);
  }
  const int64_t need = (batch.first_block[count] + kWarps - 1) / kWarps;
  if (need == 0 && !advances) return cudaSuccess;
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(std::max<int64_t>(need, 1), static_cast<int64_t>(eight ? kResidentEight : kResident) * dev.sms));
  if (eight)
    adamw_kernel<true, Capacity><<<grid, kThreads, 0, stream>>>(batch, k, step);
  else
    adamw_kernel<false, Capacity><<<grid, kThreads, 0, stream>>>(batch, k, step);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_adamw(const fhb_adamw_tensor* tensors, int64_t n_tensors, int state_bits,
                         int64_t* step, double lr, double beta1, double beta2, double eps,
                         double weight_decay, const DeviceInfo& dev, cudaStream_t stream) {
  const Constants k{beta1, beta2, lr, static_cast<float>(beta1), static_cast<float>(1.0 - beta1),
                    static_cast<float>(beta2), static_cast<float>(1.0 - beta2),
                    static_cast<float>(1.0 - lr * weight_decay), static_cast<float>(eps)};
  auto* counter = reinterpret_cast<unsigned long long*>(step);
  int64_t first = 0;
  do {
    const int64_t left = n_tensors - first;
    const int64_t count = std::min<int64_t>(left, kManyTensors);
    const bool last = count == left;
    const cudaError_t e =
        count <= kFewTensors
            ? launch<kFewTensors>(tensors + first, count, state_bits == 8, last, counter, k, dev, stream)
            : launch<kManyTensors>(tensors + first, count, state_bits == 8, last, counter, k, dev, stream);
    if (e != cudaSuccess) return e;
    first += count;
  } while (first < n_tensors);
  return cudaSuccess;
}

}  // namespace fhb
