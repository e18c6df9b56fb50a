// The gated feed-forward block for a few tokens (serving one token or point at a time), without
// gradients: every weight is used once, so the time is that of reading the weights. Two launches
// of one dot-product kernel, straight from the caller's weights:
//     h = act(x Wg^T + bg) (x Wu^T + bu),   y = h Wd^T + bd.
// A result feature is one to eight warps: each lane takes 16 bytes of the weight row (both rows
// of the gate) every 512 bytes, four such loads in flight, times the same place of every token.
// h is rounded to the block's type, as where it is an operand of the products: a token's answer has the
// same roundings alone and in a batch. The second launch is a dependent one: its first weights are on
// their way before it waits for h.
// 1024 x 4096, both launches: bf16 11.3 us for one token (2.2 TB/s; the two launches themselves
// are about half of it), fp32 15.0 us (3.4 TB/s).
#include <algorithm>

#include "common.cuh"
#include "gated_ffn.cuh"

namespace fhb {
namespace {

constexpr int kWarps = 8;
constexpr int kInFlight = 4;

struct DotArgs {
  const void* x;
  int64_t x_stride;
  const void* w[2];
  int64_t w_stride[2];
  const void* bias[2];
  void* out;  // [token][out_stride]
  int64_t out_stride;
  int64_t features, k;
  int split;  // warps of one feature
  int tokens, activation;
};

// 16 bytes of a row of T from element k0 on, zeros past `k`: one load where rows are aligned.
template <typename T, bool Wide>
__device__ __forceinline__ uint4 load16(const T* row, int64_t k0, int64_t k) {
  constexpr int kEach = 16 / sizeof(T);
  if (Wide) return k0 < k ? __ldg(reinterpret_cast<const uint4*>(row + k0)) : make_uint4(0, 0, 0, 0);
  uint32_t w[4] = {};
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    if (k0 + i >= k) break;
    if constexpr (sizeof(T) == 4)
      w[i] = __float_as_uint(row[k0 + i]);
    else
      w[i / 2] |= static_cast<uint32_t>(__bfloat16_as_ushort(row[k0 + i])) << (16 * (i & 1));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T>
__device__ __forceinline__ void unpack16(uint4 v, float (&f)[16 / sizeof(T)]) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      f[i] = __uint_as_float(u[i]);
    } else {
      f[2 * i] = __uint_as_float(u[i] << 16);
      f[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
    }
  }
}

template <typename T, int Rows, int Tokens, bool Wide>
__global__ void __launch_bounds__(kWarps * 32) dot_kernel(const __grid_constant__ DotArgs a) {
  constexpr int kEach = 16 / sizeof(T);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int64_t feature = blockIdx.x * static_cast<int64_t>(kWarps / a.split) + warp / a.split;
  const bool real = feature < a.features;
  const int64_t step = static_cast<int64_t>(a.split) * 32 * kEach;
  int64_t k0 = (warp % a.split) * 32 * kEach + lane * kEach;
  const T* w[Rows];
#pragma unroll
  for (int r = 0; r < Rows; ++r) w[r] = static_cast<const T*>(a.w[r]) + (real ? feature : 0) * a.w_stride[r];
  float acc[Rows][Tokens] = {};
  uint4 words[kInFlight][Rows];
  const auto load = [&] {
#pragma unroll
    for (int i = 0; i < kInFlight; ++i)
#pragma unroll
      for (int r = 0; r < Rows; ++r) words[i][r] = load16<T, Wide>(w[r], k0 + i * step, a.k);
  };
  load();
  if (Rows == 2) allow_dependents();
  else wait_for_prerequisites();  // x is the first launch's h
  const T* x = static_cast<const T*>(a.x);
  while (k0 < a.k) {
#pragma unroll
    for (int i = 0; i < kInFlight; ++i) {
      if (k0 + i * step >= a.k) break;
      float f[Rows][kEach];
#pragma unroll
      for (int r = 0; r < Rows; ++r) unpack16<T>(words[i][r], f[r]);
#pragma unroll
      for (int t = 0; t < Tokens; ++t) {
        // a launch for more tokens than there are takes the last one again
        const T* row = x + min(t, a.tokens - 1) * a.x_stride;
        float v[kEach];
        // not __ldg: h was written by the kernel before this one, which may still have run
        // when this one began
        unpack16<T>(Wide ? *reinterpret_cast<const uint4*>(row + k0 + i * step)
                         : load16<T, false>(row, k0 + i * step, a.k), v);
#pragma unroll
        for (int r = 0; r < Rows; ++r)
#pragma unroll
          for (int j = 0; j < kEach; ++j) acc[r][t] = fmaf(f[r][j], v[j], acc[r][t]);
      }
    }
    k0 += kInFlight * step;
    if (k0 < a.k) load();
  }
  __shared__ float part[kWarps][Rows][Tokens];
#pragma unroll
  for (int r = 0; r < Rows; ++r)
#pragma unroll
    for (int t = 0; t < Tokens; ++t) {
      const float s = warp_sum(acc[r][t]);
      if (lane == 0) part[warp][r][t] = s;
    }
  __syncthreads();
  if (warp % a.split != 0 || lane >= a.tokens || lane >= Tokens || !real) return;
  float s[Rows];
#pragma unroll
  for (int r = 0; r < Rows; ++r) {
    s[r] = 0.0f;
    for (int i = 0; i < a.split; ++i) s[r] += part[warp + i][r][lane];
    if (a.bias[r] != nullptr) s[r] += to_float(static_cast<const T*>(a.bias[r])[feature]);
  }
  float result = s[0];
  if constexpr (Rows == 2) {
    float act, slope;
    if (a.activation == FHB_ACTIVATION_TANH) block_activation<true>(s[0], act, slope);
    else block_activation<false>(s[0], act, slope);
    result = act * s[1];
  }
  static_cast<T*>(a.out)[lane * a.out_stride + feature] = from_float<T>(result);
}

// Warps of a feature: as many as bring the launch to about 28 warps an SM, each with a step.
int split_of(const DotArgs& a, int each, const DeviceInfo& dev) {
  int split = 1;
  while (split < kWarps && a.features * split < 28ll * dev.sms && a.k > 2ll * split * 32 * each) split *= 2;
  return split;
}

template <typename T, int Rows, bool Wide>
cudaError_t launch_dots(const DotArgs& a, cudaStream_t stream) {
  const int64_t each = kWarps / a.split;
  const dim3 grid(static_cast<unsigned>((a.features + each - 1) / each)), block(kWarps * 32);
  const auto go = [&](auto kernel) {
    if (Rows == 1) return launch_dependent(kernel, grid, block, 0, stream, a);
    kernel<<<grid, block, 0, stream>>>(a);
    return cudaGetLastError();
  };
  if (a.tokens == 1) return go(dot_kernel<T, Rows, 1, Wide>);
  if (sizeof(T) == 2 || a.tokens == 2) return go(dot_kernel<T, Rows, 2, Wide>);
  if constexpr (sizeof(T) == 4) {
    if (a.tokens <= 4) return go(dot_kernel<T, Rows, 4, Wide>);
    return go(dot_kernel<T, Rows, 8, Wide>);
  }
  return cudaErrorInvalidValue;
}

template <typename T, int Rows>
cudaError_t dots(DotArgs a, const DeviceInfo& dev, cudaStream_t stream) {
  constexpr int kEach = 16 / sizeof(T);
  a.split = split_of(a, kEach, dev);
  const auto aligned = [](const void* p, int64_t stride) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % kEach == 0;
  };
  bool wide = a.k % kEach == 0 && aligned(a.x, a.x_stride);
  for (int r = 0; r < Rows; ++r) wide = wide && aligned(a.w[r], a.w_stride[r]);
  return wide ? launch_dots<T, Rows, true>(a, stream) : launch_dots<T, Rows, false>(a, stream);
}

template <typename T>
cudaError_t forward(const fhb_ffn_problem& p, void* y, void* h, const DeviceInfo& dev, cudaStream_t stream) {
  const int64_t h_stride = (p.hidden + 7) / 8 * 8;
  DotArgs gate{p.x, p.x_stride, {p.w_gate, p.w_up}, {p.w_gate_stride, p.w_up_stride},
               {p.b_gate, p.b_up}, h, h_stride, p.hidden, p.width, 1,
               static_cast<int>(p.tokens), p.activation};
  const cudaError_t e = dots<T, 2>(gate, dev, stream);
  if (e != cudaSuccess) return e;
  DotArgs down{h, h_stride, {p.w_down, nullptr}, {p.w_down_stride, 0}, {p.b_down, nullptr},
               y, p.out_width, p.out_width, p.hidden, 1, static_cast<int>(p.tokens), p.activation};
  return dots<T, 1>(down, dev, stream);
}

}  // namespace

size_t ffn_small_bytes(const fhb_ffn_problem& p) {
  return static_cast<size_t>(p.tokens) * ((p.hidden + 7) / 8 * 8) * dtype_bytes(p.dtype);
}

cudaError_t launch_ffn_small(const fhb_ffn_problem& p, void* y, void* h, const DeviceInfo& dev,
                             cudaStream_t stream) {
  return p.dtype == FHB_DTYPE_F32 ? forward<float>(p, y, h, dev, stream)
                                  : forward<bf16>(p, y, h, dev, stream);
}

}  // namespace fhb
