// The gated feed-forward block: g = x Wg^T + bg, u = x Wu^T + bu, h = act(g) u,
// y = h Wd^T + bd, and its gradients
//     dh = dy Wd,  du = dh act(g),  dg = dh u act'(g),
//     dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x,  dWd = dy^T h,  db = column sums.
#include "blocks.cuh"

namespace fhb {
namespace {

// C[m][n] = sum over terms t, k of A_t(m, k) B_t(n, k) + bias[n], operands with any strides,
// FP32 sums. One 64 x 64 tile per CTA, 16 of K at a time, 4 x 4 results per thread.
constexpr int kTile = 64, kStep = 16;

template <typename T>
struct Operand {
  const T* p;
  int64_t mn, k;  // strides along the result's dimension and along K
};
template <typename T>
struct Product {
  Operand<T> a[2], b[2];
  int terms;
  int64_t m, n, k;
  const T* bias;
};

template <typename T, typename TC>
__global__ void __launch_bounds__(256)
    gemm_kernel(Product<T> p, TC* __restrict__ c, int64_t c_stride) {
  __shared__ float as[kStep][kTile + 4], bs[kStep][kTile + 4];
  const int64_t tiles_n = (p.n + kTile - 1) / kTile;
  const int64_t m0 = (blockIdx.x / tiles_n) * kTile, n0 = (blockIdx.x % tiles_n) * kTile;
  const int tm = (threadIdx.x / 16) * 4, tn = (threadIdx.x % 16) * 4;
  float acc[4][4] = {};
  for (int t = 0; t < p.terms; ++t) {
    const Operand<T> a = p.a[t], b = p.b[t];
    for (int64_t k0 = 0; k0 < p.k; k0 += kStep) {
      for (int i = threadIdx.x; i < kTile * kStep; i += 256) {
        // consecutive threads follow the operand's unit stride
        const int am = a.k == 1 ? i / kStep : i % kTile, ak = a.k == 1 ? i % kStep : i / kTile;
        const int bn = b.k == 1 ? i / kStep : i % kTile, bk = b.k == 1 ? i % kStep : i / kTile;
        as[ak][am] = m0 + am < p.m && k0 + ak < p.k
                         ? to_float(a.p[(m0 + am) * a.mn + (k0 + ak) * a.k]) : 0.0f;
        bs[bk][bn] = n0 + bn < p.n && k0 + bk < p.k
                         ? to_float(b.p[(n0 + bn) * b.mn + (k0 + bk) * b.k]) : 0.0f;
      }
      __syncthreads();
#pragma unroll
      for (int kk = 0; kk < kStep; ++kk)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(as[kk][tm + i], bs[kk][tn + j], acc[i][j]);
      __syncthreads();
    }
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int64_t row = m0 + tm + i, col = n0 + tn + j;
      if (row >= p.m || col >= p.n) continue;
      const float v = acc[i][j] + (p.bias != nullptr ? to_float(p.bias[col]) : 0.0f);
      c[row * c_stride + col] = from_float<TC>(v);
    }
}

template <typename T, typename TC>
cudaError_t gemm(const Product<T>& p, TC* c, int64_t c_stride, cudaStream_t stream) {
  const int64_t tiles = ((p.m + kTile - 1) / kTile) * ((p.n + kTile - 1) / kTile);
  if (tiles == 0) return cudaSuccess;
  if (tiles > 0x7FFFFFFF) return cudaErrorInvalidValue;
  gemm_kernel<<<static_cast<unsigned>(tiles), 256, 0, stream>>>(p, c, c_stride);
  return cudaGetLastError();
}

template <typename T>
__global__ void gate_kernel(const float* __restrict__ g, const float* __restrict__ u,
                            T* __restrict__ h, int64_t count, int activation) {
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < count; i += gridDim.x * 256ll) {
    float a, slope;
    block_activation(activation, g[i], a, slope);
    h[i] = from_float<T>(a * u[i]);
  }
}

template <typename T>
__global__ void gate_backward_kernel(const float* __restrict__ dh, const float* __restrict__ g,
                                     const float* __restrict__ u, T* __restrict__ dg,
                                     T* __restrict__ du, int64_t count, int activation) {
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < count; i += gridDim.x * 256ll) {
    float a, slope;
    block_activation(activation, g[i], a, slope);
    du[i] = from_float<T>(dh[i] * a);
    dg[i] = from_float<T>(dh[i] * u[i] * slope);
  }
}

// out[c] = sum over rows of in[r][c], in row order.
template <typename T>
__global__ void column_sum_kernel(const T* __restrict__ in, int64_t stride, int64_t rows,
                                  int64_t columns, T* __restrict__ out) {
  const int64_t c = blockIdx.x * 64ll + threadIdx.x;
  if (c >= columns) return;
  float s = 0.0f;
  for (int64_t r = 0; r < rows; ++r) s += to_float(in[r * stride + c]);
  out[c] = from_float<T>(s);
}

template <typename T>
void column_sum(const T* in, int64_t stride, int64_t rows, int64_t columns, void* out,
                cudaStream_t stream) {
  if (out != nullptr)
    column_sum_kernel<<<static_cast<unsigned>((columns + 63) / 64), 64, 0, stream>>>(
        in, stride, rows, columns, static_cast<T*>(out));
}

int64_t round16(int64_t bytes) { return (bytes + 15) & ~int64_t{15}; }

// Saved for the backward: g and u in FP32, h in the block's type.
struct Saved {
  float *g, *u;
  void* h;
};
Saved saved_at(const fhb_ffn_problem& p, void* base) {
  char* c = static_cast<char*>(base);
  const int64_t wide = round16(p.tokens * p.hidden * 4);
  return {reinterpret_cast<float*>(c), reinterpret_cast<float*>(c + wide), c + 2 * wide};
}

template <typename T>
cudaError_t forward(const fhb_ffn_problem& p, void* y, void* saved, void* workspace,
                    cudaStream_t stream) {
  const Saved s = saved_at(p, saved != nullptr ? saved : workspace);
  const int64_t t = p.tokens, d = p.width, h = p.hidden, o = p.out_width;
  const Operand<T> x{static_cast<const T*>(p.x), p.x_stride, 1};
  const Operand<T> wg{static_cast<const T*>(p.w_gate), p.w_gate_stride, 1};
  const Operand<T> wu{static_cast<const T*>(p.w_up), p.w_up_stride, 1};
  const Operand<T> wd{static_cast<const T*>(p.w_down), p.w_down_stride, 1};
  const Operand<T> hidden{static_cast<const T*>(s.h), h, 1};
  cudaError_t e = gemm(Product<T>{{x}, {wg}, 1, t, h, d, static_cast<const T*>(p.b_gate)}, s.g, h, stream);
  if (e == cudaSuccess)
    e = gemm(Product<T>{{x}, {wu}, 1, t, h, d, static_cast<const T*>(p.b_up)}, s.u, h, stream);
  if (e != cudaSuccess) return e;
  gate_kernel<<<1184, 256, 0, stream>>>(s.g, s.u, static_cast<T*>(s.h), t * h, p.activation);
  return gemm(Product<T>{{hidden}, {wd}, 1, t, o, h, static_cast<const T*>(p.b_down)},
              static_cast<T*>(y), o, stream);
}

template <typename T>
cudaError_t backward(const fhb_ffn_problem& p, const T* dy, int64_t dy_stride, const void* saved,
                     const fhb_ffn_grads& out, void* workspace, cudaStream_t stream) {
  const Saved s = saved_at(p, const_cast<void*>(saved));
  const int64_t t = p.tokens, d = p.width, h = p.hidden, o = p.out_width;
  const int64_t wide = round16(t * h * 4), narrow = round16(t * h * sizeof(T));
  char* ws = static_cast<char*>(workspace);
  float* dh = reinterpret_cast<float*>(ws);
  T* dg = reinterpret_cast<T*>(ws + wide);
  T* du = reinterpret_cast<T*>(ws + wide + narrow);
  const T* x = static_cast<const T*>(p.x);
  const T *wg = static_cast<const T*>(p.w_gate), *wu = static_cast<const T*>(p.w_up);
  cudaError_t e = gemm(Product<T>{{{dy, dy_stride, 1}},
                                  {{static_cast<const T*>(p.w_down), 1, p.w_down_stride}}, 1, t, h, o},
                       dh, h, stream);
  if (e != cudaSuccess) return e;
  if (t > 0)
    gate_backward_kernel<<<1184, 256, 0, stream>>>(dh, s.g, s.u, dg, du, t * h, p.activation);
  if (out.x != nullptr)
    e = gemm(Product<T>{{{dg, h, 1}, {du, h, 1}}, {{wg, 1, p.w_gate_stride}, {wu, 1, p.w_up_stride}},
                        2, t, d, h},
             static_cast<T*>(out.x), d, stream);
  if (e == cudaSuccess && out.w_gate != nullptr)
    e = gemm(Product<T>{{{dg, 1, h}}, {{x, 1, p.x_stride}}, 1, h, d, t}, static_cast<T*>(out.w_gate), d, stream);
  if (e == cudaSuccess && out.w_up != nullptr)
    e = gemm(Product<T>{{{du, 1, h}}, {{x, 1, p.x_stride}}, 1, h, d, t}, static_cast<T*>(out.w_up), d, stream);
  if (e == cudaSuccess && out.w_down != nullptr)
    e = gemm(Product<T>{{{dy, 1, dy_stride}}, {{static_cast<const T*>(s.h), 1, h}}, 1, o, h, t},
             static_cast<T*>(out.w_down), h, stream);
  if (e != cudaSuccess) return e;
  column_sum(dg, h, t, h, out.b_gate, stream);
  column_sum(du, h, t, h, out.b_up, stream);
  column_sum(dy, dy_stride, t, o, out.b_down, stream);
  return cudaGetLastError();
}

}  // namespace

size_t ffn_saved_bytes(const fhb_ffn_problem& p) {
  return 2 * round16(p.tokens * p.hidden * 4) + round16(p.tokens * p.hidden * dtype_bytes(p.dtype));
}

size_t ffn_workspace_bytes(const fhb_ffn_problem& p, bool backward, const DeviceInfo&) {
  if (!backward) return ffn_saved_bytes(p);
  return round16(p.tokens * p.hidden * 4) + 2 * round16(p.tokens * p.hidden * dtype_bytes(p.dtype));
}

cudaError_t launch_ffn_forward(const fhb_ffn_problem& p, void* y, void* saved, void* workspace,
                               const DeviceInfo&, cudaStream_t stream) {
  return p.dtype == FHB_DTYPE_F32 ? forward<float>(p, y, saved, workspace, stream)
                                  : forward<bf16>(p, y, saved, workspace, stream);
}

cudaError_t launch_ffn_backward(const fhb_ffn_problem& p, const void* grad_y, int64_t grad_y_stride,
                                const void* saved, const fhb_ffn_grads& grads, void* workspace,
                                const DeviceInfo&, cudaStream_t stream) {
  return p.dtype == FHB_DTYPE_F32
             ? backward(p, static_cast<const float*>(grad_y), grad_y_stride, saved, grads, workspace, stream)
             : backward(p, static_cast<const bf16*>(grad_y), grad_y_stride, saved, grads, workspace, stream);
}

}  // namespace fhb
