// The RMS norms before and after a block with its gate and residual scale:
//     z = b ib wpost,  t = a r + c z,  n = t it wpre,
// with ib = 1 / sqrt(mean(b^2) + eps) and it = 1 / sqrt(mean(t^2) + eps) per row. Gradients,
// with th = t it, bh = b ib, q = dn wpre and means over the row:
//     dt = dT + it (q - th mean(q th)),   dr = a dt,   da = sum dt r,   dwpre = sum dn th,
//     dc = dt z,   dwpost = sum dt c bh,   db = ib (p - bh mean(p bh)),   p = dt c wpost.
// t is recomputed from r and b: it is not read rounded. mean(p bh) = mean(dt c z) is linear in
// mean(q th), so the backward needs one round of three row sums:
//     S1 = sum q th,   A = sum (dT + it q) c z,   B = sum th c z,
//     sum dt c z = A - it (S1 / width) B.
#include "blocks.cuh"

namespace fhb {
namespace {

constexpr int kThreads = 256;

// Sums of K values over the CTA, in a fixed order, to every thread.
template <int K>
__device__ __forceinline__ void block_sum(float (&v)[K]) {
  __shared__ float part[K][kThreads / 32];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) {
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], m);
    if (threadIdx.x % 32 == 0) part[k][threadIdx.x / 32] = v[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) {
    v[k] = 0.0f;
    for (int w = 0; w < kThreads / 32; ++w) v[k] += part[k][w];
  }
}

struct NormArgs {
  const void *residual, *branch, *pre_weight, *post_weight, *gate;
  int64_t rows, width, residual_stride, branch_stride, gate_rows;
  const float* scale_ptr;
  float scale, eps;
};

// One CTA per row (grid-stride).
template <typename TR, typename T>
__global__ void __launch_bounds__(kThreads)
    norm_kernel(NormArgs a, TR* __restrict__ total, T* __restrict__ normed,
                float* __restrict__ stats) {
  const float scale = a.scale_ptr != nullptr ? *a.scale_ptr : a.scale;
  const T *pre = static_cast<const T*>(a.pre_weight), *post = static_cast<const T*>(a.post_weight);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const TR* r = static_cast<const TR*>(a.residual) + row * a.residual_stride;
    const T* b = a.branch != nullptr ? static_cast<const T*>(a.branch) + row * a.branch_stride : nullptr;
    const T* gate = a.gate != nullptr
                        ? static_cast<const T*>(a.gate) + row / a.gate_rows * a.width : nullptr;
    float ib = 1.0f;
    if (post != nullptr) {
      float s[1] = {};
      for (int64_t c = threadIdx.x; c < a.width; c += kThreads) {
        const float v = to_float(b[c]);
        s[0] += v * v;
      }
      block_sum(s);
      ib = 1.0f / sqrtf(s[0] / a.width + a.eps);
    }
    const auto value = [&](int64_t c) {
      float t = scale * to_float(r[c]);
      if (b != nullptr) {
        float z = to_float(b[c]);
        if (post != nullptr) z = z * ib * to_float(post[c]);
        t += gate != nullptr ? to_float(gate[c]) * z : z;
      }
      return t;
    };
    float s[1] = {};
    for (int64_t c = threadIdx.x; c < a.width; c += kThreads) {
      const float t = value(c);
      s[0] += t * t;
    }
    block_sum(s);
    const float it = 1.0f / sqrtf(s[0] / a.width + a.eps);
    for (int64_t c = threadIdx.x; c < a.width; c += kThreads) {
      const float t = value(c);
      if (total != nullptr) total[row * a.width + c] = from_float<TR>(t);
      normed[row * a.width + c] = from_float<T>(t * it * to_float(pre[c]));
    }
    if (stats != nullptr && threadIdx.x == 0) {
      stats[2 * row] = ib;
      stats[2 * row + 1] = it;
    }
  }
}

struct NormGrads {
  const void *total, *normed;
  int64_t total_stride, normed_stride;
  void *residual, *branch;
  float *dt;  // [rows][width], the gradient of t
};

// Row part: dr, db and dt.
template <typename TR, typename T>
__global__ void __launch_bounds__(kThreads)
    norm_backward_kernel(NormArgs a, NormGrads g, const float* __restrict__ stats) {
  const float scale = a.scale_ptr != nullptr ? *a.scale_ptr : a.scale;
  const T *pre = static_cast<const T*>(a.pre_weight), *post = static_cast<const T*>(a.post_weight);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const TR* r = static_cast<const TR*>(a.residual) + row * a.residual_stride;
    const T* b = a.branch != nullptr ? static_cast<const T*>(a.branch) + row * a.branch_stride : nullptr;
    const T* gate = a.gate != nullptr
                        ? static_cast<const T*>(a.gate) + row / a.gate_rows * a.width : nullptr;
    const TR* dtotal = g.total != nullptr ? static_cast<const TR*>(g.total) + row * g.total_stride : nullptr;
    const T* dn = g.normed != nullptr ? static_cast<const T*>(g.normed) + row * g.normed_stride : nullptr;
    const float ib = stats[2 * row], it = stats[2 * row + 1];
    const auto pieces = [&](int64_t c, float& cz, float& th, float& q, float& dT) {
      cz = 0.0f;
      if (b != nullptr) {
        cz = to_float(b[c]);
        if (post != nullptr) cz = cz * ib * to_float(post[c]);
        if (gate != nullptr) cz *= to_float(gate[c]);
      }
      th = (scale * to_float(r[c]) + cz) * it;
      q = dn != nullptr ? to_float(dn[c]) * to_float(pre[c]) : 0.0f;
      dT = dtotal != nullptr ? to_float(dtotal[c]) : 0.0f;
    };
    float s[3] = {};
    float cz, th, q, dT;
    for (int64_t c = threadIdx.x; c < a.width; c += kThreads) {
      pieces(c, cz, th, q, dT);
      s[0] += q * th;
      s[1] += (dT + it * q) * cz;
      s[2] += th * cz;
    }
    block_sum(s);
    const float m1 = s[0] / a.width, m2 = (s[1] - it * m1 * s[2]) / a.width;
    for (int64_t c = threadIdx.x; c < a.width; c += kThreads) {
      pieces(c, cz, th, q, dT);
      const float dt = dT + it * (q - th * m1);
      g.dt[row * a.width + c] = dt;
      if (g.residual != nullptr) static_cast<TR*>(g.residual)[row * a.width + c] = from_float<TR>(scale * dt);
      if (g.branch != nullptr) {
        float p = gate != nullptr ? dt * to_float(gate[c]) : dt;
        if (post != nullptr) p = ib * (p * to_float(post[c]) - to_float(b[c]) * ib * m2);
        static_cast<T*>(g.branch)[row * a.width + c] = from_float<T>(p);
      }
    }
  }
}

// Column part: one thread per column sums dwpre, dwpost and dgate over the rows in row order,
// and each CTA leaves its part of da.
template <typename TR, typename T>
__global__ void __launch_bounds__(kThreads)
    norm_columns_kernel(NormArgs a, NormGrads g, const float* __restrict__ stats, T* dpre,
                        T* dpost, T* dgate, float* __restrict__ da_parts) {
  const int64_t c = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x;
  const float scale = a.scale_ptr != nullptr ? *a.scale_ptr : a.scale;
  float spre = 0.0f, spost = 0.0f, sgate = 0.0f, sda[1] = {};
  if (c < a.width) {
    const T* post = static_cast<const T*>(a.post_weight);
    const float wpost = post != nullptr ? to_float(post[c]) : 1.0f;
    for (int64_t row = 0; row < a.rows; ++row) {
      const float r = to_float(static_cast<const TR*>(a.residual)[row * a.residual_stride + c]);
      const float ib = stats[2 * row], it = stats[2 * row + 1];
      const float dt = g.dt[row * a.width + c];
      const int64_t group = row / a.gate_rows;
      const float gate = a.gate != nullptr ? to_float(static_cast<const T*>(a.gate)[group * a.width + c]) : 1.0f;
      float bh = 0.0f;
      if (a.branch != nullptr) bh = to_float(static_cast<const T*>(a.branch)[row * a.branch_stride + c]) * ib;
      if (g.normed != nullptr)
        spre += to_float(static_cast<const T*>(g.normed)[row * g.normed_stride + c]) *
                ((scale * r + gate * bh * wpost) * it);
      spost += dt * gate * bh;
      sgate += dt * bh * wpost;
      sda[0] += dt * r;
      if (dgate != nullptr && (row + 1 == a.rows || (row + 1) / a.gate_rows != group)) {
        dgate[group * a.width + c] = from_float<T>(sgate);
        sgate = 0.0f;
      }
    }
    if (dpre != nullptr) dpre[c] = from_float<T>(spre);
    if (dpost != nullptr) dpost[c] = from_float<T>(spost);
    if (dgate != nullptr && a.rows == 0) dgate[c] = from_float<T>(0.0f);
  }
  block_sum(sda);
  if (threadIdx.x == 0) da_parts[blockIdx.x] = sda[0];
}

__global__ void sum_parts_kernel(const float* __restrict__ parts, int64_t count, float* out) {
  double s = 0.0;
  for (int64_t i = 0; i < count; ++i) s += parts[i];
  *out = static_cast<float>(s);
}

NormArgs arguments(const fhb_norm_problem& p) {
  return {p.residual, p.branch, p.pre_weight, p.post_weight, p.gate, p.rows, p.width,
          p.residual_stride, p.branch_stride, p.gate != nullptr ? p.gate_rows : (p.rows > 0 ? p.rows : 1),
          p.residual_scale_ptr, p.residual_scale, p.eps};
}

template <typename TR, typename T>
cudaError_t forward(const fhb_norm_problem& p, void* total, void* normed, float* stats,
                    const DeviceInfo& dev, cudaStream_t stream) {
  const int64_t most = 8ll * dev.sms;
  norm_kernel<TR, T><<<static_cast<unsigned>(p.rows < most ? p.rows : most), kThreads, 0, stream>>>(
      arguments(p), static_cast<TR*>(total), static_cast<T*>(normed), stats);
  return cudaGetLastError();
}

template <typename TR, typename T>
cudaError_t backward(const fhb_norm_problem& p, const NormGrads& g, const fhb_norm_grads& out,
                     const float* stats, float* parts, const DeviceInfo& dev, cudaStream_t stream) {
  const int64_t most = 8ll * dev.sms;
  if (p.rows > 0)
    norm_backward_kernel<TR, T><<<static_cast<unsigned>(p.rows < most ? p.rows : most), kThreads, 0, stream>>>(
        arguments(p), g, stats);
  const int64_t blocks = (p.width + kThreads - 1) / kThreads;
  norm_columns_kernel<TR, T><<<static_cast<unsigned>(blocks), kThreads, 0, stream>>>(
      arguments(p), g, stats, static_cast<T*>(out.pre_weight), static_cast<T*>(out.post_weight),
      static_cast<T*>(out.gate), parts);
  if (out.residual_scale != nullptr)
    sum_parts_kernel<<<1, 1, 0, stream>>>(parts, blocks, out.residual_scale);
  return cudaGetLastError();
}

int64_t parts_bytes(const fhb_norm_problem& p) {
  return ((p.width + kThreads - 1) / kThreads * 4 + 15) & ~15ll;
}

}  // namespace

cudaError_t launch_residual_norm(const fhb_norm_problem& p, void* total, void* normed,
                                 float* stats, const DeviceInfo& dev, cudaStream_t stream) {
  if (p.residual_dtype == FHB_DTYPE_F32)
    return p.dtype == FHB_DTYPE_F32 ? forward<float, float>(p, total, normed, stats, dev, stream)
                                    : forward<float, bf16>(p, total, normed, stats, dev, stream);
  return forward<bf16, bf16>(p, total, normed, stats, dev, stream);
}

size_t residual_norm_workspace_bytes(const fhb_norm_problem& p, const DeviceInfo&) {
  return parts_bytes(p) + p.rows * p.width * 4;
}

cudaError_t launch_residual_norm_backward(const fhb_norm_problem& p, const void* grad_total,
                                          int64_t grad_total_stride, const void* grad_normed,
                                          int64_t grad_normed_stride, const float* stats,
                                          const fhb_norm_grads& out, void* workspace,
                                          const DeviceInfo& dev, cudaStream_t stream) {
  float* parts = static_cast<float*>(workspace);
  const NormGrads g{grad_total, grad_normed, grad_total_stride, grad_normed_stride, out.residual,
                    out.branch,
                    reinterpret_cast<float*>(static_cast<char*>(workspace) + parts_bytes(p))};
  if (p.residual_dtype == FHB_DTYPE_F32)
    return p.dtype == FHB_DTYPE_F32 ? backward<float, float>(p, g, out, stats, parts, dev, stream)
                                    : backward<float, bf16>(p, g, out, stats, parts, dev, stream);
  return backward<bf16, bf16>(p, g, out, stats, parts, dev, stream);
}

}  // namespace fhb
