// The gated feed-forward block: g = x Wg^T + bg, u = x Wu^T + bu, h = act(g) u,
// y = h Wd^T + bd, and its gradients
//     dh = dy Wd,  du = dh act(g),  dg = dh u act'(g),
//     dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x,  dWd = dy^T h,  db = column sums.
//
// Two products forward (both projections, the activation and the gate in the first), four
// backward (dg and du in the first; dx as one sum over both weights; dWg and dWu in one launch),
// on the tensor cores (gemm_tc.cu).
#include <algorithm>

#include "common.cuh"
#include "gated_ffn.cuh"
#include "gemm_tc.cuh"

namespace fhb {
namespace {

int64_t round_up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

// Pieces of one buffer, 128-byte aligned; without a buffer it only counts.
struct Room {
  char* base;
  size_t used = 0;
  void* take(size_t bytes) {
    void* p = base != nullptr ? base + used : nullptr;
    used += static_cast<size_t>(round_up(static_cast<int64_t>(bytes), 128));
    return p;
  }
};

// What the forward makes: h in operand form, and for a backward the activation's factors.
struct Saved {
  TcMatrix h;
  TcFactors factors;
};
Saved saved_in(const fhb_ffn_problem& p, Room& room, bool keep) {
  Saved s;
  s.h = tc_result(room.take(tc_result_bytes(p.tokens, p.hidden, p.dtype)), p.tokens, p.hidden, p.dtype);
  if (keep)
    s.factors = tc_factors(room.take(tc_factor_bytes(p.tokens, p.hidden, p.dtype)), p.tokens, p.hidden, p.dtype);
  return s;
}

// ---- column sums (the biases' gradients) ----
// dg's and du's come as sums over 32 rows from the product that makes them, dy's from itself.
// One part: 64 columns of up to part_rows rows over 8 warps; then the parts, in order.
struct ColumnSource {
  const void* p;
  int64_t stride, columns, rows;
  bool sums;  // FP32 sums, else values of the block's type
  void* out;
};
struct ColumnSources {
  ColumnSource source[3];
  int64_t part_rows, part_count, widest;
  float* parts;  // [source][part][widest]
};
// Rows of one part: 256, more where there would be over 1,024 parts.
int64_t part_rows_of(int64_t rows) { return std::max<int64_t>(256, (rows + 1023) / 1024); }

template <typename S>
__device__ __forceinline__ void add_rows(const S* p, int64_t stride, int64_t first, int64_t last,
                                         const int64_t (&c)[2], int64_t columns, float (&sum)[2]) {
  int64_t r = first;
  for (; r + 56 < last; r += 64) {  // eight rows in flight
    float v[8][2];
#pragma unroll
    for (int k = 0; k < 8; ++k)
#pragma unroll
      for (int j = 0; j < 2; ++j) v[k][j] = c[j] < columns ? to_float(p[(r + 8 * k) * stride + c[j]]) : 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k)
#pragma unroll
      for (int j = 0; j < 2; ++j) sum[j] += v[k][j];
  }
  for (; r < last; r += 8)
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (c[j] < columns) sum[j] += to_float(p[r * stride + c[j]]);
}

template <typename T>
__global__ void __launch_bounds__(256) column_parts_kernel(const __grid_constant__ ColumnSources s) {
  allow_dependents();
  wait_for_prerequisites();
  const ColumnSource& src = s.source[blockIdx.z];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int64_t c0 = blockIdx.x * 64ll, c[2] = {c0 + lane, c0 + lane + 32};
  if (c0 >= src.columns) return;
  const int64_t first = blockIdx.y * s.part_rows, last = min(first + s.part_rows, src.rows);
  float sum[2] = {};
  if (src.sums)
    add_rows(static_cast<const float*>(src.p), src.stride, first + warp, last, c, src.columns, sum);
  else
    add_rows(static_cast<const T*>(src.p), src.stride, first + warp, last, c, src.columns, sum);
  __shared__ float by_warp[8][64];
  by_warp[warp][lane] = sum[0];
  by_warp[warp][lane + 32] = sum[1];
  __syncthreads();
  if (threadIdx.x < 64 && c0 + threadIdx.x < src.columns) {
    float total = 0.0f;
    for (int w = 0; w < 8; ++w) total += by_warp[w][threadIdx.x];
    s.parts[(blockIdx.z * s.part_count + blockIdx.y) * s.widest + c0 + threadIdx.x] = total;
  }
}

template <typename T>
__global__ void __launch_bounds__(256) column_totals_kernel(const __grid_constant__ ColumnSources s) {
  allow_dependents();
  wait_for_prerequisites();
  const ColumnSource& src = s.source[blockIdx.y];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int64_t c = blockIdx.x * 32ll + lane;
  const int64_t parts = (src.rows + s.part_rows - 1) / s.part_rows;
  float total = 0.0f;
  if (c < src.columns) {
    const float* in = s.parts + blockIdx.y * s.part_count * s.widest + c;
    int64_t part = warp;
    for (; part + 56 < parts; part += 64) {  // eight parts in flight
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = in[(part + 8 * k) * s.widest];
#pragma unroll
      for (int k = 0; k < 8; ++k) total += v[k];
    }
    for (; part < parts; part += 8) total += in[part * s.widest];
  }
  __shared__ float by_warp[8][32];
  by_warp[warp][lane] = total;
  __syncthreads();
  if (warp != 0 || c >= src.columns) return;
  total = 0.0f;
  for (int w = 0; w < 8; ++w) total += by_warp[w][lane];
  static_cast<T*>(src.out)[c] = from_float<T>(total);
}

template <typename T>
cudaError_t column_sums(const ColumnSources& s, int count, cudaStream_t stream) {
  if (count == 0) return cudaSuccess;
  const cudaError_t e = launch_dependent(
      column_parts_kernel<T>, dim3(static_cast<unsigned>((s.widest + 63) / 64),
                                   static_cast<unsigned>(s.part_count), count),
      dim3(256), 0, stream, s);
  if (e != cudaSuccess) return e;
  return launch_dependent(column_totals_kernel<T>,
                          dim3(static_cast<unsigned>((s.widest + 31) / 32), count), dim3(256), 0,
                          stream, s);
}

// ---- the products ----
struct Operands {
  TcMatrix x, w_gate, w_up, w_down, dy;
};

// Operand forms of the inputs; those that have to be copied take their place in `room`.
struct Inputs {
  TcInput in[5];
  TcMatrix out[5];
};
Inputs inputs_in(const fhb_ffn_problem& p, const void* dy, int64_t dy_stride, Room& room, Operands& o) {
  Inputs x{{{p.x, p.tokens, p.width, p.x_stride},
            {p.w_gate, p.hidden, p.width, p.w_gate_stride},
            {p.w_up, p.hidden, p.width, p.w_up_stride},
            {p.w_down, p.out_width, p.hidden, p.w_down_stride},
            {dy, p.tokens, p.out_width, dy_stride}}, {}};
  TcMatrix* const to[] = {&o.x, &o.w_gate, &o.w_up, &o.w_down, &o.dy};
  for (int i = 0; i < 5; ++i) {
    if (x.in[i].p == nullptr) continue;
    void* place = room.take(tc_operand_bytes(x.in[i], p.dtype));
    *to[i] = x.out[i] = tc_operand(x.in[i], p.dtype, place);
  }
  return x;
}

TcProduct gate_product(const fhb_ffn_problem& p, const Operands& o, const Saved& s) {
  TcProduct q;
  q.m = p.tokens, q.n = p.hidden, q.k = p.width;
  q.a[0] = o.x, q.b[0] = o.w_gate, q.b[1] = o.w_up;
  q.epilogue = TcEpilogue::kGate;
  q.dtype = p.dtype;
  q.bias[0] = p.b_gate, q.bias[1] = p.b_up;
  q.gated[0] = s.h;
  q.factors = s.factors;
  q.activation = p.activation;
  return q;
}

TcProduct store_product(const fhb_ffn_problem& p, int64_t m, int64_t n, int64_t k, void* out) {
  TcProduct q;
  q.m = m, q.n = n, q.k = k;
  q.dtype = p.dtype;
  q.out[0] = out;
  q.out_stride = n;
  return q;
}

TcProduct down_product(const fhb_ffn_problem& p, const Operands& o, const Saved& s, void* y) {
  TcProduct q = store_product(p, p.tokens, p.out_width, p.hidden, y);
  q.a[0] = s.h, q.b[0] = o.w_down;
  q.bias[0] = p.b_down;
  return q;
}

struct Backward {
  TcMatrix dg, du;
  TcProduct hidden;
  TcProduct rest[kTcMaxProducts];  // the projections', w_down's and x's gradients
};
Backward backward_of(const fhb_ffn_problem& p, const Operands& o, const Saved& s,
                     const fhb_ffn_grads& out, Room& room) {
  Backward b;
  const size_t bytes = tc_result_bytes(p.tokens, p.hidden, p.dtype);
  b.dg = tc_result(room.take(bytes), p.tokens, p.hidden, p.dtype);
  b.du = tc_result(room.take(bytes), p.tokens, p.hidden, p.dtype);
  b.hidden = store_product(p, p.tokens, p.hidden, p.out_width, nullptr);
  b.hidden.a[0] = o.dy, b.hidden.b[0] = o.w_down;
  b.hidden.b_k_major = false;
  b.hidden.epilogue = TcEpilogue::kGateGrad;
  b.hidden.gated[0] = b.dg, b.hidden.gated[1] = b.du;
  b.hidden.factors = s.factors;
  if (out.b_gate != nullptr || out.b_up != nullptr) {
    b.hidden.row_sums_stride = round_up(p.hidden, 32);
    b.hidden.row_sums = static_cast<float*>(room.take(
        static_cast<size_t>((p.tokens + 31) / 32 * 2 * b.hidden.row_sums_stride * 4)));
  }
  // the long sums over the tokens first: in one launch their items are its longest
  TcProduct &weights = b.rest[0], &down = b.rest[1], &x = b.rest[2];
  weights = store_product(p, p.hidden, p.width, p.tokens, out.w_gate);
  weights.out[1] = out.w_up;
  weights.groups = 2;
  weights.a[0] = b.dg, weights.a[1] = b.du, weights.b[0] = o.x;
  weights.a_k_major = weights.b_k_major = false;
  down = store_product(p, p.out_width, p.hidden, p.tokens, out.w_down);
  down.a[0] = o.dy, down.b[0] = s.h;
  down.a_k_major = down.b_k_major = false;
  x = store_product(p, p.tokens, p.width, p.hidden, out.x);
  x.a[0] = b.dg, x.a[1] = b.du, x.b[0] = o.w_gate, x.b[1] = o.w_up;
  x.b_k_major = false;
  x.sum_terms = 2;
  return b;
}

// Stands for "every gradient wanted" where sizes are asked for before the outputs exist.
fhb_ffn_grads all_grads() {
  static char any;
  return {&any, &any, &any, &any, &any, &any, &any};
}

int64_t column_part_count(const fhb_ffn_problem& p) {
  const int64_t rows = part_rows_of(p.tokens);
  return (p.tokens + rows - 1) / rows;
}

size_t column_bytes(const fhb_ffn_problem& p) {
  return static_cast<size_t>(3 * column_part_count(p) * std::max(p.hidden, p.out_width) * 4);
}

}  // namespace

size_t ffn_saved_bytes(const fhb_ffn_problem& p) {
  Room room{nullptr};
  saved_in(p, room, true);
  return room.used;
}

size_t ffn_workspace_bytes(const fhb_ffn_problem& p, int pass, const DeviceInfo& dev) {
  Room room{nullptr};
  Operands o;
  if (p.tokens == 0) return 0;
  if (pass != FHB_FFN_BACKWARD) {
    const bool keep = pass == FHB_FFN_FORWARD_SAVING;
    inputs_in(p, nullptr, 0, room, o);
    Room aside{nullptr};
    const Saved s = saved_in(p, keep ? aside : room, keep);
    const TcProduct down = down_product(p, o, s, nullptr);
    room.take(gemm_tc_workspace_bytes(&down, 1, dev));
    return !keep && ffn_takes_small(p) ? ffn_small_bytes(p) : room.used;
  }
  // the upstream gradient may need a copy: the size asked for does not depend on it
  inputs_in(p, nullptr, 0, room, o);
  room.take(tc_result_bytes(p.tokens, p.out_width, p.dtype));
  Room aside{nullptr};
  const Saved s = saved_in(p, aside, true);
  const Backward b = backward_of(p, o, s, all_grads(), room);
  room.take(column_bytes(p));
  room.take(gemm_tc_workspace_bytes(b.rest, kTcMaxProducts, dev));
  return room.used;
}

cudaError_t launch_ffn_forward(const fhb_ffn_problem& p, void* y, void* saved, void* workspace,
                               const DeviceInfo& dev, cudaStream_t stream) {
  if (saved == nullptr && ffn_takes_small(p))
    return launch_ffn_small(p, y, workspace, dev, stream);
  Room room{static_cast<char*>(workspace)}, kept{static_cast<char*>(saved)};
  Operands o;
  const Inputs x = inputs_in(p, nullptr, 0, room, o);
  bool packed = false;
  cudaError_t e = launch_pack(x.in, x.out, 5, p.dtype, &packed, stream);
  if (e != cudaSuccess) return e;
  const Saved s = saved_in(p, saved != nullptr ? kept : room, saved != nullptr);
  const TcProduct gate = gate_product(p, o, s);
  e = launch_gemm_tc(&gate, 1, nullptr, packed, dev, stream);
  if (e != cudaSuccess) return e;
  const TcProduct down = down_product(p, o, s, y);
  return launch_gemm_tc(&down, 1, room.take(0), true, dev, stream);
}

cudaError_t launch_ffn_backward(const fhb_ffn_problem& p, const void* grad_y, int64_t grad_y_stride,
                                const void* saved, const fhb_ffn_grads& out, void* workspace,
                                const DeviceInfo& dev, cudaStream_t stream) {
  const size_t size = dtype_bytes(p.dtype);
  if (p.tokens == 0) {
    const struct {
      void* p;
      int64_t count;
    } zero[] = {{out.w_gate, p.hidden * p.width}, {out.w_up, p.hidden * p.width},
                {out.w_down, p.out_width * p.hidden}, {out.b_gate, p.hidden}, {out.b_up, p.hidden},
                {out.b_down, p.out_width}};
    for (const auto& z : zero) {
      if (z.p == nullptr) continue;
      const cudaError_t e = cudaMemsetAsync(z.p, 0, z.count * size, stream);
      if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
  }
  Room room{static_cast<char*>(workspace)}, kept{static_cast<char*>(const_cast<void*>(saved))};
  Operands o;
  const Inputs x = inputs_in(p, grad_y, grad_y_stride, room, o);
  bool packed = false;
  cudaError_t e = launch_pack(x.in, x.out, 5, p.dtype, &packed, stream);
  if (e != cudaSuccess) return e;
  const Saved s = saved_in(p, kept, true);
  const Backward b = backward_of(p, o, s, out, room);
  float* column_parts = static_cast<float*>(room.take(column_bytes(p)));
  void* sums = room.take(0);  // the rest
  e = launch_gemm_tc(&b.hidden, 1, nullptr, packed, dev, stream);
  if (e == cudaSuccess) e = launch_gemm_tc(b.rest, kTcMaxProducts, sums, true, dev, stream);
  if (e != cudaSuccess) return e;
  ColumnSources columns{};
  int count = 0;
  const int64_t row_sums = (p.tokens + 31) / 32, sums_stride = b.hidden.row_sums_stride;
  if (out.b_gate != nullptr)
    columns.source[count++] = {b.hidden.row_sums, 2 * sums_stride, p.hidden, row_sums, true, out.b_gate};
  if (out.b_up != nullptr)
    columns.source[count++] = {b.hidden.row_sums + sums_stride, 2 * sums_stride, p.hidden, row_sums, true, out.b_up};
  if (out.b_down != nullptr)
    columns.source[count++] = {grad_y, grad_y_stride, p.out_width, p.tokens, false, out.b_down};
  columns.part_rows = part_rows_of(p.tokens);
  columns.part_count = column_part_count(p);
  columns.widest = std::max(p.hidden, p.out_width);
  columns.parts = column_parts;
  return p.dtype == FHB_DTYPE_F32 ? column_sums<float>(columns, count, stream)
                                  : column_sums<bf16>(columns, count, stream);
}

}  // namespace fhb
