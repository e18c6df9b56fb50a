// Matrix products on the tensor cores for the gated feed-forward block: operands, the plan of a
// product and its launcher (gemm_tc.cu).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "blocks.cuh"

namespace fhb {

// A bf16 matrix in memory, rows x columns, rows `stride` elements apart (a multiple of 8, base
// 16-byte aligned: what a TMA tile copy needs). An FP32 matrix is three such planes whose sum
// it is (split_pair in gemm_tc.cu), `plane` elements apart.
struct TcMatrix {
  const bf16* p = nullptr;
  int64_t rows = 0, cols = 0, stride = 0, plane = 0;
  int planes = 1;
};

// What a product does with its sums.
enum class TcEpilogue {
  kStore,     // out[m][n] = sum + bias[n], in the output type (or FP32 sums of one part of K into
              // the workspace, added up by a second kernel)
  kGate,      // two products g, u side by side: h = act(g) u, and what the backward needs
  kGateGrad,  // the gradients of g and u from that of h
};

// What the forward keeps of the activation for the backward, for 16 consecutive hidden features
// of one token: f1 = act(g) and f2 = u act'(g), so that du = dh f1 and dg = dh f2.
// bf16 block: f16 values times one power of 2 for each of the two groups of 16 (an exponent
// byte each), so the range is FP32's and the rounding 2^-12 of the group's largest finite value --
// 16 times below the bf16 rounding of dg and du that follows. FP32 block: FP32 values.
constexpr int kFactorGroup = 16;
struct TcFactors {
  void* values = nullptr;          // [token][group][2][16], __half or float
  unsigned char* exponents = nullptr;  // [token][group][2]
  int64_t groups = 0;
};

// One product, or two of the same shape that share a launch: C[m][n] = sum over terms and k of
// A(m, k) B(n, k). An operand is K-major (memory rows are m or n) or not (memory rows are k).
struct TcProduct {
  int64_t m = 0, n = 0, k = 0;
  TcMatrix a[2], b[2];
  bool a_k_major = true, b_k_major = true;
  int groups = 1;     // 2: A = a[0] or a[1] (B = b[0] in both), results to out[0] and out[1]
  int sum_terms = 1;  // 2: the sum of a[0] b[0] and a[1] b[1]
  TcEpilogue epilogue = TcEpilogue::kStore;
  int dtype = FHB_DTYPE_BF16;  // of the block: the type of out and bias; FP32: three planes
  void* out[2] = {nullptr, nullptr};
  int64_t out_stride = 0;
  const void* bias[2] = {nullptr, nullptr};
  // kGate: h; kGateGrad: dg and du (TcMatrix rows x cols are theirs)
  TcMatrix gated[2];
  TcFactors factors;
  int activation = 0;
  // kGateGrad: the column sums of dg and du over every 32 rows, [m / 32][2][row_sums_stride]
  float* row_sums = nullptr;
  int64_t row_sums_stride = 0;
};

// Products of one call, none of which needs another's result: kGate and kGateGrad alone, up to
// three of kStore. One whose outputs are null is left out, though not of the plan. Short ones go
// into one launch, where their tiles share its rounds of the SMs (training passes, us: 1,000 x 201
// x 533 fp32 87 apart and 67 together, 1,024 x 512 x 2048 bf16 76 and 64); for long ones it makes
// no difference (4,096 x 1024 x 4096) or loses a little, as tiles that drift apart share less in
// L2 (16,384 x 2048 x 5632: 2,780 and 2,817).
constexpr int kTcMaxProducts = 3;
// Workspace of a call: the FP32 partial sums of the parts of K (0 where there is one of each).
size_t gemm_tc_workspace_bytes(const TcProduct* products, int count, const DeviceInfo& dev);
// `dependent`: launched as a dependent of the kernel before it in the stream, which has to be
// one of this file's or gated_ffn.cu's (they wait for their own predecessors, so a chain of them
// keeps its order; the first kernel of a call is an ordinary launch).
cudaError_t launch_gemm_tc(const TcProduct* products, int count, void* workspace, bool dependent,
                           const DeviceInfo& dev, cudaStream_t stream);

// A caller's matrix: `rows` x `cols` elements of the block's type, rows `stride` apart.
struct TcInput {
  const void* p;
  int64_t rows, cols, stride;
};
// The input as tensor-core operand: itself where TMA can copy its tiles, else its copy in `room`
// (bytes: tc_operand_bytes, 0 where no copy is needed), which launch_pack makes.
size_t tc_operand_bytes(const TcInput& in, int dtype);
TcMatrix tc_operand(const TcInput& in, int dtype, void* room);
cudaError_t launch_pack(const TcInput* in, const TcMatrix* out, int count, int dtype,
                        bool* launched, cudaStream_t stream);
// A matrix of the block's type in operand form at `room`, to be written by a product.
size_t tc_result_bytes(int64_t rows, int64_t cols, int dtype);
TcMatrix tc_result(void* room, int64_t rows, int64_t cols, int dtype);
size_t tc_factor_bytes(int64_t tokens, int64_t hidden, int dtype);
TcFactors tc_factors(void* room, int64_t tokens, int64_t hidden, int dtype);

}  // namespace fhb
