// extern "C" entry points of the gated residual trunk's operators (include/fused_hoad_b200.h):
// argument validation before any device work, then the launchers of blocks.cuh.
#include <cmath>

#include "blocks.cuh"

namespace {

constexpr int64_t kMaxRows = int64_t{1} << 30;    // rows of an activation
constexpr int64_t kMaxColumns = int64_t{1} << 22;  // values of a row
constexpr int64_t kMaxNormWidth = 32768;         // values of a row that a CTA can hold
constexpr uintptr_t kRoomAlignment = 128;         // of workspaces and saved buffers
constexpr int64_t kMaxCount = int64_t{1} << 40;   // values of a tensor

bool valid_dtype(int dtype) { return dtype == FHB_DTYPE_F32 || dtype == FHB_DTYPE_BF16; }

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

// A matrix of rows x columns with a row stride: given (unless empty), long enough, aligned.
int check_matrix(const void* p, int64_t rows, int64_t columns, int64_t stride, int dtype) {
  if (rows == 0) return FHB_OK;
  if (p == nullptr || stride < columns) return FHB_ERR_INVALID_ARGUMENT;
  if (stride > kMaxCount / rows) return FHB_ERR_TOO_LARGE;
  return aligned(p, fhb::dtype_bytes(dtype)) ? FHB_OK : FHB_ERR_MISALIGNED;
}

int check_vector(const void* p, int dtype, bool required) {
  if (p == nullptr) return required ? FHB_ERR_INVALID_ARGUMENT : FHB_OK;
  return aligned(p, fhb::dtype_bytes(dtype)) ? FHB_OK : FHB_ERR_MISALIGNED;
}

int check_workspace(const void* workspace, size_t bytes, size_t need) {
  if (need == 0) return FHB_OK;
  if (workspace == nullptr || bytes < need) return FHB_ERR_WORKSPACE;
  return aligned(workspace, kRoomAlignment) ? FHB_OK : FHB_ERR_MISALIGNED;
}

// The first code that is not FHB_OK.
template <typename... Codes>
int first_of(Codes... codes) {
  int result = FHB_OK;
  ((result = result == FHB_OK ? codes : result), ...);
  return result;
}

int check_ffn_sizes(const fhb_ffn_problem* p) {
  if (p == nullptr || !valid_dtype(p->dtype) ||
      (p->activation != FHB_ACTIVATION_TANH && p->activation != FHB_ACTIVATION_SILU) ||
      p->tokens < 0 || p->width < 1 || p->hidden < 1 || p->out_width < 1)
    return FHB_ERR_INVALID_ARGUMENT;
  if (p->tokens > kMaxRows || p->width > kMaxColumns || p->hidden > kMaxColumns ||
      p->out_width > kMaxColumns || p->tokens * p->hidden > kMaxCount ||
      p->tokens * p->width > kMaxCount || p->tokens * p->out_width > kMaxCount ||
      p->hidden * p->width > kMaxCount || p->hidden * p->out_width > kMaxCount)
    return FHB_ERR_TOO_LARGE;
  return FHB_OK;
}

int check_ffn(const fhb_ffn_problem* p) {
  const int code = check_ffn_sizes(p);
  if (code != FHB_OK) return code;
  return first_of(check_matrix(p->x, p->tokens, p->width, p->x_stride, p->dtype),
                  check_matrix(p->w_gate, p->hidden, p->width, p->w_gate_stride, p->dtype),
                  check_matrix(p->w_up, p->hidden, p->width, p->w_up_stride, p->dtype),
                  check_matrix(p->w_down, p->out_width, p->hidden, p->w_down_stride, p->dtype),
                  check_vector(p->b_gate, p->dtype, false), check_vector(p->b_up, p->dtype, false),
                  check_vector(p->b_down, p->dtype, false));
}

int check_norm_sizes(const fhb_norm_problem* p) {
  if (p == nullptr || !valid_dtype(p->dtype) || !valid_dtype(p->residual_dtype) ||
      (p->residual_dtype == FHB_DTYPE_BF16 && p->dtype == FHB_DTYPE_F32) || p->rows < 0 ||
      p->width < 1 || !(p->eps >= 0.0f) ||
      (p->branch == nullptr && p->rows > 0 && (p->gate != nullptr || p->post_weight != nullptr)) ||
      (p->gate != nullptr && p->gate_rows < 1))
    return FHB_ERR_INVALID_ARGUMENT;
  return p->rows > kMaxRows || p->width > kMaxNormWidth ? FHB_ERR_TOO_LARGE : FHB_OK;
}

int check_norm(const fhb_norm_problem* p) {
  const int code = check_norm_sizes(p);
  if (code != FHB_OK) return code;
  return first_of(
      check_matrix(p->residual, p->rows, p->width, p->residual_stride, p->residual_dtype),
      p->branch == nullptr ? FHB_OK
                           : check_matrix(p->branch, p->rows, p->width, p->branch_stride, p->dtype),
      check_vector(p->pre_weight, p->dtype, true), check_vector(p->post_weight, p->dtype, false),
      check_vector(p->gate, p->dtype, false),
      check_vector(p->residual_scale_ptr, FHB_DTYPE_F32, false));
}

}  // namespace

extern "C" {

size_t fhb_ffn_saved_bytes(const fhb_ffn_problem* problem) {
  return check_ffn_sizes(problem) == FHB_OK ? fhb::ffn_saved_bytes(*problem) : 0;
}

size_t fhb_ffn_workspace_bytes(const fhb_ffn_problem* problem, int pass) {
  const fhb::DeviceInfo* dev = nullptr;
  if (check_ffn_sizes(problem) != FHB_OK || pass < FHB_FFN_FORWARD || pass > FHB_FFN_FORWARD_SAVING ||
      fhb::current_device_info(&dev) != FHB_OK)
    return 0;
  return fhb::ffn_workspace_bytes(*problem, pass, *dev);
}

int fhb_ffn_forward(const fhb_ffn_problem* problem, void* y, void* saved, void* workspace,
                    size_t workspace_bytes, fhb_stream_t stream) {
  int code = check_ffn(problem);
  if (code != FHB_OK) return code;
  if (problem->tokens == 0) return FHB_OK;
  code = check_vector(y, problem->dtype, true);
  if (code != FHB_OK) return code;
  if (!aligned(saved, kRoomAlignment)) return FHB_ERR_MISALIGNED;
  const fhb::DeviceInfo* dev = nullptr;
  code = fhb::current_device_info(&dev);
  if (code != FHB_OK) return code;
  const int pass = saved != nullptr ? FHB_FFN_FORWARD_SAVING : FHB_FFN_FORWARD;
  code = check_workspace(workspace, workspace_bytes, fhb::ffn_workspace_bytes(*problem, pass, *dev));
  if (code != FHB_OK) return code;
  return fhb::record_cuda_error(
      fhb::launch_ffn_forward(*problem, y, saved, workspace, *dev, stream));
}

int fhb_ffn_backward(const fhb_ffn_problem* problem, const void* grad_y, int64_t grad_y_stride,
                     const void* saved, const fhb_ffn_grads* grads, void* workspace,
                     size_t workspace_bytes, fhb_stream_t stream) {
  int code = check_ffn(problem);
  if (code != FHB_OK) return code;
  if (grads == nullptr) return FHB_ERR_INVALID_ARGUMENT;
  const int dtype = problem->dtype;
  code = first_of(
      check_matrix(grad_y, problem->tokens, problem->out_width, grad_y_stride, dtype),
      check_vector(grads->x, dtype, false), check_vector(grads->w_gate, dtype, false),
      check_vector(grads->w_up, dtype, false), check_vector(grads->w_down, dtype, false),
      check_vector(grads->b_gate, dtype, false), check_vector(grads->b_up, dtype, false),
      check_vector(grads->b_down, dtype, false));
  if (code != FHB_OK) return code;
  if (problem->tokens > 0 && saved == nullptr) return FHB_ERR_INVALID_ARGUMENT;
  if (!aligned(saved, kRoomAlignment)) return FHB_ERR_MISALIGNED;
  const fhb::DeviceInfo* dev = nullptr;
  code = fhb::current_device_info(&dev);
  if (code != FHB_OK) return code;
  code = check_workspace(workspace, workspace_bytes, fhb::ffn_workspace_bytes(*problem, FHB_FFN_BACKWARD, *dev));
  if (code != FHB_OK) return code;
  return fhb::record_cuda_error(fhb::launch_ffn_backward(*problem, grad_y, grad_y_stride, saved,
                                                         *grads, workspace, *dev, stream));
}

int fhb_residual_norm(const fhb_norm_problem* problem, void* total, void* normed, float* stats,
                      fhb_stream_t stream) {
  int code = check_norm(problem);
  if (code != FHB_OK) return code;
  if (problem->rows == 0) return FHB_OK;
  code = first_of(check_vector(total, problem->residual_dtype, false),
                  check_vector(normed, problem->dtype, true),
                  check_vector(stats, FHB_DTYPE_F32, false));
  if (code != FHB_OK) return code;
  const fhb::DeviceInfo* dev = nullptr;
  code = fhb::current_device_info(&dev);
  if (code != FHB_OK) return code;
  return fhb::record_cuda_error(
      fhb::launch_residual_norm(*problem, total, normed, stats, *dev, stream));
}

size_t fhb_residual_norm_workspace_bytes(const fhb_norm_problem* problem) {
  const fhb::DeviceInfo* dev = nullptr;
  if (check_norm_sizes(problem) != FHB_OK || fhb::current_device_info(&dev) != FHB_OK) return 0;
  return fhb::residual_norm_workspace_bytes(*problem, *dev);
}

int fhb_residual_norm_backward(const fhb_norm_problem* problem, const void* grad_total,
                               int64_t grad_total_stride, const void* grad_normed,
                               int64_t grad_normed_stride, const float* stats,
                               const fhb_norm_grads* grads, void* workspace,
                               size_t workspace_bytes, fhb_stream_t stream) {
  int code = check_norm(problem);
  if (code != FHB_OK) return code;
  if (grads == nullptr || (problem->rows > 0 && stats == nullptr) ||
      (grads->branch != nullptr && problem->rows > 0 && problem->branch == nullptr) ||
      (grads->gate != nullptr && problem->gate == nullptr) ||
      (grads->post_weight != nullptr && problem->post_weight == nullptr))
    return FHB_ERR_INVALID_ARGUMENT;
  const int64_t rows = problem->rows, width = problem->width;
  code = first_of(
      grad_total == nullptr ? FHB_OK
                            : check_matrix(grad_total, rows, width, grad_total_stride, problem->residual_dtype),
      grad_normed == nullptr ? FHB_OK
                             : check_matrix(grad_normed, rows, width, grad_normed_stride, problem->dtype),
      check_vector(stats, FHB_DTYPE_F32, false),
      check_vector(grads->residual, problem->residual_dtype, false),
      check_vector(grads->branch, problem->dtype, false),
      check_vector(grads->pre_weight, problem->dtype, false),
      check_vector(grads->post_weight, problem->dtype, false),
      check_vector(grads->gate, problem->dtype, false),
      check_vector(grads->residual_scale, FHB_DTYPE_F32, false));
  if (code != FHB_OK) return code;
  const fhb::DeviceInfo* dev = nullptr;
  code = fhb::current_device_info(&dev);
  if (code != FHB_OK) return code;
  code = check_workspace(workspace, workspace_bytes, fhb::residual_norm_workspace_bytes(*problem, *dev));
  if (code != FHB_OK) return code;
  return fhb::record_cuda_error(fhb::launch_residual_norm_backward(
      *problem, grad_total, grad_total_stride, grad_normed, grad_normed_stride, stats, *grads,
      workspace, *dev, stream));
}

int fhb_debug_staged_wait_selftest(const float* rows, float* out, fhb_stream_t stream) {
  if (rows == nullptr || out == nullptr) return FHB_ERR_INVALID_ARGUMENT;
  if (!aligned(rows, 16) || !aligned(out, 4)) return FHB_ERR_MISALIGNED;
  const fhb::DeviceInfo* dev = nullptr;
  const int code = fhb::current_device_info(&dev);
  if (code != FHB_OK) return code;
  return fhb::record_cuda_error(fhb::launch_staged_wait_selftest(rows, out, *dev, stream));
}

int fhb_adamw_step(const fhb_adamw_tensor* tensors, int64_t n_tensors, int state_bits,
                   int64_t* step, double lr, double beta1, double beta2, double eps,
                   double weight_decay, fhb_stream_t stream) {
  if (n_tensors < 0 || (n_tensors > 0 && tensors == nullptr) || step == nullptr ||
      (state_bits != 8 && state_bits != 32) || !(lr >= 0.0) || !(beta1 >= 0.0 && beta1 < 1.0) ||
      !(beta2 >= 0.0 && beta2 < 1.0) || !(eps >= 0.0) || !(weight_decay >= 0.0))
    return FHB_ERR_INVALID_ARGUMENT;
  if (!aligned(step, 8)) return FHB_ERR_MISALIGNED;
  for (int64_t i = 0; i < n_tensors; ++i) {
    const fhb_adamw_tensor& t = tensors[i];
    if (t.count < 0 || !valid_dtype(t.dtype)) return FHB_ERR_INVALID_ARGUMENT;
    if (t.count > kMaxCount) return FHB_ERR_TOO_LARGE;
    if (t.count == 0) continue;
    const int code = first_of(
        check_vector(t.param, t.dtype, true), check_vector(t.grad, t.dtype, true),
        state_bits == 8 ? FHB_OK : check_vector(t.exp_avg, FHB_DTYPE_F32, true),
        state_bits == 8 ? FHB_OK : check_vector(t.exp_avg_sq, FHB_DTYPE_F32, true),
        check_vector(t.exp_avg_scale, FHB_DTYPE_F32, state_bits == 8),
        check_vector(t.exp_avg_sq_scale, FHB_DTYPE_F32, state_bits == 8));
    if (code != FHB_OK) return code;
    if (t.exp_avg == nullptr || t.exp_avg_sq == nullptr) return FHB_ERR_INVALID_ARGUMENT;
  }
  const fhb::DeviceInfo* dev = nullptr;
  const int code = fhb::current_device_info(&dev);
  if (code != FHB_OK) return code;
  return fhb::record_cuda_error(fhb::launch_adamw(tensors, n_tensors, state_bits, step, lr, beta1,
                                                  beta2, eps, weight_decay, *dev, stream));
}

}  // extern "C"
