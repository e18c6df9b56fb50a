// Torch binding of the gated residual trunk's operators (include/fused_hoad_b200.h): part of
// the module fused_hoad._C. Outputs, workspaces and what the backward keeps come from the ATen
// caching allocator on the current stream, so the ops stay asynchronous and graph-capturable.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_runtime.h>
#include <torch/extension.h>

#include <string>
#include <tuple>
#include <vector>

#include "../../include/fused_hoad_b200.h"

namespace {

using OptionalTensor = c10::optional<torch::Tensor>;

// Numbers go into messages as text: formatting them through a stream crashes in extensions
// built with this toolchain.
std::string text(int64_t n) { return std::to_string(n); }

void check_status(int code, const char* op) {
  if (code == FHB_OK) return;
  if (code == FHB_ERR_CUDA) {
    const auto err = static_cast<cudaError_t>(fhb_last_cuda_error());
    TORCH_CHECK(false, op, " failed: ", fhb_status_string(code), ": ", cudaGetErrorString(err));
  }
  TORCH_CHECK(false, op, " failed: ", fhb_status_string(code));
}

int activation_code(const std::string& activation) {
  if (activation == "tanh") return FHB_ACTIVATION_TANH;
  if (activation == "silu") return FHB_ACTIVATION_SILU;
  TORCH_CHECK(false, "activation must be \"tanh\" or \"silu\"");
  return -1;
}

int dtype_code(const torch::Tensor& t, const char* what) {
  if (t.scalar_type() == torch::kFloat32) return FHB_DTYPE_F32;
  TORCH_CHECK(t.scalar_type() == torch::kBFloat16, what, " must use float32 or bfloat16");
  return FHB_DTYPE_BF16;
}

void check_like(const torch::Tensor& t, const torch::Tensor& like, const char* what,
                const char* like_what) {
  TORCH_CHECK(t.is_cuda(), what, " must be a CUDA tensor");
  TORCH_CHECK(t.device() == like.device(), what, " must be on the same device as ", like_what);
  TORCH_CHECK(t.scalar_type() == like.scalar_type(), what, " must have the type of ", like_what);
}

void check_vector(const torch::Tensor& t, const torch::Tensor& like, int64_t size,
                  const char* what, const char* like_what) {
  check_like(t, like, what, like_what);
  TORCH_CHECK(t.dim() == 1 && t.size(0) == size, what, " must have shape [", text(size), "]");
  TORCH_CHECK(t.is_contiguous(), what, " must be contiguous");
}

// `t` as rows of its last dimension with unit stride: a view where the strides allow it (any
// row stride), else a contiguous copy.
torch::Tensor as_rows(const torch::Tensor& t) {
  torch::Tensor rows = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
  // a row stride below the row's length (an expanded tensor) is no layout of separate rows
  if ((rows.size(1) > 1 && rows.stride(1) != 1) ||
      (rows.size(0) > 1 && rows.stride(0) < rows.size(1)))
    rows = rows.contiguous();
  return rows;
}

int64_t row_stride(const torch::Tensor& rows) {
  return rows.size(0) > 1 ? rows.stride(0) : rows.size(1);
}

torch::Tensor bytes_for(size_t bytes, const torch::Tensor& like) {
  return torch::empty({static_cast<int64_t>(bytes)}, like.options().dtype(torch::kUInt8));
}

void* data_of(const torch::Tensor& t) { return t.numel() ? t.data_ptr() : nullptr; }
void* data_of(const OptionalTensor& t) { return t.has_value() ? t->data_ptr() : nullptr; }

// ---- gated feed-forward block ----

// The problem, and the row views that its pointers belong to.
struct Ffn {
  fhb_ffn_problem problem{};
  torch::Tensor x, w_gate, w_up, w_down;
};

Ffn ffn_of(const torch::Tensor& x, const torch::Tensor& w_gate, const torch::Tensor& w_up,
           const torch::Tensor& w_down, const OptionalTensor& b_gate, const OptionalTensor& b_up,
           const OptionalTensor& b_down, const std::string& activation) {
  const int act = activation_code(activation);
  TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
  const int dtype = dtype_code(x, "x");
  TORCH_CHECK(x.dim() >= 1, "x must have shape [..., width]");
  const int64_t width = x.size(-1);
  TORCH_CHECK(width >= 1, "x must have shape [..., width] with a width of at least 1");
  check_like(w_gate, x, "w_gate", "x");
  check_like(w_up, x, "w_up", "x");
  check_like(w_down, x, "w_down", "x");
  TORCH_CHECK(w_gate.dim() == 2 && w_gate.size(1) == width && w_gate.size(0) >= 1,
              "w_gate must have shape [hidden, ", text(width), "]");
  const int64_t hidden = w_gate.size(0);
  TORCH_CHECK(w_up.dim() == 2 && w_up.size(0) == hidden && w_up.size(1) == width,
              "w_up must have shape [", text(hidden), ", ", text(width), "]");
  TORCH_CHECK(w_down.dim() == 2 && w_down.size(1) == hidden && w_down.size(0) >= 1,
              "w_down must have shape [out_width, ", text(hidden), "]");
  if (b_gate) check_vector(*b_gate, x, hidden, "b_gate", "x");
  if (b_up) check_vector(*b_up, x, hidden, "b_up", "x");
  if (b_down) check_vector(*b_down, x, w_down.size(0), "b_down", "x");
  Ffn f;
  f.x = as_rows(x);
  f.w_gate = as_rows(w_gate);
  f.w_up = as_rows(w_up);
  f.w_down = as_rows(w_down);
  fhb_ffn_problem& p = f.problem;
  p.tokens = f.x.size(0);
  p.width = width;
  p.hidden = hidden;
  p.out_width = w_down.size(0);
  p.dtype = dtype;
  p.activation = act;
  p.x = data_of(f.x);
  p.w_gate = data_of(f.w_gate);
  p.w_up = data_of(f.w_up);
  p.w_down = data_of(f.w_down);
  p.x_stride = row_stride(f.x);
  p.w_gate_stride = row_stride(f.w_gate);
  p.w_up_stride = row_stride(f.w_up);
  p.w_down_stride = row_stride(f.w_down);
  p.b_gate = data_of(b_gate);
  p.b_up = data_of(b_up);
  p.b_down = data_of(b_down);
  return f;
}

// (y [..., out_width], what the backward needs or an empty tensor)
std::tuple<torch::Tensor, torch::Tensor> gated_feed_forward(
    torch::Tensor x, torch::Tensor w_gate, torch::Tensor w_up, torch::Tensor w_down,
    OptionalTensor b_gate, OptionalTensor b_up, OptionalTensor b_down,
    const std::string& activation, bool want_saved) {
  const Ffn f = ffn_of(x, w_gate, w_up, w_down, b_gate, b_up, b_down, activation);
  const c10::cuda::CUDAGuard device_guard(x.device());
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = f.problem.out_width;
  auto y = torch::empty(shape, x.options());
  auto saved = bytes_for(want_saved ? fhb_ffn_saved_bytes(&f.problem) : 0, x);
  if (f.problem.tokens == 0) return {y, saved};
  auto workspace = bytes_for(fhb_ffn_workspace_bytes(&f.problem, 0), x);
  check_status(fhb_ffn_forward(&f.problem, y.data_ptr(), want_saved ? saved.data_ptr() : nullptr,
                               data_of(workspace), static_cast<size_t>(workspace.numel()),
                               at::cuda::getCurrentCUDAStream()),
               "gated_feed_forward");
  return {y, saved};
}

// Gradients of x, w_gate, w_up, w_down, b_gate, b_up, b_down, in that order; an undefined
// tensor (None) where wants[i] is false.
std::vector<OptionalTensor> gated_feed_forward_backward(
    torch::Tensor grad_y, torch::Tensor x, torch::Tensor w_gate, torch::Tensor w_up,
    torch::Tensor w_down, OptionalTensor b_gate, OptionalTensor b_up, OptionalTensor b_down,
    const std::string& activation, torch::Tensor saved, std::vector<bool> wants) {
  const Ffn f = ffn_of(x, w_gate, w_up, w_down, b_gate, b_up, b_down, activation);
  const fhb_ffn_problem& p = f.problem;
  TORCH_CHECK(wants.size() == 7, "wants must have 7 entries");
  check_like(grad_y, x, "grad_y", "x");
  TORCH_CHECK(grad_y.dim() >= 1 && grad_y.size(-1) == p.out_width &&
                  grad_y.numel() == p.tokens * p.out_width,
              "grad_y must have shape [..., ", text(p.out_width), "]");
  const c10::cuda::CUDAGuard device_guard(x.device());
  TORCH_CHECK(saved.is_cuda() && saved.is_contiguous() && saved.scalar_type() == torch::kUInt8 &&
                  static_cast<size_t>(saved.numel()) >= fhb_ffn_saved_bytes(&p),
              "saved must be what gated_feed_forward returned for these arguments");
  const torch::Tensor dy = as_rows(grad_y);
  const auto like = [&](bool want, at::IntArrayRef shape) -> OptionalTensor {
    if (!want) return c10::nullopt;
    return torch::empty(shape, x.options());
  };
  std::vector<OptionalTensor> out{like(wants[0], x.sizes()),
                                  like(wants[1], w_gate.sizes()),
                                  like(wants[2], w_up.sizes()),
                                  like(wants[3], w_down.sizes()),
                                  like(wants[4] && b_gate, {p.hidden}),
                                  like(wants[5] && b_up, {p.hidden}),
                                  like(wants[6] && b_down, {p.out_width})};
  const fhb_ffn_grads grads{data_of(out[0]), data_of(out[1]), data_of(out[2]), data_of(out[3]),
                            data_of(out[4]), data_of(out[5]), data_of(out[6])};
  auto workspace = bytes_for(fhb_ffn_workspace_bytes(&p, 1), x);
  check_status(fhb_ffn_backward(&p, data_of(dy), row_stride(dy), data_of(saved), &grads,
                                data_of(workspace), static_cast<size_t>(workspace.numel()),
                                at::cuda::getCurrentCUDAStream()),
               "gated_feed_forward_backward");
  return out;
}

// ---- norms with gate and residual scale ----

struct Norm {
  fhb_norm_problem problem{};
  torch::Tensor residual, branch, gate;
};

Norm norm_of(const torch::Tensor& residual, const OptionalTensor& branch,
             const torch::Tensor& pre_weight, const OptionalTensor& post_weight,
             const OptionalTensor& gate, const OptionalTensor& scale_tensor, double scale,
             double eps) {
  TORCH_CHECK(residual.is_cuda(), "residual must be a CUDA tensor");
  const int residual_dtype = dtype_code(residual, "residual");
  TORCH_CHECK(residual.dim() >= 1 && residual.size(-1) >= 1,
              "residual must have shape [..., width] with a width of at least 1");
  const int64_t width = residual.size(-1);
  TORCH_CHECK(pre_weight.is_cuda(), "pre_weight must be a CUDA tensor");
  const int dtype = dtype_code(pre_weight, "pre_weight");
  TORCH_CHECK(residual_dtype == FHB_DTYPE_F32 || dtype == FHB_DTYPE_BF16,
              "a bfloat16 residual goes with bfloat16 weights and branch");
  TORCH_CHECK(pre_weight.device() == residual.device(),
              "pre_weight must be on the same device as residual");
  check_vector(pre_weight, pre_weight, width, "pre_weight", "residual");
  TORCH_CHECK(branch || (!gate && !post_weight), "gate and post_weight need a branch");
  TORCH_CHECK(eps >= 0.0, "eps must be >= 0");
  Norm n;
  fhb_norm_problem& p = n.problem;
  n.residual = as_rows(residual);
  p.rows = n.residual.size(0);
  p.width = width;
  p.residual_dtype = residual_dtype;
  p.dtype = dtype;
  p.residual = data_of(n.residual);
  p.residual_stride = row_stride(n.residual);
  p.gate_rows = p.rows > 0 ? p.rows : 1;
  if (branch) {
    check_like(*branch, pre_weight, "branch", "pre_weight");
    TORCH_CHECK(branch->sizes() == residual.sizes(), "branch must have the shape of residual");
    n.branch = as_rows(*branch);
    p.branch = data_of(n.branch);
    p.branch_stride = row_stride(n.branch);
  }
  if (post_weight) check_vector(*post_weight, pre_weight, width, "post_weight", "pre_weight");
  if (gate) {
    // [width]; or the residual's shape with ones from some dimension on: one gate row for
    // that many consecutive rows; or the residual's shape.
    check_like(*gate, pre_weight, "gate", "pre_weight");
    const int64_t dims = residual.dim();
    bool fits = gate->dim() >= 1 && gate->size(-1) == width;
    int64_t groups = 1;
    if (gate->dim() > 1) {
      fits = fits && gate->dim() == dims;
      bool ones = false;  // a size of 1 where residual has more: from here on all are
      for (int64_t d = 0; fits && d + 1 < dims; ++d) {
        if (gate->size(d) == 1 && residual.size(d) != 1) ones = true;
        else if (gate->size(d) != residual.size(d) || (ones && residual.size(d) != 1)) fits = false;
        groups *= gate->size(d);
      }
    }
    TORCH_CHECK(fits, "gate must have shape [width], the residual's shape, or the residual's "
                      "shape with ones in its last leading dimensions");
    n.gate = gate->contiguous();
    p.gate = data_of(n.gate);
    p.gate_rows = groups > 0 && p.rows > 0 ? p.rows / groups : 1;
  }
  if (scale_tensor) {
    TORCH_CHECK(scale_tensor->is_cuda() && scale_tensor->device() == residual.device() &&
                    scale_tensor->scalar_type() == torch::kFloat32 && scale_tensor->numel() == 1,
                "residual_scale must be a number or a float32 CUDA tensor with one element on "
                "the residual's device");
    p.residual_scale_ptr = scale_tensor->data_ptr<float>();
  }
  p.pre_weight = data_of(pre_weight);
  p.post_weight = data_of(post_weight);
  p.residual_scale = static_cast<float>(scale);
  p.eps = static_cast<float>(eps);
  return n;
}

// (total or an empty tensor, normed, stats or an empty tensor)
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> residual_norm(
    torch::Tensor residual, OptionalTensor branch, torch::Tensor pre_weight,
    OptionalTensor post_weight, OptionalTensor gate, OptionalTensor scale_tensor, double scale,
    double eps, bool want_total, bool want_stats) {
  const Norm n = norm_of(residual, branch, pre_weight, post_weight, gate, scale_tensor, scale, eps);
  const c10::cuda::CUDAGuard device_guard(residual.device());
  auto total = want_total ? torch::empty(residual.sizes(), residual.options())
                          : torch::empty({0}, residual.options());
  auto normed = torch::empty(residual.sizes(), pre_weight.options());
  auto stats = torch::empty({want_stats ? 2 * n.problem.rows : 0},
                            residual.options().dtype(torch::kFloat32));
  check_status(fhb_residual_norm(&n.problem, data_of(total), data_of(normed),
                                 static_cast<float*>(data_of(stats)),
                                 at::cuda::getCurrentCUDAStream()),
               "residual_norm");
  return {total, normed, stats};
}

// Gradients of residual, branch, pre_weight, post_weight, gate, residual_scale; None where
// wants[i] is false.
std::vector<OptionalTensor> residual_norm_backward(
    OptionalTensor grad_total, OptionalTensor grad_normed, torch::Tensor residual,
    OptionalTensor branch, torch::Tensor pre_weight, OptionalTensor post_weight,
    OptionalTensor gate, OptionalTensor scale_tensor, double scale, double eps,
    torch::Tensor stats, std::vector<bool> wants) {
  const Norm n = norm_of(residual, branch, pre_weight, post_weight, gate, scale_tensor, scale, eps);
  const fhb_norm_problem& p = n.problem;
  TORCH_CHECK(wants.size() == 6, "wants must have 6 entries");
  TORCH_CHECK(stats.is_cuda() && stats.is_contiguous() &&
                  stats.scalar_type() == torch::kFloat32 && stats.numel() == 2 * p.rows,
              "stats must be what residual_norm returned for these arguments");
  const c10::cuda::CUDAGuard device_guard(residual.device());
  torch::Tensor dt, dn;
  if (grad_total) {
    check_like(*grad_total, residual, "grad_total", "residual");
    TORCH_CHECK(grad_total->numel() == residual.numel() && grad_total->size(-1) == p.width,
                "grad_total must have the shape of residual");
    dt = as_rows(*grad_total);
  }
  if (grad_normed) {
    check_like(*grad_normed, pre_weight, "grad_normed", "pre_weight");
    TORCH_CHECK(grad_normed->numel() == residual.numel() && grad_normed->size(-1) == p.width,
                "grad_normed must have the shape of residual");
    dn = as_rows(*grad_normed);
  }
  const auto like = [](bool want, const torch::Tensor& t) -> OptionalTensor {
    if (!want) return c10::nullopt;
    return torch::empty(t.sizes(), t.options());
  };
  std::vector<OptionalTensor> out{
      like(wants[0], residual),
      like(wants[1] && branch, branch ? *branch : residual),
      like(wants[2], pre_weight),
      like(wants[3] && post_weight, post_weight ? *post_weight : residual),
      like(wants[4] && gate, gate ? *gate : residual),
      like(wants[5] && scale_tensor, scale_tensor ? *scale_tensor : residual)};
  const fhb_norm_grads grads{data_of(out[0]), data_of(out[1]), data_of(out[2]), data_of(out[3]),
                             data_of(out[4]), static_cast<float*>(data_of(out[5]))};
  auto workspace = bytes_for(fhb_residual_norm_workspace_bytes(&p), residual);
  check_status(
      fhb_residual_norm_backward(
          &p, grad_total ? data_of(dt) : nullptr, grad_total ? row_stride(dt) : 0,
          grad_normed ? data_of(dn) : nullptr, grad_normed ? row_stride(dn) : 0,
          static_cast<const float*>(data_of(stats)), &grads, data_of(workspace),
          static_cast<size_t>(workspace.numel()), at::cuda::getCurrentCUDAStream()),
      "residual_norm_backward");
  return out;
}

// ---- AdamW over many tensors ----

void adamw_step(const std::vector<torch::Tensor>& params, const std::vector<torch::Tensor>& grads,
                const std::vector<torch::Tensor>& exp_avgs,
                const std::vector<torch::Tensor>& exp_avg_sqs,
                const c10::optional<std::vector<torch::Tensor>>& exp_avg_scales,
                const c10::optional<std::vector<torch::Tensor>>& exp_avg_sq_scales,
                torch::Tensor step, double lr, double beta1, double beta2, double eps,
                double weight_decay) {
  const size_t n = params.size();
  TORCH_CHECK(grads.size() == n && exp_avgs.size() == n && exp_avg_sqs.size() == n,
              "params, grads, exp_avgs and exp_avg_sqs must have the same length");
  const bool eight = exp_avg_scales.has_value();
  TORCH_CHECK(eight == exp_avg_sq_scales.has_value(),
              "exp_avg_scales and exp_avg_sq_scales go together");
  if (eight)
    TORCH_CHECK(exp_avg_scales->size() == n && exp_avg_sq_scales->size() == n,
                "params and the scales must have the same length");
  TORCH_CHECK(step.is_cuda() && step.scalar_type() == torch::kInt64 && step.numel() == 1,
              "step must be a CUDA int64 tensor with one element");
  TORCH_CHECK(lr >= 0.0, "lr must be >= 0");
  TORCH_CHECK(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0,
              "betas must be in [0, 1)");
  TORCH_CHECK(eps >= 0.0, "eps must be >= 0");
  TORCH_CHECK(weight_decay >= 0.0, "weight_decay must be >= 0");
  const auto state_type = eight ? torch::kFloat8_e4m3fn : torch::kFloat32;
  const auto check_state = [&](const torch::Tensor& t, size_t i, torch::ScalarType type,
                               int64_t numel, const char* what) {
    TORCH_CHECK(t.is_cuda() && t.device() == step.device(), what, "[", text(static_cast<int64_t>(i)),
                "] must be on the device of step");
    TORCH_CHECK(t.scalar_type() == type, what, "[", text(static_cast<int64_t>(i)), "] must use ",
                c10::toString(type));
    TORCH_CHECK(t.is_contiguous() && t.numel() == numel, what, "[",
                text(static_cast<int64_t>(i)), "] must be contiguous with ", text(numel), " values");
  };
  std::vector<fhb_adamw_tensor> table(n);
  for (size_t i = 0; i < n; ++i) {
    const torch::Tensor &p = params[i], &g = grads[i];
    const int64_t count = p.numel(), blocks = (count + FHB_ADAMW_BLOCK - 1) / FHB_ADAMW_BLOCK;
    const int dtype = dtype_code(p, "params");
    check_state(p, i, p.scalar_type(), count, "params");
    check_state(g, i, p.scalar_type(), count, "grads");
    check_state(exp_avgs[i], i, state_type, count, "exp_avgs");
    check_state(exp_avg_sqs[i], i, state_type, count, "exp_avg_sqs");
    table[i] = {data_of(p), data_of(g), data_of(exp_avgs[i]), data_of(exp_avg_sqs[i]),
                nullptr, nullptr, count, dtype};
    if (eight) {
      check_state((*exp_avg_scales)[i], i, torch::kFloat32, blocks, "exp_avg_scales");
      check_state((*exp_avg_sq_scales)[i], i, torch::kFloat32, blocks, "exp_avg_sq_scales");
      table[i].exp_avg_scale = static_cast<float*>(data_of((*exp_avg_scales)[i]));
      table[i].exp_avg_sq_scale = static_cast<float*>(data_of((*exp_avg_sq_scales)[i]));
    }
  }
  const c10::cuda::CUDAGuard device_guard(step.device());
  check_status(fhb_adamw_step(table.data(), static_cast<int64_t>(n), eight ? 8 : 32,
                              step.data_ptr<int64_t>(), lr, beta1, beta2, eps, weight_decay,
                              at::cuda::getCurrentCUDAStream()),
               "adamw_step");
}

}  // namespace

void bind_blocks(pybind11::module& module) {
  using pybind11::arg;
  module.def("gated_feed_forward", &gated_feed_forward,
             "Gated feed-forward block (CUDA, sm_100a): (y, saved)", arg("x"), arg("w_gate"),
             arg("w_up"), arg("w_down"), arg("b_gate") = pybind11::none(),
             arg("b_up") = pybind11::none(), arg("b_down") = pybind11::none(),
             arg("activation") = "silu", arg("want_saved") = false);
  module.def("gated_feed_forward_backward", &gated_feed_forward_backward,
             "Gradients of the gated feed-forward block (CUDA, sm_100a)", arg("grad_y"), arg("x"),
             arg("w_gate"), arg("w_up"), arg("w_down"), arg("b_gate"), arg("b_up"), arg("b_down"),
             arg("activation"), arg("saved"), arg("wants"));
  module.def("residual_norm", &residual_norm,
             "RMS norms before and after a block with its gate and residual scale (CUDA, "
             "sm_100a): (total, normed, stats)",
             arg("residual"), arg("branch"), arg("pre_weight"), arg("post_weight"), arg("gate"),
             arg("scale_tensor"), arg("scale"), arg("eps"), arg("want_total"), arg("want_stats"));
  module.def("residual_norm_backward", &residual_norm_backward,
             "Gradients of residual_norm (CUDA, sm_100a)", arg("grad_total"), arg("grad_normed"),
             arg("residual"), arg("branch"), arg("pre_weight"), arg("post_weight"), arg("gate"),
             arg("scale_tensor"), arg("scale"), arg("eps"), arg("stats"), arg("wants"));
  module.def("adamw_step", &adamw_step, "AdamW over many tensors, 32- or 8-bit states",
             arg("params"), arg("grads"), arg("exp_avgs"), arg("exp_avg_sqs"),
             arg("exp_avg_scales"), arg("exp_avg_sq_scales"), arg("step"), arg("lr"),
             arg("beta1"), arg("beta2"), arg("eps"), arg("weight_decay"));
}
