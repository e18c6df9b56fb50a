// Torch binding of the gated residual trunk's operators (include/fused_hoad_b200.h): part of
// the module fused_hoad._C. Outputs, workspaces and what the backward keeps come from the ATen
// caching allocator on the current stream, so the ops stay asynchronous and graph-capturable.
// Gradients are autograd nodes in C++: autograd's threads need no Python for them (a node in
// Python costs about 70 us a backward pass).
#include <ATen/cuda/CUDAContext.h>
#include <c10/core/AutogradState.h>
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

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

OptionalTensor given(const torch::Tensor& t) {
  return t.defined() ? OptionalTensor(t) : OptionalTensor();
}
torch::Tensor or_undefined(const OptionalTensor& t) { return t ? *t : torch::Tensor(); }

bool records_gradients(const variable_list& tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const torch::Tensor& t : tensors)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}
// The backwards are not differentiable themselves. Recording a graph of one (create_graph) would
// cut it off there, and gradients of gradients would silently lack a part: it raises instead.
void check_differentiated_once(const char* op) {
  TORCH_CHECK(!at::GradMode::is_enabled(), op,
              " is differentiable once: its backward does not support create_graph");
}
// Forward-mode derivatives are not computed: a result without its tangent would read as a zero
// derivative, so an input that carries one is refused.
void check_no_tangents(const char* op, const variable_list& tensors) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const torch::Tensor& t : tensors)
    TORCH_CHECK(!t.defined() || !t._fw_grad(/*level=*/0).defined(), op,
                " does not support forward-mode derivatives");
}

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

// y [..., out_width]; `saved`, where given, becomes what the backward needs.
torch::Tensor ffn_forward(const Ffn& f, const torch::Tensor& x, torch::Tensor* saved) {
  const c10::cuda::CUDAGuard device_guard(x.device());
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = f.problem.out_width;
  auto y = torch::empty(shape, x.options());
  if (saved != nullptr) *saved = bytes_for(fhb_ffn_saved_bytes(&f.problem), x);
  if (f.problem.tokens == 0) return y;
  const int pass = saved != nullptr ? FHB_FFN_FORWARD_SAVING : FHB_FFN_FORWARD;
  auto workspace = bytes_for(fhb_ffn_workspace_bytes(&f.problem, pass), x);
  check_status(fhb_ffn_forward(&f.problem, y.data_ptr(),
                               saved != nullptr ? saved->data_ptr() : nullptr, data_of(workspace),
                               static_cast<size_t>(workspace.numel()),
                               at::cuda::getCurrentCUDAStream()),
               "gated_feed_forward");
  return y;
}

class FfnNode : public torch::autograd::Function<FfnNode> {
 public:
  static torch::Tensor forward(AutogradContext* ctx, const torch::Tensor& x,
                               const torch::Tensor& w_gate, const torch::Tensor& w_up,
                               const torch::Tensor& w_down, const OptionalTensor& b_gate,
                               const OptionalTensor& b_up, const OptionalTensor& b_down,
                               const std::string& activation) {
    const Ffn f = ffn_of(x, w_gate, w_up, w_down, b_gate, b_up, b_down, activation);
    torch::Tensor saved;
    auto y = ffn_forward(f, x, &saved);
    ctx->saved_data["activation"] = activation;
    ctx->save_for_backward({saved, x, w_gate, w_up, w_down, or_undefined(b_gate), or_undefined(b_up),
                            or_undefined(b_down)});
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list upstream) {
    check_differentiated_once("gated_feed_forward");
    check_no_tangents("gated_feed_forward's backward", upstream);
    const variable_list t = ctx->get_saved_variables();
    const torch::Tensor &saved = t[0], &x = t[1], &grad_y = upstream[0];
    const Ffn f = ffn_of(x, t[2], t[3], t[4], given(t[5]), given(t[6]), given(t[7]),
                         ctx->saved_data["activation"].toStringRef());
    const fhb_ffn_problem& p = f.problem;
    check_like(grad_y, x, "grad_y", "x");
    variable_list out(8);
    const c10::cuda::CUDAGuard device_guard(x.device());
    const torch::Tensor dy = as_rows(grad_y);
    for (int i = 0, edge = 0; i < 7; ++i)  // only tensors that were given have an edge
      if (t[i + 1].defined() && ctx->needs_input_grad(edge++)) out[i] = torch::empty(t[i + 1].sizes(), x.options());
    const auto place = [&](int i) { return out[i].defined() ? data_of(out[i]) : nullptr; };
    const fhb_ffn_grads grads{place(0), place(1), place(2), place(3), place(4), place(5), place(6)};
    auto workspace = bytes_for(fhb_ffn_workspace_bytes(&p, FHB_FFN_BACKWARD), x);
    check_status(fhb_ffn_backward(&p, data_of(dy), row_stride(dy), data_of(saved), &grads,
                                  data_of(workspace), static_cast<size_t>(workspace.numel()),
                                  at::cuda::getCurrentCUDAStream()),
                 "gated_feed_forward's backward");
    return out;
  }
};

torch::Tensor gated_feed_forward(torch::Tensor x, torch::Tensor w_gate, torch::Tensor w_up,
                                 torch::Tensor w_down, OptionalTensor b_gate, OptionalTensor b_up,
                                 OptionalTensor b_down, const std::string& activation) {
  const variable_list tensors{x, w_gate, w_up, w_down, or_undefined(b_gate), or_undefined(b_up),
                              or_undefined(b_down)};
  check_no_tangents("gated_feed_forward", tensors);
  if (records_gradients(tensors))
    return FfnNode::apply(x, w_gate, w_up, w_down, b_gate, b_up, b_down, activation);
  return ffn_forward(ffn_of(x, w_gate, w_up, w_down, b_gate, b_up, b_down, activation), x, nullptr);
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

// (total or an undefined tensor, normed); `stats`, where given, becomes what the backward needs.
std::pair<torch::Tensor, torch::Tensor> norm_forward(const Norm& n, const torch::Tensor& residual,
                                                     const torch::Tensor& pre_weight,
                                                     bool want_total, torch::Tensor* stats) {
  const c10::cuda::CUDAGuard device_guard(residual.device());
  torch::Tensor total;
  if (want_total) total = torch::empty(residual.sizes(), residual.options());
  auto normed = torch::empty(residual.sizes(), pre_weight.options());
  if (stats != nullptr)
    *stats = torch::empty({2 * n.problem.rows}, residual.options().dtype(torch::kFloat32));
  check_status(fhb_residual_norm(&n.problem, want_total ? data_of(total) : nullptr, data_of(normed),
                                 stats != nullptr ? static_cast<float*>(data_of(*stats)) : nullptr,
                                 at::cuda::getCurrentCUDAStream()),
               "residual_norm");
  return {total, normed};
}

// Without a branch it is the norm alone, and there is no total.
class NormNode : public torch::autograd::Function<NormNode> {
 public:
  static variable_list forward(AutogradContext* ctx, const torch::Tensor& residual,
                               const OptionalTensor& branch, const torch::Tensor& pre_weight,
                               const OptionalTensor& post_weight, const OptionalTensor& gate,
                               const OptionalTensor& scale_tensor, double scale, double eps) {
    const Norm n = norm_of(residual, branch, pre_weight, post_weight, gate, scale_tensor, scale, eps);
    torch::Tensor stats;
    auto [total, normed] = norm_forward(n, residual, pre_weight, branch.has_value(), &stats);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["eps"] = eps;
    ctx->save_for_backward({stats, residual, or_undefined(branch), pre_weight, or_undefined(post_weight),
                            or_undefined(gate), or_undefined(scale_tensor)});
    ctx->set_materialize_grads(false);
    if (branch) return {total, normed};
    return {normed};
  }

  static variable_list backward(AutogradContext* ctx, variable_list upstream) {
    check_differentiated_once("residual_norm");
    check_no_tangents("residual_norm's backward", upstream);
    const variable_list t = ctx->get_saved_variables();
    const torch::Tensor &stats = t[0], &residual = t[1], &branch = t[2], &pre_weight = t[3];
    const Norm n = norm_of(residual, given(branch), pre_weight, given(t[4]), given(t[5]), given(t[6]),
                           ctx->saved_data["scale"].toDouble(), ctx->saved_data["eps"].toDouble());
    const fhb_norm_problem& p = n.problem;
    const torch::Tensor grad_total = branch.defined() ? upstream[0] : torch::Tensor();
    const torch::Tensor grad_normed = upstream.back();
    variable_list out(8);
    const c10::cuda::CUDAGuard device_guard(residual.device());
    torch::Tensor dt, dn;
    if (grad_total.defined()) {
      check_like(grad_total, residual, "grad_total", "residual");
      dt = as_rows(grad_total);
    }
    if (grad_normed.defined()) {
      check_like(grad_normed, pre_weight, "grad_normed", "pre_weight");
      dn = as_rows(grad_normed);
    }
    // without rows there may still be groups, each with a gate whose gradient is zero
    for (int i = 0, edge = 0; i < 6; ++i)
      if (t[i + 1].defined() && ctx->needs_input_grad(edge++))
        out[i] = p.rows > 0 ? torch::empty(t[i + 1].sizes(), t[i + 1].options())
                            : torch::zeros(t[i + 1].sizes(), t[i + 1].options());
    if (p.rows == 0) return out;
    const auto place = [&](int i) { return out[i].defined() ? data_of(out[i]) : nullptr; };
    const fhb_norm_grads grads{place(0), place(1), place(2), place(3), place(4),
                               static_cast<float*>(place(5))};
    auto workspace = bytes_for(fhb_residual_norm_workspace_bytes(&p), residual);
    check_status(
        fhb_residual_norm_backward(
            &p, dt.defined() ? data_of(dt) : nullptr, dt.defined() ? row_stride(dt) : 0,
            dn.defined() ? data_of(dn) : nullptr, dn.defined() ? row_stride(dn) : 0,
            static_cast<const float*>(data_of(stats)), &grads, data_of(workspace),
            static_cast<size_t>(workspace.numel()), at::cuda::getCurrentCUDAStream()),
        "residual_norm's backward");
    return out;
  }
};

// (total, normed), or (normed,) without a branch
variable_list residual_norm(torch::Tensor residual, OptionalTensor branch, torch::Tensor pre_weight,
                            OptionalTensor post_weight, OptionalTensor gate,
                            OptionalTensor scale_tensor, double scale, double eps) {
  const variable_list tensors{residual, or_undefined(branch), pre_weight, or_undefined(post_weight),
                              or_undefined(gate), or_undefined(scale_tensor)};
  check_no_tangents("residual_norm", tensors);
  if (records_gradients(tensors))
    return NormNode::apply(residual, branch, pre_weight, post_weight, gate, scale_tensor, scale, eps);
  const Norm n = norm_of(residual, branch, pre_weight, post_weight, gate, scale_tensor, scale, eps);
  auto [total, normed] = norm_forward(n, residual, pre_weight, branch.has_value(), nullptr);
  if (branch) return {total, normed};
  return {normed};
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
  // in place, as autograd sees it: a backward that saved one of these before the step raises
  const auto written = [](const std::vector<torch::Tensor>& tensors) {
    for (const torch::Tensor& t : tensors)
      if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  };
  written(params);
  written(exp_avgs);
  written(exp_avg_sqs);
  if (eight) {
    written(*exp_avg_scales);
    written(*exp_avg_sq_scales);
  }
  written({step});
}

}  // namespace

void bind_blocks(pybind11::module& module) {
  using pybind11::arg;
  module.def("gated_feed_forward", &gated_feed_forward,
             "Gated feed-forward block (CUDA, sm_100a), differentiable once", arg("x"),
             arg("w_gate"), arg("w_up"), arg("w_down"), arg("b_gate") = pybind11::none(),
             arg("b_up") = pybind11::none(), arg("b_down") = pybind11::none(),
             arg("activation") = "silu");
  module.def("residual_norm", &residual_norm,
             "RMS norms before and after a block with its gate and residual scale (CUDA, "
             "sm_100a), differentiable once: (total, normed), or (normed,) without a branch",
             arg("residual"), arg("branch"), arg("pre_weight"), arg("post_weight"), arg("gate"),
             arg("scale_tensor"), arg("scale"), arg("eps"));
  module.def("adamw_step", &adamw_step, "AdamW over many tensors, 32- or 8-bit states",
             arg("params"), arg("grads"), arg("exp_avgs"), arg("exp_avg_sqs"),
             arg("exp_avg_scales"), arg("exp_avg_sq_scales"), arg("step"), arg("lr"),
             arg("beta1"), arg("beta2"), arg("eps"), arg("weight_decay"));
}
