// Tokens sorted by expert and back, with gradients: moe_permute, moe_unpermute and their backward passes.  The reference gathers inside its GEMM
// and reduces without a gradient (src/moe_gather_rs/ths_op/topk_scatter_reduce.cc:30-56), so these have no counterpart there.
#include <c10/core/DeviceGuard.h>

#include "autograd_checks.h"
#include "ths_ops.h"

namespace flux_amd {
namespace {

int32_t row_type(const torch::Tensor &t, const char *name) {
  const at::ScalarType st = t.scalar_type();
  TORCH_CHECK(st == at::kBFloat16 || st == at::kHalf || st == at::kFloat, name, " must be bfloat16, float16 or float32, got ", st);
  return st == at::kBFloat16 ? FLUXMI_ROWS_BF16 : st == at::kFloat ? FLUXMI_ROWS_FP32 : FLUXMI_ROWS_FP16;
}

void check_rows(const torch::Tensor &t, const char *name) {
  refuse_tangent(t, name);
  refuse_lazy_view(t, name);
  TORCH_CHECK(t.is_cuda(), name, " must be a device tensor");
  TORCH_CHECK(t.dim() == 2, name, " must have 2 dimensions, got ", t.dim());
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
  TORCH_CHECK(t.size(1) <= INT32_MAX, name, " is wider than 2^31 - 1 columns");
}

// scatter_index: int32 [tokens, topk] on the device of `like`.
void check_index(const torch::Tensor &scatter_index, const torch::Tensor &like) {
  FLUX_AMD_CHECK_INPUT(scatter_index, at::kInt);
  FLUX_AMD_CHECK_NDIM(scatter_index, 2);
  TORCH_CHECK(scatter_index.size(1) >= 1, "scatter_index must have at least one column");
  TORCH_CHECK(scatter_index.numel() <= (int64_t{1} << 30), "scatter_index has more than 2^30 entries");
  TORCH_CHECK(scatter_index.device() == like.device(), "scatter_index is on ", scatter_index.device(), ", the rows are on ", like.device());
}

void check_pair_rows(const torch::Tensor &rows, const torch::Tensor &scatter_index, const char *name) {
  TORCH_CHECK(rows.size(0) == scatter_index.numel(), name, " must have one row per entry of scatter_index: ", rows.size(0), " rows, ",
              scatter_index.numel(), " entries");
}

int32_t check_weights(const torch::Tensor &weights, const torch::Tensor &scatter_index) {
  refuse_tangent(weights, "weights");
  refuse_lazy_view(weights, "weights");
  TORCH_CHECK(weights.is_cuda(), "weights must be a device tensor");
  TORCH_CHECK(weights.sizes() == scatter_index.sizes(), "weights shape mismatch: ", weights.sizes(), " expected ", scatter_index.sizes());
  TORCH_CHECK(weights.is_contiguous(), "weights must be contiguous");
  TORCH_CHECK(weights.device() == scatter_index.device(), "weights are on ", weights.device(), ", scatter_index is on ", scatter_index.device());
  return row_type(weights, "weights");
}

int32_t tokens_of(const torch::Tensor &scatter_index) { return static_cast<int32_t>(scatter_index.size(0)); }
int32_t topk_of(const torch::Tensor &scatter_index) { return static_cast<int32_t>(scatter_index.size(1)); }

torch::Tensor permute(const torch::Tensor &input, const torch::Tensor &scatter_index) {
  const c10::DeviceGuard guard(input.device());
  torch::Tensor rows = empty_on(input, {scatter_index.numel(), input.size(1)}, input.scalar_type());
  check_status(fluxmi_moe_permute(input.data_ptr(), scatter_index.data_ptr<int32_t>(), tokens_of(scatter_index), topk_of(scatter_index),
                                  input.size(1) * static_cast<int64_t>(input.element_size()), rows.data_ptr(), current_stream()),
               "fluxmi_moe_permute");
  return rows;
}

torch::Tensor unpermute(const torch::Tensor &rows, const torch::Tensor &scatter_index, const torch::Tensor &weights) {
  const c10::DeviceGuard guard(rows.device());
  torch::Tensor out = empty_on(rows, {scatter_index.size(0), rows.size(1)}, rows.scalar_type());
  check_status(fluxmi_moe_unpermute(rows.data_ptr(), row_type(rows, "rows"), scatter_index.data_ptr<int32_t>(),
                                    weights.defined() ? weights.data_ptr() : nullptr, weights.defined() ? row_type(weights, "weights") : FLUXMI_ROWS_FP32,
                                    tokens_of(scatter_index), topk_of(scatter_index), static_cast<int32_t>(rows.size(1)), out.data_ptr(), current_stream()),
               "fluxmi_moe_unpermute");
  return out;
}

// An undefined result: not asked for.
std::tuple<torch::Tensor, torch::Tensor> unpermute_backward(const torch::Tensor &grad_out, const torch::Tensor &rows, const torch::Tensor &scatter_index,
                                                            const torch::Tensor &weights, bool want_rows, bool want_weights) {
  const c10::DeviceGuard guard(grad_out.device());
  torch::Tensor grad_rows, grad_weights;
  if (want_rows) grad_rows = empty_on(grad_out, {scatter_index.numel(), grad_out.size(1)}, grad_out.scalar_type());
  if (want_weights) grad_weights = empty_on(weights, weights.sizes(), weights.scalar_type());
  check_status(fluxmi_moe_unpermute_backward(grad_out.data_ptr(), want_weights ? rows.data_ptr() : nullptr, row_type(grad_out, "grad_out"),
                                             scatter_index.data_ptr<int32_t>(), weights.data_ptr(), row_type(weights, "weights"), tokens_of(scatter_index),
                                             topk_of(scatter_index), static_cast<int32_t>(grad_out.size(1)), want_rows ? grad_rows.data_ptr() : nullptr,
                                             want_weights ? grad_weights.data_ptr() : nullptr, current_stream()),
               "fluxmi_moe_unpermute_backward");
  return {grad_rows, grad_weights};
}

struct Permute : torch::autograd::Function<Permute> {
  static torch::Tensor forward(torch::autograd::AutogradContext *ctx, const torch::Tensor &input, const torch::Tensor &scatter_index) {
    ctx->save_for_backward({scatter_index});
    return permute(input, scatter_index);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
    refuse_second_derivative("moe_permute", grads[0]);
    refuse_leaves_of_another_stream("moe_permute");
    return {unpermute(grads[0].resolve_neg().contiguous(), ctx->get_saved_variables()[0], {}), {}};
  }
};

// Without weights.
struct Sum : torch::autograd::Function<Sum> {
  static torch::Tensor forward(torch::autograd::AutogradContext *ctx, const torch::Tensor &rows, const torch::Tensor &scatter_index) {
    ctx->save_for_backward({scatter_index});
    return unpermute(rows, scatter_index, {});
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
    refuse_second_derivative("moe_unpermute", grads[0]);
    refuse_leaves_of_another_stream("moe_unpermute");
    return {permute(grads[0].resolve_neg().contiguous(), ctx->get_saved_variables()[0]), {}};
  }
};

struct Unpermute : torch::autograd::Function<Unpermute> {
  static torch::Tensor forward(torch::autograd::AutogradContext *ctx, const torch::Tensor &rows, const torch::Tensor &scatter_index,
                               const torch::Tensor &weights) {
    // (rows are read for the gradient of the weights only)
    ctx->save_for_backward({scatter_index, weights, weights.requires_grad() ? rows : torch::Tensor()});
    ctx->saved_data["rows"] = rows.requires_grad();
    return unpermute(rows, scatter_index, weights);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
    refuse_second_derivative("moe_unpermute", grads[0]);
    refuse_leaves_of_another_stream("moe_unpermute");
    const auto saved = ctx->get_saved_variables();
    const torch::Tensor grad = grads[0].resolve_neg().contiguous(), &scatter_index = saved[0], &weights = saved[1], &rows = saved[2];
    const bool want_rows = ctx->saved_data["rows"].toBool(), want_weights = rows.defined();
    const auto [grad_rows, grad_weights] = unpermute_backward(grad, rows, scatter_index, weights, want_rows, want_weights);
    return {grad_rows, {}, grad_weights};
  }
};

}  // namespace

torch::Tensor moe_permute(torch::Tensor input, torch::Tensor scatter_index) {
  check_rows(input, "input");
  check_index(scatter_index, input);
  TORCH_CHECK(input.size(0) == scatter_index.size(0), "input has ", input.size(0), " tokens, scatter_index ", scatter_index.size(0));
  if (at::GradMode::is_enabled() && input.requires_grad()) {
    row_type(input, "an input with a gradient");
    return Permute::apply(input, scatter_index);
  }
  return permute(input, scatter_index);
}

torch::Tensor moe_permute_backward(torch::Tensor grad_rows, torch::Tensor scatter_index) {
  check_rows(grad_rows, "grad_rows");
  row_type(grad_rows, "grad_rows");
  check_index(scatter_index, grad_rows);
  check_pair_rows(grad_rows, scatter_index, "grad_rows");
  return unpermute(grad_rows, scatter_index, {});
}

torch::Tensor moe_unpermute(torch::Tensor rows, torch::Tensor scatter_index, std::optional<torch::Tensor> weights) {
  check_rows(rows, "rows");
  row_type(rows, "rows");
  check_index(scatter_index, rows);
  check_pair_rows(rows, scatter_index, "rows");
  torch::Tensor w;
  if (weights.has_value()) {
    w = *weights;
    check_weights(w, scatter_index);
  }
  if (at::GradMode::is_enabled()) {
    if (w.defined() && (rows.requires_grad() || w.requires_grad())) return Unpermute::apply(rows, scatter_index, w);
    if (!w.defined() && rows.requires_grad()) return Sum::apply(rows, scatter_index);
  }
  return unpermute(rows, scatter_index, w);
}

std::tuple<torch::Tensor, torch::Tensor> moe_unpermute_backward(torch::Tensor grad_out, torch::Tensor rows, torch::Tensor scatter_index,
                                                                torch::Tensor weights) {
  check_rows(grad_out, "grad_out");
  check_rows(rows, "rows");
  row_type(rows, "rows");
  check_index(scatter_index, rows);
  check_pair_rows(rows, scatter_index, "rows");
  check_weights(weights, scatter_index);
  TORCH_CHECK(grad_out.device() == rows.device(), "grad_out is on ", grad_out.device(), ", rows are on ", rows.device());
  TORCH_CHECK(grad_out.scalar_type() == rows.scalar_type(), "grad_out is ", grad_out.scalar_type(), ", rows are ", rows.scalar_type());
  FLUX_AMD_CHECK_2D(grad_out, scatter_index.size(0), rows.size(1));
  return unpermute_backward(grad_out, rows, scatter_index, weights, true, true);
}

}  // namespace flux_amd
