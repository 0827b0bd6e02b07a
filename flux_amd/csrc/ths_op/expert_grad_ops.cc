// Experts that learn: the gradients of the grouped product, activation checkpoints in 8 bits, and both joined to layers with autograd.  The reference has no
// gradients of its MoE operators; moe_linear's forward pass is the product of GemmGroupedV3 (src/comm_none/ths_op/gemm_grouped_v3.cc:43-171).
#include <ATen/MemoryOverlap.h>
#include <c10/core/DeviceGuard.h>

#include "autograd_checks.h"
#include "ths_ops.h"

namespace flux_amd {
namespace {

constexpr at::ScalarType kCodes = at::ScalarType::Float8_e4m3fn, kScales = at::ScalarType::Float8_e8m0fnu;
constexpr int64_t kBlock = 32;

int64_t blocks_of(int64_t cols) { return (cols + kBlock - 1) / kBlock; }

int32_t row_type(const torch::Tensor &t) { return t.scalar_type() == at::kHalf ? FLUXMI_ROWS_FP16 : FLUXMI_ROWS_BF16; }

void check_operand(const torch::Tensor &t, const char *name, int64_t dims) {
  refuse_tangent(t, name);
  refuse_lazy_view(t, name);
  TORCH_CHECK(t.is_cuda(), name, " must be a device tensor");
  TORCH_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf, name, " must be bfloat16 or float16, got ", t.scalar_type());
  TORCH_CHECK(t.dim() == dims, name, " must have ", dims, " dimensions, got ", t.dim());
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}

void check_like(const torch::Tensor &t, const char *name, const torch::Tensor &like, const char *like_name) {
  TORCH_CHECK(t.scalar_type() == like.scalar_type(), name, " is ", t.scalar_type(), ", ", like_name, " is ", like.scalar_type());
  TORCH_CHECK(t.device() == like.device(), name, " is on ", t.device(), ", ", like_name, " is on ", like.device());
}

void check_splits(const torch::Tensor &splits, const torch::Tensor &like, int64_t experts) {
  refuse_lazy_view(splits, "splits");
  FLUX_AMD_CHECK_NDIM(splits, 1);
  TORCH_CHECK(splits.scalar_type() == at::kInt, "splits must be int32, got ", splits.scalar_type());
  TORCH_CHECK(splits.is_contiguous(), "splits must be contiguous");
  TORCH_CHECK(splits.size(0) <= 1024, "at most 1024 experts, got ", splits.size(0));
  TORCH_CHECK(experts < 0 || splits.size(0) == experts, "splits 0-dim mismatch: ", splits.size(0), " != ", experts);
  TORCH_CHECK(splits.is_cuda() ? splits.device() == like.device() : splits.device().is_cpu(), "splits must be on the host or on ", like.device());
}

// Counts on the host are copied in the stream's order (a replay of a captured call reads them again, so that they have to live as long as the graph); what they have past
// the rows does not exist for the kernels.
torch::Tensor on_device(const torch::Tensor &splits, const torch::Tensor &like) {
  return splits.is_cuda() ? splits : splits.to(like.device(), /*non_blocking=*/true);
}

void check_weight(const torch::Tensor &weight, const char *name, const torch::Tensor &rows, const char *rows_name, int64_t dim) {
  check_operand(weight, name, 3);
  check_like(weight, name, rows, rows_name);
  TORCH_CHECK(weight.size(dim) == rows.size(1), name, " ", dim, "-dim mismatch: ", weight.size(dim), " != ", rows.size(1));
}

// Codes [rows, cols] and scales [rows, halves * blocks] of a checkpoint.
void check_kept(const torch::Tensor &codes, const torch::Tensor &scale, const torch::Tensor &like, int64_t halves) {
  refuse_lazy_view(codes, "input");
  refuse_lazy_view(scale, "input_scale");
  TORCH_CHECK(codes.is_cuda() && scale.is_cuda(), "input and input_scale must be device tensors");
  TORCH_CHECK(codes.scalar_type() == kCodes, "an input with a scale must be float8_e4m3fn, got ", codes.scalar_type());
  TORCH_CHECK(scale.scalar_type() == kScales, "input_scale must be float8_e8m0fnu, got ", scale.scalar_type());
  TORCH_CHECK(codes.is_contiguous() && scale.is_contiguous(), "input and input_scale must be contiguous");
  TORCH_CHECK(codes.device() == like.device() && scale.device() == like.device(), "input is on ", codes.device(), ", input_scale on ", scale.device(),
              ", the gradient on ", like.device());
  FLUX_AMD_CHECK_NDIM(codes, 2);
  FLUX_AMD_CHECK_2D(scale, codes.size(0), halves * blocks_of(codes.size(1) / halves));
}

// ---- the calls ------------------------------------------------------------------------------------------------

torch::Tensor product(const torch::Tensor &input, const torch::Tensor &weight, const torch::Tensor &splits) {
  constexpr int64_t kMost = 1 << 24;  // the gradients' limits
  TORCH_CHECK(input.size(0) <= kMost && weight.size(1) <= kMost && weight.size(2) <= kMost, "at most 2^24 rows and weights of 2^24 x 2^24, got ", input.size(0), " rows, ",
              weight.size(1), " x ", weight.size(2));
  const c10::DeviceGuard guard(input.device());
  torch::Tensor out = empty_on(input, {input.size(0), weight.size(1)}, input.scalar_type());
  if (out.numel() == 0) return out;
  fluxmi_grouped_gemm_args args{};
  args.dtype = to_fluxmi_dtype(input.scalar_type());
  args.nexperts = static_cast<int32_t>(weight.size(0));
  args.max_rows = static_cast<int32_t>(input.size(0));
  args.n = static_cast<int32_t>(weight.size(1));
  args.k = static_cast<int32_t>(weight.size(2));
  args.a = input.data_ptr();
  args.b = weight.data_ptr();
  args.d = out.data_ptr();
  args.splits = splits.data_ptr<int32_t>();
  args.scalar_scale = 1.0f;
  apply_launch_tuning(args, 1, 0);
  check_status(fluxmi_grouped_gemm(&args, nullptr, 0, current_stream()), "fluxmi_grouped_gemm");
  check_status(fluxmi_moe_clear_rest(out.data_ptr(), args.splits, args.nexperts, out.size(0), out.size(1) * 2, current_stream()), "fluxmi_moe_clear_rest");
  return out;
}

torch::Tensor input_gradient(const torch::Tensor &grad, const torch::Tensor &weight, const torch::Tensor &splits) {
  const c10::DeviceGuard guard(grad.device());
  torch::Tensor out = empty_on(grad, {grad.size(0), weight.size(2)}, grad.scalar_type());
  const size_t ws_bytes = fluxmi_moe_dgrad_workspace_bytes(static_cast<int32_t>(weight.size(0)), grad.size(0), grad.size(1), weight.size(2));
  torch::Tensor ws;
  if (ws_bytes > 0) ws = empty_on(grad, {static_cast<int64_t>(ws_bytes)}, at::kByte);
  check_status(fluxmi_moe_dgrad(grad.data_ptr(), weight.data_ptr(), row_type(grad), splits.data_ptr<int32_t>(), static_cast<int32_t>(weight.size(0)),
                                grad.size(0), grad.size(1), weight.size(2), out.data_ptr(), ws_bytes > 0 ? ws.data_ptr() : nullptr, ws_bytes, current_stream()),
               "fluxmi_moe_dgrad");
  return out;
}

// scale: undefined where input is of 16 bits.
void weight_gradient(const torch::Tensor &grad, const torch::Tensor &input, const torch::Tensor &scale, const torch::Tensor &splits, const torch::Tensor &out,
                     bool accumulate) {
  const c10::DeviceGuard guard(grad.device());
  const int32_t experts = static_cast<int32_t>(splits.size(0));
  const size_t ws_bytes = fluxmi_moe_wgrad_workspace_bytes(experts, grad.size(0), grad.size(1), input.size(1));
  torch::Tensor ws;
  if (ws_bytes > 0) ws = empty_on(grad, {static_cast<int64_t>(ws_bytes)}, at::kByte);
  check_status(fluxmi_moe_wgrad(grad.data_ptr(), input.data_ptr(), scale.defined() ? scale.data_ptr() : nullptr, row_type(grad), splits.data_ptr<int32_t>(),
                                experts, grad.size(0), grad.size(1), input.size(1), out.data_ptr(),
                                out.scalar_type() == at::kFloat ? FLUXMI_ROWS_FP32 : row_type(out), accumulate, ws_bytes > 0 ? ws.data_ptr() : nullptr, ws_bytes,
                                current_stream()),
               "fluxmi_moe_wgrad");
}

torch::Tensor weight_gradient_like(const torch::Tensor &grad, const torch::Tensor &input, const torch::Tensor &scale, const torch::Tensor &splits) {
  torch::Tensor out = empty_on(grad, {splits.size(0), grad.size(1), input.size(1)}, grad.scalar_type());
  weight_gradient(grad, input, scale, splits, out, false);
  return out;
}

using Kept = std::tuple<torch::Tensor, torch::Tensor>;

Kept keep(const torch::Tensor &input) {
  const c10::DeviceGuard guard(input.device());
  torch::Tensor codes = empty_on(input, input.sizes(), kCodes), scale = empty_on(input, {input.size(0), blocks_of(input.size(1))}, kScales);
  check_status(fluxmi_checkpoint_e4m3(input.data_ptr(), row_type(input), input.size(0), input.size(1), codes.data_ptr(), scale.data_ptr(), current_stream()),
               "fluxmi_checkpoint_e4m3");
  return {codes, scale};
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> swiglu(const torch::Tensor &input, bool kept) {
  const c10::DeviceGuard guard(input.device());
  const int64_t rows = input.size(0), cols = input.size(1) / 2;
  torch::Tensor out = empty_on(input, {rows, cols}, input.scalar_type()), codes, scale;
  if (kept) {
    codes = empty_on(input, {rows, 2 * cols}, kCodes);
    scale = empty_on(input, {rows, 2 * blocks_of(cols)}, kScales);
  }
  check_status(fluxmi_swiglu(input.data_ptr(), row_type(input), rows, cols, out.data_ptr(), kept ? codes.data_ptr() : nullptr, kept ? scale.data_ptr() : nullptr,
                             current_stream()),
               "fluxmi_swiglu");
  return {out, codes, scale};
}

// The second result is undefined unless asked for.
std::tuple<torch::Tensor, torch::Tensor> swiglu_gradient(const torch::Tensor &grad, const torch::Tensor &input, const torch::Tensor &scale, bool want_out) {
  const c10::DeviceGuard guard(grad.device());
  torch::Tensor grad_input = empty_on(grad, input.sizes(), grad.scalar_type()), out;
  if (want_out) out = empty_on(grad, grad.sizes(), grad.scalar_type());
  check_status(fluxmi_swiglu_backward(grad.data_ptr(), input.data_ptr(), scale.defined() ? scale.data_ptr() : nullptr, row_type(grad), grad.size(0), grad.size(1),
                                      grad_input.data_ptr(), want_out ? out.data_ptr() : nullptr, current_stream()),
               "fluxmi_swiglu_backward");
  return {grad_input, out};
}

// The activation alone, from what swiglu_gradient has it from.
torch::Tensor activation(const torch::Tensor &input, const torch::Tensor &scale, at::ScalarType dtype) {
  const c10::DeviceGuard guard(input.device());
  torch::Tensor out = empty_on(input, {input.size(0), input.size(1) / 2}, dtype);
  check_status(fluxmi_swiglu_backward(nullptr, input.data_ptr(), scale.defined() ? scale.data_ptr() : nullptr, row_type(out), out.size(0), out.size(1), nullptr, out.data_ptr(),
                                      current_stream()),
               "fluxmi_swiglu_backward");
  return out;
}

// ---- autograd -------------------------------------------------------------------------------------------------

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

torch::Tensor incoming(const char *who, const variable_list &grads) {
  refuse_second_derivative(who, grads[0]);
  refuse_leaves_of_another_stream(who);
  return grads[0].resolve_neg().contiguous();
}

// What the backward pass keeps of an activation: itself, or codes and scale.
Kept kept_of(const torch::Tensor &t, bool wanted, bool checkpoint) {
  if (!wanted) return {};
  if (!checkpoint) return {t, torch::Tensor()};
  return keep(t);
}

struct Linear : torch::autograd::Function<Linear> {
  static torch::Tensor forward(AutogradContext *ctx, const torch::Tensor &input, const torch::Tensor &weight, const torch::Tensor &splits, bool checkpoint) {
    const auto [x, x_scale] = kept_of(input, weight.requires_grad(), checkpoint);
    ctx->save_for_backward({splits, x, x_scale, input.requires_grad() ? weight : torch::Tensor()});
    return product(input, weight, splits);
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const torch::Tensor grad = incoming("moe_linear", grads);
    const auto saved = ctx->get_saved_variables();
    const torch::Tensor &splits = saved[0], &x = saved[1], &x_scale = saved[2], &weight = saved[3];
    return {ctx->needs_input_grad(0) ? input_gradient(grad, weight, splits) : torch::Tensor(),
            ctx->needs_input_grad(1) ? weight_gradient_like(grad, x, x_scale, splits) : torch::Tensor(), {}, {}};
  }
};

struct Swiglu : torch::autograd::Function<Swiglu> {
  static torch::Tensor forward(AutogradContext *ctx, const torch::Tensor &input, bool checkpoint) {
    const auto [out, codes, scale] = swiglu(input, checkpoint);
    ctx->save_for_backward({checkpoint ? codes : input, scale});
    return out;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const torch::Tensor grad = incoming("moe_swiglu", grads);
    const auto saved = ctx->get_saved_variables();
    return {std::get<0>(swiglu_gradient(grad, saved[0], saved[1], false)), {}};
  }
};

// The same with the codes and scales among the results, which have no gradients of their own.
struct SwigluKept : torch::autograd::Function<SwigluKept> {
  static variable_list forward(AutogradContext *ctx, const torch::Tensor &input) {
    const auto [out, codes, scale] = swiglu(input, true);
    ctx->mark_non_differentiable({codes, scale});
    ctx->set_materialize_grads(false);  // (theirs would be zeros of 8 bits)
    ctx->save_for_backward({codes, scale});
    return {out, codes, scale};
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    if (!grads[0].defined()) return {torch::Tensor()};
    const torch::Tensor grad = incoming("moe_swiglu_checkpoint", grads);
    const auto saved = ctx->get_saved_variables();
    return {std::get<0>(swiglu_gradient(grad, saved[0], saved[1], false))};
  }
};

// Of what lies between the two products the backward pass keeps the activation's input alone; its output is computed again beside the gradient.  A backward pass may be asked for fewer
// gradients than the forward pass kept for (torch.autograd.grad), and computes those.
struct Mlp : torch::autograd::Function<Mlp> {
  static torch::Tensor forward(AutogradContext *ctx, const torch::Tensor &input, const torch::Tensor &weight1, const torch::Tensor &weight2,
                               const torch::Tensor &splits, bool checkpoint) {
    const bool below = input.requires_grad() || weight1.requires_grad();
    const auto [x, x_scale] = kept_of(input, weight1.requires_grad(), checkpoint);
    const torch::Tensor hidden = product(input, weight1, splits);
    const auto [act, codes, scale] = swiglu(hidden, checkpoint);
    ctx->save_for_backward({splits, x, x_scale, checkpoint ? codes : hidden, scale, input.requires_grad() ? weight1 : torch::Tensor(), below ? weight2 : torch::Tensor()});
    return product(act, weight2, splits);
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const torch::Tensor grad = incoming("moe_mlp", grads);
    const auto saved = ctx->get_saved_variables();
    const torch::Tensor &splits = saved[0], &x = saved[1], &x_scale = saved[2], &hidden = saved[3], &scale = saved[4], &weight1 = saved[5], &weight2 = saved[6];
    const bool want_input = ctx->needs_input_grad(0), want_weight1 = ctx->needs_input_grad(1), want_weight2 = ctx->needs_input_grad(2);
    torch::Tensor grad_hidden, act, grad_input, grad_weight1, grad_weight2;
    // (the second weights' gradient alone takes the activation, but no gradient of its input, which comes through those weights)
    if (want_input || want_weight1) std::tie(grad_hidden, act) = swiglu_gradient(input_gradient(grad, weight2, splits), hidden, scale, want_weight2);
    else if (want_weight2) act = activation(hidden, scale, grad.scalar_type());
    if (want_weight2) grad_weight2 = weight_gradient_like(grad, act, {}, splits);
    if (want_weight1) grad_weight1 = weight_gradient_like(grad_hidden, x, x_scale, splits);
    if (want_input) grad_input = input_gradient(grad_hidden, weight1, splits);
    return {grad_input, grad_weight1, grad_weight2, {}, {}};
  }
};

}  // namespace

torch::Tensor moe_linear(torch::Tensor input, torch::Tensor weight, torch::Tensor splits, bool checkpoint) {
  check_operand(input, "input", 2);
  check_weight(weight, "weight", input, "input", 2);
  TORCH_CHECK(weight.size(2) > 0, "weight must have columns");
  check_splits(splits, input, weight.size(0));
  const c10::DeviceGuard guard(input.device());
  const torch::Tensor counts = on_device(splits, input);
  if (at::GradMode::is_enabled() && (input.requires_grad() || weight.requires_grad())) return Linear::apply(input, weight, counts, checkpoint);
  return product(input, weight, counts);
}

torch::Tensor moe_swiglu(torch::Tensor input, bool checkpoint) {
  check_operand(input, "input", 2);
  TORCH_CHECK(input.size(1) % 2 == 0, "input must have gate and up columns, got ", input.size(1));
  if (at::GradMode::is_enabled() && input.requires_grad()) return Swiglu::apply(input, checkpoint);
  return std::get<0>(swiglu(input, false));
}

torch::Tensor moe_mlp(torch::Tensor input, torch::Tensor weight1, torch::Tensor weight2, torch::Tensor splits, bool checkpoint) {
  check_operand(input, "input", 2);
  check_weight(weight1, "weight1", input, "input", 2);
  check_operand(weight2, "weight2", 3);
  check_like(weight2, "weight2", input, "input");
  TORCH_CHECK(weight1.size(2) > 0 && weight2.size(2) > 0, "weights must have columns");
  TORCH_CHECK(weight1.size(0) == weight2.size(0), "weight1 has ", weight1.size(0), " experts, weight2 ", weight2.size(0));
  TORCH_CHECK(weight1.size(1) == 2 * weight2.size(2), "weight1 must have gate and up rows for each column of weight2: ", weight1.size(1), " != 2 * ", weight2.size(2));
  check_splits(splits, input, weight1.size(0));
  const c10::DeviceGuard guard(input.device());
  const torch::Tensor counts = on_device(splits, input);
  if (at::GradMode::is_enabled() && (input.requires_grad() || weight1.requires_grad() || weight2.requires_grad()))
    return Mlp::apply(input, weight1, weight2, counts, checkpoint);
  return product(std::get<0>(swiglu(product(input, weight1, counts), false)), weight2, counts);
}

torch::Tensor moe_dgrad(torch::Tensor grad, torch::Tensor weight, torch::Tensor splits) {
  check_operand(grad, "grad", 2);
  check_weight(weight, "weight", grad, "grad", 1);
  check_splits(splits, grad, weight.size(0));
  const c10::DeviceGuard guard(grad.device());
  return input_gradient(grad, weight, on_device(splits, grad));
}

torch::Tensor moe_wgrad(torch::Tensor grad, torch::Tensor input, torch::Tensor splits, std::optional<torch::Tensor> input_scale,
                        std::optional<torch::Tensor> output, bool accumulate, std::optional<at::ScalarType> output_dtype) {
  check_operand(grad, "grad", 2);
  if (input_scale.has_value()) {
    check_kept(input, *input_scale, grad, 1);
  } else {
    check_operand(input, "input", 2);
    check_like(input, "input", grad, "grad");
  }
  TORCH_CHECK(input.size(0) == grad.size(0), "input has ", input.size(0), " rows, grad ", grad.size(0));
  check_splits(splits, grad, -1);
  const at::ScalarType out_type = output.has_value() ? output->scalar_type() : output_dtype.value_or(grad.scalar_type());
  TORCH_CHECK(out_type == grad.scalar_type() || out_type == at::kFloat, "the weights' gradient can be ", grad.scalar_type(), " or float32, got ", out_type);
  TORCH_CHECK(!output.has_value() || output_dtype.value_or(out_type) == out_type, "output is ", out_type, ", output_dtype ", output_dtype.value_or(out_type));
  TORCH_CHECK(output.has_value() || !accumulate, "accumulate needs an output");
  const c10::DeviceGuard guard(grad.device());
  torch::Tensor out;
  if (output.has_value()) {
    out = *output;
    refuse_tangent(out, "output");
    refuse_lazy_view(out, "output");
    FLUX_AMD_CHECK_INPUT(out, out_type);
    FLUX_AMD_CHECK_3D(out, splits.size(0), grad.size(1), input.size(1));
    TORCH_CHECK(out.device() == grad.device(), "output is on ", out.device(), ", grad is on ", grad.device());
    TORCH_CHECK(!at::GradMode::is_enabled() || !out.requires_grad(), "output requires a gradient: write it under no_grad()");
    for (const torch::Tensor &t : {grad, input, splits, input_scale.value_or(splits)})
      TORCH_CHECK(at::get_overlap_status(out, t) == at::MemOverlapStatus::No, "output lies in the memory of an operand");
  } else {
    out = empty_on(grad, {splits.size(0), grad.size(1), input.size(1)}, out_type);
  }
  weight_gradient(grad, input, input_scale.value_or(torch::Tensor()), on_device(splits, grad), out, accumulate);
  if (output.has_value() && !out.is_inference()) torch::autograd::impl::bump_version(out);
  return out;
}

std::tuple<torch::Tensor, torch::Tensor> moe_checkpoint(torch::Tensor input) {
  check_operand(input, "input", 2);
  return keep(input);
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> moe_swiglu_checkpoint(torch::Tensor input) {
  check_operand(input, "input", 2);
  TORCH_CHECK(input.size(1) % 2 == 0, "input must have gate and up columns, got ", input.size(1));
  if (at::GradMode::is_enabled() && input.requires_grad()) {
    const variable_list results = SwigluKept::apply(input);
    return {results[0], results[1], results[2]};
  }
  return swiglu(input, true);
}

std::tuple<torch::Tensor, torch::Tensor> moe_swiglu_backward(torch::Tensor grad, torch::Tensor input, std::optional<torch::Tensor> input_scale) {
  check_operand(grad, "grad", 2);
  if (input_scale.has_value()) {
    TORCH_CHECK(input.dim() == 2 && input.size(1) % 2 == 0, "input must have gate and up columns, got ", input.sizes());
    check_kept(input, *input_scale, grad, 2);
  } else {
    check_operand(input, "input", 2);
    check_like(input, "input", grad, "grad");
  }
  FLUX_AMD_CHECK_2D(input, grad.size(0), 2 * grad.size(1));
  return swiglu_gradient(grad, input, input_scale.value_or(torch::Tensor()), true);
}

}  // namespace flux_amd
