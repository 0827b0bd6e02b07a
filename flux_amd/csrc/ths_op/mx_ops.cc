// Microscaled 4-bit floating point: Quantization::quantize_mx / dequantize_mx and MxGemm.  No counterpart in the reference; the classes follow
// Quantization (src/quantization/ths_op/quantization.cc) and BlockScaleGemm (src/comm_none/ths_op/blockscale_gemm.cc).
#include <c10/core/DeviceGuard.h>

#include "ths_ops.h"

namespace flux_amd {
namespace {

constexpr at::ScalarType kCodes = at::ScalarType::Float4_e2m1fn_x2, kScales = at::ScalarType::Float8_e8m0fnu;
constexpr int64_t kMxBlock = 32;

int64_t blocks_of(int64_t cols) { return (cols + kMxBlock - 1) / kMxBlock; }

int32_t mx_type(at::ScalarType st) { return st == at::kBFloat16 ? FLUXMI_ROWS_BF16 : st == at::kFloat ? FLUXMI_ROWS_FP32 : FLUXMI_ROWS_FP16; }

// Codes [..., rows, 16 kb] and scales [..., rows, kb] of one operand.
void check_operand(const torch::Tensor &codes, const torch::Tensor &scale, const char *name, int64_t dims) {
  TORCH_CHECK(codes.is_cuda() && scale.is_cuda(), name, " and its scale must be device tensors");
  TORCH_CHECK(codes.scalar_type() == kCodes, name, " must be float4_e2m1fn_x2, got ", codes.scalar_type());
  TORCH_CHECK(scale.scalar_type() == kScales, name, "'s scale must be float8_e8m0fnu, got ", scale.scalar_type());
  TORCH_CHECK(codes.dim() == dims && scale.dim() == dims, name, " and its scale must have ", dims, " dimensions, got ", codes.dim(), " and ", scale.dim());
  TORCH_CHECK(codes.is_contiguous() && scale.is_contiguous(), name, " and its scale must be contiguous");
  TORCH_CHECK(codes.device() == scale.device(), name, " is on ", codes.device(), ", its scale on ", scale.device());
  bool fits = codes.size(-1) == scale.size(-1) * (kMxBlock / 2);
  for (int64_t d = 0; d + 1 < dims; ++d) fits = fits && codes.size(d) == scale.size(d);
  TORCH_CHECK(fits, name, " shape mismatch: codes ", codes.sizes(), " take scales of 1 for every 16 bytes, got ", scale.sizes());
}

}  // namespace

Quantization::Result Quantization::quantize_mx(torch::Tensor input, bool return_transpose) {
  TORCH_CHECK(output_dtype_ == kCodes, "quantize_mx needs a Quantization whose output dtype is float4_e2m1fn_x2, this one's is ", output_dtype_);
  TORCH_CHECK(input.dim() == 2 || input.dim() == 3, "Input must have 2 or 3 dimensions.");
  FLUX_AMD_CHECK_INPUT(input, input_dtype_);
  const c10::DeviceGuard guard(input.device());
  const bool batched = input.dim() == 3;
  const int64_t batch = batched ? input.size(0) : 1, rows = input.size(-2), cols = input.size(-1);
  auto make = [&](int64_t r, int64_t c, at::ScalarType st) {
    return batched ? empty_on(input, {batch, r, c}, st) : empty_on(input, {r, c}, st);
  };
  torch::Tensor codes = make(rows, blocks_of(cols) * 16, kCodes), scale = make(rows, blocks_of(cols), kScales);
  std::optional<torch::Tensor> codes_t, scale_t;
  if (return_transpose) {
    codes_t = make(cols, blocks_of(rows) * 16, kCodes);
    scale_t = make(cols, blocks_of(rows), kScales);
  }
  // Without the transposed copy the batch is so many rows more.
  const int64_t matrices = return_transpose ? batch : 1;
  check_status(fluxmi_quant_mx(input.data_ptr(), mx_type(input_dtype_), matrices, return_transpose ? rows : batch * rows, cols, codes.data_ptr(), scale.data_ptr(),
                               return_transpose ? codes_t->data_ptr() : nullptr, return_transpose ? scale_t->data_ptr() : nullptr, current_stream()),
               "fluxmi_quant_mx");
  return {codes, scale, codes_t, scale_t};
}

torch::Tensor Quantization::dequantize_mx(torch::Tensor codes, torch::Tensor scale, std::optional<int64_t> cols) {
  TORCH_CHECK(output_dtype_ == kCodes, "dequantize_mx needs a Quantization whose output dtype is float4_e2m1fn_x2, this one's is ", output_dtype_);
  TORCH_CHECK(codes.dim() == 2 || codes.dim() == 3, "codes must have 2 or 3 dimensions.");
  check_operand(codes, scale, "codes", codes.dim());
  const int64_t kb = scale.size(-1), n = cols.value_or(kb * kMxBlock);
  TORCH_CHECK(n >= 0 && blocks_of(n) == kb, "cols=", n, " does not end in the last of ", kb, " blocks of 32");
  const c10::DeviceGuard guard(codes.device());
  std::vector<int64_t> shape = codes.sizes().vec();
  shape.back() = n;
  torch::Tensor out = empty_on(codes, shape, input_dtype_);
  check_status(fluxmi_dequant_mx(codes.data_ptr(), scale.data_ptr(), codes.dim() == 3 ? codes.size(0) * codes.size(1) : codes.size(0), n, mx_type(input_dtype_),
                                 out.data_ptr(), current_stream()),
               "fluxmi_dequant_mx");
  return out;
}

MxGemm::MxGemm(at::ScalarType output_dtype) : output_dtype_(output_dtype) {
  TORCH_CHECK(output_dtype == at::kBFloat16 || output_dtype == at::kHalf || output_dtype == at::kFloat,
              "MxGemm: output dtype must be bfloat16, float16 or float32, got ", output_dtype);
}

static torch::Tensor mx_run(const torch::Tensor &input, const torch::Tensor &input_scale, const torch::Tensor &weight, const torch::Tensor &weight_scale, int64_t nexperts,
                            int64_t max_rows, const torch::Tensor *splits, const std::optional<torch::Tensor> &gather_index, const std::optional<torch::Tensor> &row_scale,
                            std::optional<torch::Tensor> output, at::ScalarType out_dtype) {
  const c10::DeviceGuard guard(input.device());
  const int64_t n = weight.size(-2);
  auto on_device = [&](const torch::Tensor &t, const char *name) {
    TORCH_CHECK(t.device() == input.device(), name, " is on ", t.device(), ", input is on ", input.device());
  };
  on_device(weight, "weight");
  TORCH_CHECK(weight.size(-1) == input.size(-1), "weight 2-dim mismatch: ", weight.size(-1), " != ", input.size(-1), " bytes of codes");
  TORCH_CHECK(input.size(1) > 0, "K must be positive");
  for (int64_t v : {max_rows, n, input.size(0), input.size(1) * 2}) TORCH_CHECK(v <= INT32_MAX, "a size exceeds 2^31 - 1: ", v);
  torch::Tensor out;
  if (output.has_value()) {
    out = *output;
    FLUX_AMD_CHECK_INPUT(out, out_dtype);
    FLUX_AMD_CHECK_2D(out, max_rows, n);
    on_device(out, "output");
  } else {
    out = empty_on(input, {max_rows, n}, out_dtype);
  }
  fluxmi_mx_gemm_args args{};
  if (gather_index.has_value()) {
    FLUX_AMD_CHECK_INPUT(*gather_index, at::kInt);
    FLUX_AMD_CHECK_NDIM(*gather_index, 1);
    on_device(*gather_index, "gather_index");
    TORCH_CHECK(max_rows == 0 || input.size(0) > 0, "gather_index names rows of an empty input");
    args.gather_a = gather_index->data_ptr<int32_t>();
  }
  if (row_scale.has_value()) {
    FLUX_AMD_CHECK_INPUT(*row_scale, at::kFloat);
    on_device(*row_scale, "row_scale");
    TORCH_CHECK(row_scale->dim() == 1 && row_scale->size(0) == max_rows, "row_scale must be [", max_rows, "], got ", row_scale->sizes());
    args.row_scale = row_scale->data_ptr<float>();
  }
  args.nexperts = static_cast<int32_t>(nexperts);
  args.max_rows = static_cast<int32_t>(max_rows);
  args.n = static_cast<int32_t>(n);
  args.k = static_cast<int32_t>(input.size(1) * 2);
  args.a_rows = static_cast<int32_t>(input.size(0));
  args.d_type = mx_type(out_dtype);
  args.a = input.data_ptr();
  args.a_scale = input_scale.data_ptr();
  args.b = weight.data_ptr();
  args.b_scale = weight_scale.data_ptr();
  args.d = out.data_ptr();
  if (splits != nullptr) args.splits = splits->data_ptr<int32_t>();
  const size_t ws_bytes = fluxmi_grouped_gemm_mx_workspace_bytes(&args);
  torch::Tensor ws;
  if (ws_bytes > 0) ws = empty_on(input, {static_cast<int64_t>(ws_bytes)}, at::kByte);
  check_status(fluxmi_grouped_gemm_mx(&args, ws_bytes > 0 ? ws.data_ptr() : nullptr, ws_bytes, current_stream()), "fluxmi_grouped_gemm_mx");
  return out;
}

torch::Tensor MxGemm::forward(torch::Tensor input, torch::Tensor weight, torch::Tensor input_scale, torch::Tensor weight_scale,
                              std::optional<torch::Tensor> output) {
  check_operand(input, input_scale, "input", 2);
  check_operand(weight, weight_scale, "weight", 2);
  return mx_run(input, input_scale, weight, weight_scale, 1, input.size(0), nullptr, std::nullopt, std::nullopt, output, output_dtype_);
}

torch::Tensor MxGemm::forward_grouped(torch::Tensor input, torch::Tensor input_splits, torch::Tensor weight, torch::Tensor input_scale, torch::Tensor weight_scale,
                                      std::optional<torch::Tensor> gather_index, std::optional<torch::Tensor> row_scale, std::optional<torch::Tensor> output) {
  check_operand(input, input_scale, "input", 2);
  check_operand(weight, weight_scale, "weight", 3);
  FLUX_AMD_CHECK_NDIM(input_splits, 1);
  TORCH_CHECK(input_splits.scalar_type() == at::kInt, "input_splits must be int32, got ", input_splits.scalar_type());
  TORCH_CHECK(input_splits.is_contiguous(), "input_splits must be contiguous");
  TORCH_CHECK(input_splits.size(0) == weight.size(0), "splits 0-dim mismatch: ", input_splits.size(0), " != ", weight.size(0));
  TORCH_CHECK(input_splits.is_cuda() ? input_splits.device() == input.device() : input_splits.device().is_cpu(), "input_splits must be on the host or on ",
              input.device());
  const int64_t max_rows = gather_index.has_value() ? gather_index->numel() : input.size(0);
  if (!input_splits.is_cuda()) {
    // Counts in pinned memory are not looked at here: a copy that the stream has yet to run may be about to write them, and the copy below, which
    // comes after it, sees what it wrote.  (The kernels compute no rows past max_rows whatever the counts.)
    TORCH_CHECK(input_splits.is_pinned() || input_splits.sum().item<int64_t>() <= max_rows, "input_splits sum exceeds the rows of the product");
    input_splits = input_splits.to(input.device(), /*non_blocking=*/true);
  }
  return mx_run(input, input_scale, weight, weight_scale, weight.size(0), max_rows, &input_splits, gather_index, row_scale, output, output_dtype_);
}

}  // namespace flux_amd
