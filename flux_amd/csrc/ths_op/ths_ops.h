// Declarations of the operator classes and free functions bound in pybind.cc.
#pragma once
#include "ths_common.h"

namespace flux_amd {

class GemmGroupedV3AGScatter {
 public:
  GemmGroupedV3AGScatter(DistEnvTPWithEP tp_env, MoeArguments moe_args);
  void clear_buffers();
  torch::Tensor forward(torch::Tensor inputs_shard, torch::Tensor weights, torch::Tensor splits_gpu,
                        torch::Tensor scatter_index, std::optional<torch::Tensor> output_scale,
                        std::optional<torch::Tensor> outputs_buf, std::optional<torch::Tensor> allgather_output,
                        bool fast_accum, int64_t sm_margin);
  std::vector<torch::Tensor> forward_multiple_weights(
      torch::Tensor inputs_shard, std::vector<torch::Tensor> weights, torch::Tensor splits_gpu,
      torch::Tensor scatter_index, std::optional<std::vector<torch::Tensor>> output_scale,
      std::optional<std::vector<torch::Tensor>> outputs_buf, std::optional<torch::Tensor> allgather_output,
      bool fast_accum, int64_t sm_margin);
  // forward() under every tile schedule, timed; the fastest is registered for the shape and recorded in
  // prof_ctx (gemm_grouped_v3_ag_scatter.cc:520-612).
  torch::Tensor profiling(torch::Tensor inputs_shard, torch::Tensor weights, torch::Tensor splits_gpu,
                          torch::Tensor scatter_index, std::optional<torch::Tensor> output_scale,
                          std::optional<torch::Tensor> outputs_buf, std::optional<torch::Tensor> allgather_output,
                          bool fast_accum, int64_t sm_margin, std::shared_ptr<ProfilingContext> prof_ctx);

 private:
  std::vector<torch::Tensor> forward_impl(torch::Tensor inputs_shard, std::vector<torch::Tensor> weights,
                                          torch::Tensor splits_gpu, torch::Tensor scatter_index,
                                          std::optional<std::vector<torch::Tensor>> output_scale,
                                          std::optional<std::vector<torch::Tensor>> outputs_buf,
                                          std::optional<torch::Tensor> allgather_output, bool fast_accum,
                                          int64_t sm_margin);
  DistEnvTPWithEP tp_env_;
  MoeArguments moe_args_;
  torch::Tensor gather_index_;
};

class GemmGroupedV3GatherRS {
 public:
  GemmGroupedV3GatherRS(int64_t total_num_experts, int64_t max_m, int64_t n_dim, int64_t topk, int64_t rank,
                        int64_t world_size, int64_t tp_world_size, int64_t ep_world_size,
                        int64_t max_input_groups, bool ep_in_dp);
  torch::Tensor forward_gather_rs(torch::Tensor input, torch::Tensor weight, torch::Tensor splits_cpu,
                                  torch::Tensor routing_idx, std::optional<torch::Tensor> n_tokens_per_rank,
                                  std::optional<torch::Tensor> input_scale,
                                  std::optional<torch::Tensor> weight_scale,
                                  std::optional<torch::Tensor> output_vec_scale, bool fast_accum,
                                  int64_t sm_margin, bool with_stream_sync);
  torch::Tensor forward_gather_rs_multiple(std::vector<torch::Tensor> inputs, std::vector<torch::Tensor> weights,
                                           torch::Tensor splits_cpu, torch::Tensor routing_idx,
                                           std::optional<torch::Tensor> n_tokens_per_rank,
                                           std::optional<std::vector<torch::Tensor>> input_scale,
                                           std::optional<std::vector<torch::Tensor>> weight_scale,
                                           std::optional<std::vector<torch::Tensor>> output_vec_scale,
                                           bool fast_accum, int64_t sm_margin, bool with_stream_sync);
  void ep_zero_buffer() {}  // expert-parallel scratch does not exist at world size 1
  // forward_gather_rs() under every tile schedule, timed; the fastest is registered for the shape and
  // recorded in prof_ctx (gemm_grouped_v3_gather_rs.cc:903-1000).
  torch::Tensor profiling(torch::Tensor input, torch::Tensor weight, torch::Tensor splits_cpu,
                          torch::Tensor routing_idx, std::optional<torch::Tensor> n_tokens_per_rank,
                          std::optional<torch::Tensor> input_scale, std::optional<torch::Tensor> weight_scale,
                          std::optional<torch::Tensor> output_vec_scale, bool fast_accum, int64_t sm_margin,
                          bool with_stream_sync, std::shared_ptr<ProfilingContext> prof_ctx);

 private:
  torch::Tensor forward_impl(std::vector<torch::Tensor> inputs, std::vector<torch::Tensor> weights,
                             torch::Tensor splits_cpu, torch::Tensor routing_idx,
                             std::optional<std::vector<torch::Tensor>> input_scale,
                             std::optional<std::vector<torch::Tensor>> weight_scale,
                             std::optional<std::vector<torch::Tensor>> output_vec_scale, bool with_stream_sync,
                             int64_t sm_margin);
  void lazy_init(const torch::Tensor &like);
  int64_t num_experts_, max_m_, n_dim_, topk_, max_input_groups_;
  bool inter_fp32_ = true;

 public:
  // Dtype of the intermediate between the GEMM and the reduction: fp32 (one rounding in the layer) or the 16-bit
  // output type (the reference's inter_D).  Only before the first forward: the buffers are allocated lazily.
  void set_intermediate_fp32(bool fp32) {
    TORCH_CHECK(inter_.empty(), "the intermediate's dtype is fixed once the op has run");
    inter_fp32_ = fp32;
  }

 private:
  int fused_mode_ = 0;  // 0: by shape, 1: always the fused epilogue reduce, 2: always GEMM + gather-reduce
  std::vector<torch::Tensor> inter_;
  torch::Tensor splits_dev_;
  torch::Tensor token_of_row_;  // inverse of routing_idx (the token of each sorted row), for the fused reduce
};

class GemmGroupedV3 {
 public:
  GemmGroupedV3(torch::Tensor weight, int64_t num_experts);
  torch::Tensor forward(torch::Tensor input, torch::Tensor splits_cpu);

 private:
  torch::Tensor weight_;
};

// Block-scaled fp8 GEMM of the reference (src/comm_none/ths_op/blockscale_gemm.h:24-94): the forward
// products, dense and grouped (forward_multistream is the same single launch).  The wgrad* methods (training-time
// weight gradients) are not on this path and are not built.
class BlockScaleGemm {
 public:
  BlockScaleGemm(at::ScalarType input_dtype, at::ScalarType weight_dtype, at::ScalarType output_dtype,
                 int32_t num_streams);
  // input [M, K] e4m3, weight [N, K] e4m3, input_scale [ceil(M/128), K/128, 128] (what
  // Quantization::quantize_vector_blockwise returns), weight_scale [ceil(N/128), K/128].
  torch::Tensor forward(torch::Tensor input, torch::Tensor weight, std::optional<torch::Tensor> bias,
                        std::optional<torch::Tensor> output, std::optional<torch::Tensor> input_scale,
                        std::optional<torch::Tensor> weight_scale);
  // input [M, K] sorted by expert, input_splits host [E], weight [E, N, K].  Scales either in the reference's
  // operand layouts (1-D tensors: per expert [K/128, M_e] back to back; per expert [K/128, N/128]:
  // blockscale_gemm.cc:703-722) or as the quantisation ops return them (3-D tensors: input_scale
  // [ceil(M/128), K/128, 128] over the sorted rows, weight_scale [E, N/128, K/128]).
  torch::Tensor forward_grouped(torch::Tensor input, torch::Tensor input_splits, torch::Tensor weight,
                                std::optional<torch::Tensor> bias, std::optional<torch::Tensor> output,
                                torch::Tensor input_scale, torch::Tensor weight_scale);
  // The grouped product with input_scale as [M, K/128] (any strides) and weight_scale [E, N/128, K/128]: the
  // arguments of the reference's multi-stream form; one launch here.
  torch::Tensor forward_multistream(torch::Tensor input, torch::Tensor input_splits, torch::Tensor weight,
                                    std::optional<torch::Tensor> bias, std::optional<torch::Tensor> output,
                                    std::optional<torch::Tensor> input_scale, std::optional<torch::Tensor> weight_scale);
  torch::Tensor reference(torch::Tensor input, torch::Tensor weight, std::optional<torch::Tensor> bias,
                          std::optional<torch::Tensor> output, std::optional<torch::Tensor> input_scale,
                          std::optional<torch::Tensor> weight_scale, bool is_groupwise_b);
  torch::Tensor profiling(torch::Tensor input, torch::Tensor weight, std::optional<torch::Tensor> bias,
                          std::optional<torch::Tensor> output, std::optional<torch::Tensor> input_scale,
                          std::optional<torch::Tensor> weight_scale, std::shared_ptr<ProfilingContext> prof_ctx);

 private:
  at::ScalarType input_dtype_, weight_dtype_, output_dtype_;
};

class Quantization {
 public:
  using Result = std::tuple<torch::Tensor, torch::Tensor, std::optional<torch::Tensor>, std::optional<torch::Tensor>>;
  Quantization(at::ScalarType input_dtype, at::ScalarType output_dtype, int32_t num_streams);
  Result quantize_vector_blockwise(torch::Tensor input, bool return_transpose, float eps);
  Result quantize_square_blockwise(torch::Tensor input, bool return_transpose, float eps);
  Result batch_quantize_square_blockwise(torch::Tensor input, bool return_transpose, float eps);
  std::tuple<torch::Tensor, torch::Tensor> quantize_rowwise(torch::Tensor input, float eps);
  // MXFP4, for output dtype float4_e2m1fn_x2 (mx_ops.cc): input [rows, cols] or [batch, rows, cols] of the input dtype -> codes [.., rows,
  // 16 kb] (two a byte), scales float8_e8m0fnu [.., rows, kb], kb = ceil(cols / 32), and with return_transpose the same of the
  // transposed matrices.
  Result quantize_mx(torch::Tensor input, bool return_transpose);
  // The values that codes and scales stand for, in the input dtype; cols: the row's length where the last block is not full.
  torch::Tensor dequantize_mx(torch::Tensor codes, torch::Tensor scale, std::optional<int64_t> cols);

 private:
  void require_e4m3(const char *method) const;
  at::ScalarType input_dtype_, output_dtype_;
};

// Products of MXFP4 operands as quantize_mx returns them, one launch on the current stream (mx_ops.cc).
class MxGemm {
 public:
  explicit MxGemm(at::ScalarType output_dtype);
  // input [M, K/2], weight [N, K/2], scales [M, K/32] and [N, K/32] -> [M, N].
  torch::Tensor forward(torch::Tensor input, torch::Tensor weight, torch::Tensor input_scale, torch::Tensor weight_scale, std::optional<torch::Tensor> output);
  // Rows sorted by expert; input_splits int32 [E] on the device or on the host, weight [E, N, K/2], weight_scale [E, N, K/32].  gather_index int32
  // [M]: the row of input that a sorted row reads; row_scale fp32 [M]: a factor of each sorted row.  Rows past the splits' sum are not touched.
  torch::Tensor forward_grouped(torch::Tensor input, torch::Tensor input_splits, torch::Tensor weight, torch::Tensor input_scale, torch::Tensor weight_scale,
                                std::optional<torch::Tensor> gather_index, std::optional<torch::Tensor> row_scale, std::optional<torch::Tensor> output);

 private:
  at::ScalarType output_dtype_;
};

torch::Tensor calc_scatter_index(torch::Tensor choosed_experts, torch::Tensor splits);
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor> moe_route_sort(torch::Tensor choosed_experts,
                                                                                      int64_t nexperts);
torch::Tensor topk_scatter_reduce(std::vector<torch::Tensor> inputs, torch::Tensor scatter_idx, int64_t topk);
torch::Tensor topk_weighted_gather_reduce(std::vector<torch::Tensor> inputs, torch::Tensor routing_idx,
                                          int64_t topk, std::optional<torch::Tensor> row_weight, double scale);
// Tokens to the rows of their experts and back (permute_ops.cc).  scatter_index int32 [tokens, topk], as calc_scatter_index gives it; entries
// outside [0, tokens * topk) are dropped pairs, the others are distinct.  Both are differentiable once; the *_backward functions are the same
// gradients for callers without autograd.
torch::Tensor moe_permute(torch::Tensor input, torch::Tensor scatter_index);
torch::Tensor moe_permute_backward(torch::Tensor grad_rows, torch::Tensor scatter_index);
torch::Tensor moe_unpermute(torch::Tensor rows, torch::Tensor scatter_index, std::optional<torch::Tensor> weights);
std::tuple<torch::Tensor, torch::Tensor> moe_unpermute_backward(torch::Tensor grad_out, torch::Tensor rows, torch::Tensor scatter_index,
                                                                torch::Tensor weights);

// Experts that learn (expert_grad_ops.cc).  Rows are sorted by expert, weight is [experts, n, k], splits int32 [experts] on the rows' device or the host; rows past
// their sum belong to no expert and are 0 in what is computed of them.  moe_linear, moe_swiglu and moe_mlp are differentiable once; checkpoint: what their
// backward pass reads of activations is kept in 8 bits.
torch::Tensor moe_linear(torch::Tensor input, torch::Tensor weight, torch::Tensor splits, bool checkpoint);
torch::Tensor moe_swiglu(torch::Tensor input, bool checkpoint);
torch::Tensor moe_mlp(torch::Tensor input, torch::Tensor weight1, torch::Tensor weight2, torch::Tensor splits, bool checkpoint);
// The gradients, for callers without autograd, and the 8 bits: e4m3 codes and a float8_e8m0fnu scale for every 32 values of a row.  They record nothing, but for
// moe_swiglu_checkpoint's first result, whose gradient is that of moe_swiglu with checkpoint.
torch::Tensor moe_dgrad(torch::Tensor grad, torch::Tensor weight, torch::Tensor splits);
torch::Tensor moe_wgrad(torch::Tensor grad, torch::Tensor input, torch::Tensor splits, std::optional<torch::Tensor> input_scale,
                        std::optional<torch::Tensor> output, bool accumulate, std::optional<at::ScalarType> output_dtype);
std::tuple<torch::Tensor, torch::Tensor> moe_checkpoint(torch::Tensor input);
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> moe_swiglu_checkpoint(torch::Tensor input);
std::tuple<torch::Tensor, torch::Tensor> moe_swiglu_backward(torch::Tensor grad, torch::Tensor input, std::optional<torch::Tensor> input_scale);
bool bitwise_check(torch::Tensor a, torch::Tensor b);

}  // namespace flux_amd
