// What every operator with a gradient of its own refuses, because its kernels would answer wrongly or the process would end.
#pragma once
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>
#include <torch/extension.h>

namespace flux_amd {

// The kernels carry no tangents: forward mode would silently lose them.
inline void refuse_tangent(const torch::Tensor &t, const char *what) {
  TORCH_CHECK(!t._fw_grad(/*level=*/0).defined(), what, ": forward-mode derivatives are not built");
}

// A conjugate or negative view stands for other values than its memory holds, which is what is moved.
inline void refuse_lazy_view(const torch::Tensor &t, const char *name) {
  TORCH_CHECK(!t.is_conj() && !t.is_neg(), name, " is a conjugate or negative view: resolve_conj() or resolve_neg() first");
}

// The gradients come from kernels that record nothing: a second derivative, in reverse or forward mode, would be silently wrong, so it is refused.
inline void refuse_second_derivative(const char *who, const torch::Tensor &grad) {
  refuse_tangent(grad, who);
  TORCH_CHECK(!at::GradMode::is_enabled(), who, ": the gradient of the gradient is not built (create_graph=True)");
}

// A backward pass that is captured hands its gradients to leaves on the stream where these were first used.  If an eager graph of a leaf is alive, that is the
// eager stream, which would be drawn into the capture and end the process: an error is raised before it comes to that.
inline void refuse_leaves_of_another_stream(const char *who) {
  const c10::hip::HIPStream current = c10::hip::getCurrentHIPStream();
  hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(current.stream(), &capture) != hipSuccess) {
    (void)hipGetLastError();
    return;
  }
  const std::shared_ptr<torch::autograd::Node> node = torch::autograd::get_current_node();
  if (capture == hipStreamCaptureStatusNone || node == nullptr) return;
  for (const torch::autograd::Edge &edge : node->next_edges()) {
    if (edge.function == nullptr || edge.function->name() != "torch::autograd::AccumulateGrad") continue;
    const std::optional<c10::Stream> stream = edge.function->stream();
    TORCH_CHECK(!stream.has_value() || stream->id() == current.id(), who,
                ": its backward pass is captured while an eager graph of the same leaf is alive; drop that graph's outputs before the capture");
  }
}

}  // namespace flux_amd
