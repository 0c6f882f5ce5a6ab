// Backward nodes of the operators whose calls are short: the node of a forward is made
// here and hung on its output, and its backward runs in torch's engine without Python.
// The host's time bounds these calls: forward and gradient of 333x1001 elements of
// dropout (3.7 us of kernels) took 75 us with a Python function and take 59 us, of an
// embedding of 64 tokens 81-90 us and 61 us.  The arithmetic is the C ABI's; the
// forward, with its checks, is the Python module's.
//
// A gradient that is to be differentiated again (create_graph) comes out right and
// refuses that, the linear operators' where the upstream gradient is differentiable.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/pybind.h>

#include <memory>
#include <mutex>
#include <optional>
#include <string>

#include "metallora_b200.h"

namespace {

using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

// A refusal becomes the package's own exception, as it does from Python.
void check(int status, const char* what) {
  if (status == MLORA_OK) return;
  pybind11::gil_scoped_acquire gil;
  try {
    pybind11::module_::import("metallora_b200._lib").attr("check")(status, what);
  } catch (pybind11::error_already_set& e) {
    e.restore();
    python_error raised;
    raised.persist();
    throw raised;
  }
}

// The entry points, of the library that Python has loaded: the forward's and these are
// of one build.
struct {
  decltype(&mlora_dropout) dropout;
  decltype(&mlora_embedding_backward) embedding_backward;
  decltype(&mlora_embedding_backward_workspace_bytes) embedding_backward_workspace_bytes;
  decltype(&mlora_linear_cross_entropy_backward) linear_cross_entropy_backward;
} abi;

void bind(uintptr_t dropout, uintptr_t embedding_backward, uintptr_t embedding_backward_workspace_bytes,
          uintptr_t linear_cross_entropy_backward) {
  abi.dropout = reinterpret_cast<decltype(abi.dropout)>(dropout);
  abi.embedding_backward = reinterpret_cast<decltype(abi.embedding_backward)>(embedding_backward);
  abi.embedding_backward_workspace_bytes =
      reinterpret_cast<decltype(abi.embedding_backward_workspace_bytes)>(
          embedding_backward_workspace_bytes);
  abi.linear_cross_entropy_backward =
      reinterpret_cast<decltype(abi.linear_cross_entropy_backward)>(linear_cross_entropy_backward);
}

void* current_stream() { return c10::cuda::getCurrentCUDAStream().stream(); }

// depends: whether the gradient is a function of something to be differentiated.
variable_list once(at::Tensor grad, bool depends) {
  if (!c10::GradMode::is_enabled() || !depends) return {std::move(grad)};
  grad = grad.detach();
  grad.set_requires_grad(true);
  auto refuse = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice an operator that can be differentiated once", 1);
  return (*refuse)({std::move(grad)});
}

// The node becomes out's, and x's gradient its only result.
template <typename N>
void attach(const at::Tensor& out, const at::Tensor& x, std::unique_ptr<N> made) {
  std::shared_ptr<Node> node(made.release(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(x));
  torch::autograd::set_history(out, node);
}

struct MloraDropoutBackward : Node {
  int64_t n;
  int threshold, scaled, dtype;
  uint64_t seed, call;
  std::optional<SavedVariable> seed_tensor;  // in the place of seed

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined()) return {at::Tensor()};
    const at::Tensor held = seed_tensor ? seed_tensor->unpack() : at::Tensor();
    const at::Tensor dy = grads[0].contiguous();
    at::Tensor dx = at::empty_like(dy);
    if (n > 0)
      check(abi.dropout(dy.const_data_ptr(), dx.data_ptr(), n, threshold, scaled, seed,
                          held.defined() ? held.const_data_ptr<int64_t>() : nullptr, call, dtype,
                          current_stream()),
            "mlora_dropout");
    return once(std::move(dx), dy.requires_grad());
  }
  void release_variables() override {
    if (seed_tensor) seed_tensor->reset_data();
  }
  std::string name() const override { return "MloraDropoutBackward"; }
};

struct MloraEmbeddingBackward : Node {
  int64_t T, V, D, padding, workspace;
  float scale;
  int dtype;
  SavedVariable idx;

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined()) return {at::Tensor()};
    const at::Tensor dy = grads[0].contiguous(), index = idx.unpack();
    at::Tensor grad = at::empty({V, D}, dy.options());
    if (T == 0 || D == 0) {
      grad.zero_();
    } else {
      at::Tensor ws = at::empty({workspace}, dy.options().dtype(at::kByte));
      check(abi.embedding_backward(index.const_data_ptr<int64_t>(), dy.const_data_ptr(),
                                     grad.data_ptr(), T, V, D, scale, padding, dtype, ws.data_ptr(),
                                     static_cast<size_t>(workspace), current_stream()),
            "mlora_embedding_backward");
    }
    return once(std::move(grad), dy.requires_grad());
  }
  void release_variables() override { idx.reset_data(); }
  std::string name() const override { return "MloraEmbeddingBackward"; }
};

// Of x alone: a frozen head.
struct MloraLinearCrossEntropyBackward : Node {
  int64_t M;
  bool per_row, mean;
  int dtype;
  SavedVariable state, weight;

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined()) return {at::Tensor()};
    const at::Tensor up = grads[0].contiguous(), s = state.unpack();
    const at::Tensor w = weight.unpack().contiguous();
    const int64_t V = w.size(0), K = w.size(1);
    at::Tensor dx = at::empty({M, K}, w.options());
    if (M > 0)
      check(abi.linear_cross_entropy_backward(s.const_data_ptr(), static_cast<size_t>(s.numel()),
                                                up.const_data_ptr<float>(), per_row, mean,
                                                w.const_data_ptr(), dx.data_ptr(), nullptr, nullptr,
                                                dtype, 0, nullptr, M, K, V, 0, dtype,
                                                MLORA_HEAD_GRAD_X, current_stream()),
            "mlora_linear_cross_entropy_backward");
    return once(std::move(dx), true);
  }
  void release_variables() override {
    state.reset_data();
    weight.reset_data();
  }
  std::string name() const override { return "MloraLinearCrossEntropyBackward"; }
};

void attach_dropout(const at::Tensor& out, const at::Tensor& x, int64_t n, int threshold, bool scaled,
                    uint64_t seed, uint64_t call, int dtype, const std::optional<at::Tensor>& seed_tensor) {
  auto node = std::make_unique<MloraDropoutBackward>();
  node->n = n;
  node->threshold = threshold;
  node->scaled = scaled;
  node->seed = seed;
  node->call = call;
  node->dtype = dtype;
  if (seed_tensor) node->seed_tensor.emplace(*seed_tensor, false);
  attach(out, x, std::move(node));
}

void attach_embedding(const at::Tensor& out, const at::Tensor& table, const at::Tensor& idx, int64_t T,
                      int64_t V, int64_t D, float scale, int64_t padding, int dtype) {
  auto node = std::make_unique<MloraEmbeddingBackward>();
  node->T = T;
  node->V = V;
  node->D = D;
  node->scale = scale;
  node->padding = padding;
  node->dtype = dtype;
  node->workspace =
      T > 0 && D > 0 ? static_cast<int64_t>(abi.embedding_backward_workspace_bytes(T, D)) : 0;
  node->idx = SavedVariable(idx, false);
  attach(out, table, std::move(node));
}

void attach_linear_cross_entropy(const at::Tensor& loss, const at::Tensor& x, const at::Tensor& state,
                                 const at::Tensor& weight, int64_t M, bool per_row, bool mean,
                                 int dtype) {
  auto node = std::make_unique<MloraLinearCrossEntropyBackward>();
  node->M = M;
  node->per_row = per_row;
  node->mean = mean;
  node->dtype = dtype;
  node->state = SavedVariable(state, false);
  node->weight = SavedVariable(weight, false);
  attach(loss, x, std::move(node));
}

}  // namespace

PYBIND11_MODULE(_autograd, m) {
  m.def("bind", &bind);
  m.def("attach_dropout", &attach_dropout);
  m.def("attach_embedding", &attach_embedding);
  m.def("attach_linear_cross_entropy", &attach_linear_cross_entropy);
}
