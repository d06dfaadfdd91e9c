// What the native layer's sources share: tensors under functorch's wrappers, allocation without the dispatcher, status codes as
// exceptions, and the node behind gradients that cannot be differentiated again.
#pragma once

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/functorch/DynamicLayer.h>
#include <ATen/functorch/TensorWrapper.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <cuda_runtime_api.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <array>
#include <atomic>
#include <memory>
#include <optional>
#include <string>
#include <vector>

#include "jvpfa.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

namespace {

inline bool is_wrapped(const Tensor& x) {
  return x.key_set().has(c10::DispatchKey::FuncTorchGradWrapper) || x.key_set().has(c10::DispatchKey::FuncTorchBatched);
}

// The tensor under functorch's wrappers.
inline Tensor unwrap(Tensor x) {
  while (x.defined()) {
    auto* w = at::functorch::maybeGetTensorWrapper(x);
    if (!w) break;
    x = Tensor(w->value());
  }
  return x;
}

inline const void* data(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }

inline int dtype_of(const Tensor& t, bool tf32) {
  switch (t.scalar_type()) {
    case at::kBFloat16:
      return JVPFA_BF16;
    case at::kHalf:
      return JVPFA_FP16;
    case at::kFloat:
      return tf32 ? JVPFA_FP32_TF32 : JVPFA_FP32;
    default:
      return -1;
  }
}

inline void check_status(int rc, const char* what) {
  if (rc == JVPFA_OK) return;
  std::string msg = std::string(what) + " failed: [" + std::to_string(rc) + "] " + jvpfa_strerror(rc);
  const std::string cuda = jvpfa_last_cuda_error();
  if (!cuda.empty()) msg += " | " + cuda;
  throw std::runtime_error(msg);
}

// Allocation without the dispatcher: these run inside functorch levels as well, and a call makes up to nine of them.
inline Tensor empty(at::IntArrayRef sizes, at::ScalarType dtype, at::Device device) {
  return Tensor(at::detail::empty_cuda(sizes, dtype, device, std::nullopt));
}

// Operators on plain tensors while a functorch level may be active: without its dispatch keys.
struct NoFunctorch {
  c10::impl::ExcludeDispatchKeyGuard guard;
  NoFunctorch()
      : guard(c10::DispatchKeySet({c10::DispatchKey::FuncTorchDynamicLayerFrontMode, c10::DispatchKey::FuncTorchDynamicLayerBackMode})) {}
};

struct NoFunctorchScope {  // the same as a Python context manager
  std::optional<NoFunctorch> guard;
};

// Stands behind gradients that cannot be differentiated again, and says so when asked.
struct Refuse : public Node {
  std::string message;
  explicit Refuse(std::string m) : message(std::move(m)) {}
  variable_list apply(variable_list&&) override { throw std::runtime_error(message); }
  std::string name() const override { return "JVPAttnRefuse"; }
};

template <typename... Ts>
void attach_refusal(const char* message, std::initializer_list<Tensor*> outs, const Ts&... inputs) {
  if (!torch::autograd::compute_requires_grad(inputs...)) return;
  auto node = std::shared_ptr<Refuse>(new Refuse(message), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(inputs...));
  for (Tensor* t : outs)
    if (t->defined()) torch::autograd::set_history(*t, node);
}

// The order of a tensor's dimensions in memory, the widest first (the last one stays innermost).
using Order = std::array<int, 4>;
inline Order order_of(const Tensor& x) {
  Order o{0, 1, 2, 3};
  std::stable_sort(o.begin(), o.begin() + 3, [&](int a, int b) { return x.stride(a) > x.stride(b); });
  return o;
}
inline Tensor empty_in_order(at::IntArrayRef sizes, const Order& o, at::ScalarType dtype, at::Device device) {
  std::array<int64_t, 4> st;
  int64_t n = 1;
  for (int d = 3; d >= 0; --d) st[o[d]] = n, n *= std::max<int64_t>(sizes[o[d]], 1);
  return Tensor(at::detail::empty_strided_cuda(sizes, st, dtype, device));
}

inline Tensor primal_of(const Tensor& x) {  // inside a forward-AD level the saved tensors are still dual
  return x.defined() && x._fw_grad(0).defined() ? x._fw_primal(0) : x;
}

}  // namespace

// The operators beside attention (native_block.cpp)
void bind_block(py::module_& m);
// The norms and residual sums (native_norm.cpp)
void bind_norm(py::module_& m);
// Linear attention (native_linear.cpp)
void bind_linear(py::module_& m);
