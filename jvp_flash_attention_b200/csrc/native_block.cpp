// Host side of the operators beside attention, rotary and gated_linear, as native.cpp is attention's: argument checks, allocation,
// launches and the autograd graph, with tangents travelling along and one node for values and tangents.  Tensors that are not on a GPU
// are handed back to the Python modules' _launch functions (the CPU suite puts its formulas there); what this layer declines (bad
// arguments, transforms other than a lone torch.func.jvp) returns None and is served by the Python modules' Functions.
#include <algorithm>
#include <mutex>

#include "native_common.h"

namespace {

py::object& rotary_module() {
  static py::object* m = new py::object(py::module_::import("jvp_flash_attention_b200.rotary"));  // lives as long as the process
  return *m;
}

// The level of the lone torch.func.jvp that is active, -1 without any transform, -2 under others.
int64_t jvp_level() {
  const auto& stack = at::functorch::getDynamicLayerStack();
  if (stack.empty()) return -1;
  return stack.size() == 1 && stack.back().key() == at::functorch::TransformType::Jvp ? stack.back().layerId() : -2;
}
Tensor at_level_below(const Tensor& x, int64_t level) {
  auto* w = x.defined() && level >= 0 ? at::functorch::maybeGetTensorWrapper(x) : nullptr;
  return w && w->level() == level ? Tensor(w->value()) : x;
}
// `value` with its tangent, at the level that its inputs came from.
py::object dual(Tensor value, Tensor tangent, int64_t level) {
  if (!tangent.defined()) return py::cast(value);
  if (level >= 0) {
    value = at::functorch::makeTensorWrapper(value, level);
    tangent = at::functorch::makeTensorWrapper(tangent, level);
  }
  value._set_fw_grad(tangent, /*level=*/0, /*is_inplace_op=*/false);
  return py::cast(value);
}
// The tangent in its value's type.
Tensor as_tangent(const Tensor& t, const Tensor& x) {
  if (!t.defined() || t.scalar_type() == x.scalar_type()) return t;
  NoFunctorch nf;
  return t.to(x.scalar_type());
}

// ---- rotary --------------------------------------------------------------------------------------------------------------
// The order of a tensor's dimensions in memory, the widest first (the last one stays innermost).
using Order = std::array<int, 4>;
Order order_of(const Tensor& x) {
  Order o{0, 1, 2, 3};
  std::stable_sort(o.begin(), o.begin() + 3, [&](int a, int b) { return x.stride(a) > x.stride(b); });
  return o;
}
Tensor empty_in_order(at::IntArrayRef sizes, const Order& o, at::ScalarType dtype, at::Device device) {
  std::array<int64_t, 4> st;
  int64_t n = 1;
  for (int d = 3; d >= 0; --d) st[o[d]] = n, n *= std::max<int64_t>(sizes[o[d]], 1);
  return Tensor(at::detail::empty_strided_cuda(sizes, st, dtype, device));
}

struct Turn {
  int64_t offset;
  bool interleaved, transposed;
  double amplitude;
};

// xs turned, each into a tensor of its own in the given order.  Undefined ones stay so.
std::vector<Tensor> launch_rotary(std::vector<Tensor> xs, const std::vector<Order>& orders, const Tensor& freq, const Tensor& positions,
                                  const Turn& turn) {
  std::vector<Tensor> ys(xs.size());
  const auto some = std::find_if(xs.begin(), xs.end(), [](const Tensor& x) { return x.defined(); });
  if (some == xs.end()) return ys;
  if (!some->is_cuda()) {
    py::gil_scoped_acquire gil;
    NoFunctorch nf;
    at::AutoGradMode no_grad(false);
    auto launch = rotary_module().attr("_launch");
    for (size_t i = 0; i < xs.size(); ++i)
      if (xs[i].defined())
        ys[i] = launch(xs[i], freq, positions.defined() ? py::cast(positions) : py::object(py::none()), turn.offset, turn.interleaved,
                       turn.amplitude, turn.transposed).cast<Tensor>();
    return ys;
  }
  c10::cuda::OptionalCUDAGuard guard;
  if (some->get_device() != c10::cuda::current_device()) guard.set_index(some->get_device());
  jvpfa_rotary_args a{};
  a.struct_size = sizeof(a);
  a.dtype = dtype_of(*some, false);
  a.B = (int)some->size(0), a.L = (int)some->size(2), a.D = (int)some->size(3), a.n_freq = (int)freq.size(0);
  a.interleaved = turn.interleaved, a.transposed = turn.transposed;
  a.amplitude = (float)turn.amplitude;
  a.freq = static_cast<const double*>(freq.const_data_ptr());
  a.offset = turn.offset;
  if (positions.defined()) {
    a.positions = positions.const_data_ptr();
    a.position_bits = positions.scalar_type() == at::kLong ? 64 : 32;
    const bool rows = positions.dim() == 2 && positions.size(0) > 1;
    a.position_stride[0] = rows ? positions.stride(0) : 0;
    a.position_stride[1] = positions.stride(-1);
  }
  for (size_t i = 0; i < xs.size(); ++i) {
    if (!xs[i].defined()) continue;
    Tensor x = xs[i];
    if (x.stride(3) != 1 && x.size(3) != 1) {
      NoFunctorch nf;
      at::AutoDispatchBelowADInplaceOrView below;
      xs[i] = x = x.contiguous();
    }
    ys[i] = empty_in_order(x.sizes(), orders[i], x.scalar_type(), x.device());
    if (x.numel() == 0) continue;
    jvpfa_rotary_tensor& t = a.t[a.n_tensors++];
    t.x = x.const_data_ptr(), t.y = ys[i].data_ptr();
    t.H = (int)x.size(1);
    for (int d = 0; d < 3; ++d) t.x_stride[d] = x.stride(d), t.y_stride[d] = ys[i].stride(d);
  }
  if (a.n_tensors) check_status(jvpfa_rotary(&a, c10::cuda::getCurrentCUDAStream(some->get_device()).stream()), "jvpfa_rotary");
  return ys;
}

// The gradient of a linear map is its transpose, at every order of differentiation: the node of values and tangents alike.
struct RotaryNode : public Node {
  Turn turn;  // of the forward
  std::vector<Order> orders;
  SavedVariable freq, positions;

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    std::vector<Tensor> plain(grads.size());
    const Tensor f = freq.unpack(), p = positions.unpack();
    Turn back = turn;
    back.transposed = !turn.transposed;
    for (size_t i = 0; i < grads.size(); ++i) {
      if (!grads[i].defined() || !task_should_compute_output(i)) continue;
      const Tensor g = primal_of(grads[i]);
      if (is_wrapped(g)) {  // the cotangent belongs to a functorch transform, which differentiates a Function
        py::gil_scoped_acquire gil;
        variable_list out(grads.size());
        auto turned = rotary_module().attr("_turn");
        for (size_t j = 0; j < grads.size(); ++j)
          if (grads[j].defined() && task_should_compute_output(j))
            out[j] = turned(grads[j], f, p.defined() ? py::cast(p) : py::object(py::none()), back.offset, back.interleaved,
                            back.amplitude, back.transposed).cast<Tensor>();
        return out;
      }
      plain[i] = g;
    }
    variable_list out = launch_rotary(plain, orders, f, p, back);
    std::vector<int> again;
    for (size_t i = 0; i < out.size(); ++i)
      if (out[i].defined() && torch::autograd::compute_requires_grad(plain[i])) again.push_back((int)i);
    connect(plain, out, again, f, p, back, orders);
    return out;
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    freq.reset_data();
    positions.reset_data();
  }
  std::string name() const override { return "RotaryBackward"; }

  // One node behind the outputs `which`.
  static void connect(const std::vector<Tensor>& xs, std::vector<Tensor>& ys, const std::vector<int>& which, const Tensor& freq,
                      const Tensor& positions, const Turn& turn, const std::vector<Order>& orders) {
    if (which.empty()) return;
    auto node = std::shared_ptr<RotaryNode>(new RotaryNode(), torch::autograd::deleteNode);
    node->turn = turn;
    torch::autograd::edge_list edges;
    for (int i : which) edges.push_back(torch::autograd::impl::gradient_edge(xs[i])), node->orders.push_back(orders[i]);
    node->set_next_edges(std::move(edges));
    node->freq = SavedVariable(freq, false);
    node->positions = SavedVariable(positions, false);
    for (int i : which) torch::autograd::set_history(ys[i], node);
  }
};

bool rotary_acceptable(const Tensor& q, const Tensor& k, const Tensor& freq, const Tensor& positions) {
  if (q.dim() != 4 || q.layout() != at::kStrided || (q.is_cuda() && dtype_of(q, false) < 0)) return false;
  if (k.defined() && (k.dim() != 4 || k.layout() != at::kStrided || k.scalar_type() != q.scalar_type() || k.device() != q.device() ||
                      k.size(0) != q.size(0) || k.size(2) != q.size(2) || k.size(3) != q.size(3)))
    return false;
  if (freq.dim() != 1 || freq.scalar_type() != at::kDouble || freq.device() != q.device() || !freq.is_contiguous() ||
      2 * freq.size(0) > q.size(3) || freq.requires_grad())
    return false;
  if (!positions.defined()) return true;
  if (positions.device() != q.device() || (positions.scalar_type() != at::kLong && positions.scalar_type() != at::kInt)) return false;
  if (positions.dim() == 1) return positions.size(0) == q.size(2);
  return positions.dim() == 2 && (positions.size(0) == 1 || positions.size(0) == q.size(0)) && positions.size(1) == q.size(2);
}

// None: not a case for this path; the caller takes its general route.
py::object rotary(const Tensor& q_in, const std::optional<Tensor>& k_in, const Tensor& freq_in, const std::optional<Tensor>& positions_in,
                  int64_t offset, bool interleaved, double amplitude) {
  const int64_t level = jvp_level();
  if (level == -2) return py::none();
  const Tensor q_ = q_in, k_ = k_in ? *k_in : Tensor();
  std::vector<Tensor> xs{q_, k_, q_._fw_grad(0), k_.defined() ? k_._fw_grad(0) : Tensor()};
  if (level >= 0 && !xs[2].defined() && !xs[3].defined()) return py::none();
  // Primals and tangents are taken off the transform's wrappers, the call runs one level down, and the results become dual again.
  for (Tensor& x : xs) x = at_level_below(x, level);
  if (level < 0)
    for (int i = 0; i < 2; ++i)
      if (xs[2 + i].defined()) xs[i] = xs[i]._fw_primal(0);
  const Tensor freq = unwrap(freq_in), positions = positions_in ? unwrap(*positions_in) : Tensor();
  for (const Tensor& x : xs)
    if (x.defined() && is_wrapped(x)) return py::none();
  if (!rotary_acceptable(xs[0], xs[1], freq, positions)) return py::none();
  for (int i = 0; i < 2; ++i) {
    if (!xs[2 + i].defined()) continue;
    if (xs[2 + i].sizes() != xs[i].sizes() || xs[2 + i].device() != xs[i].device()) return py::none();
    xs[2 + i] = as_tangent(xs[2 + i], xs[i]);
  }
  const Turn turn{offset, interleaved, false, amplitude};
  std::vector<Order> orders(4);
  std::vector<int> history;
  for (int i = 0; i < 4; ++i) {
    if (!xs[i].defined()) continue;
    orders[i] = order_of(xs[i & 1]);  // tangents in their primals' layout
    if (torch::autograd::compute_requires_grad(xs[i])) history.push_back(i);
  }
  std::vector<Tensor> ys;
  {
    std::optional<py::gil_scoped_release> no_gil;
    if (xs[0].is_cuda()) no_gil.emplace();
    ys = launch_rotary(xs, orders, freq, positions, turn);
  }
  RotaryNode::connect(xs, ys, history, freq, positions, turn, orders);
  py::object q = dual(ys[0], ys[2], level);
  if (!k_.defined()) return q;
  return py::make_tuple(q, dual(ys[1], ys[3], level));
}

}  // namespace

void bind_block(py::module_& m) {
  m.def("rotary", &rotary, py::arg("q"), py::arg("k").none(true), py::arg("inv_freq"), py::arg("positions").none(true), py::arg("offset"),
        py::arg("interleaved"), py::arg("amplitude"));
}
