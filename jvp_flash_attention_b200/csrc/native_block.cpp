// Host side of the operators beside attention, rotary and gated_linear, as native.cpp is attention's: argument checks, allocation,
// launches and the autograd graph, with tangents travelling along and one node for values and tangents.  Tensors that are not on a GPU
// are handed back to the Python modules' _launch functions (the CPU suite puts its formulas there); what this layer declines (bad
// arguments, transforms other than a lone torch.func.jvp) returns None and is served by the Python modules' Functions.
#include <algorithm>
#include <limits>
#include <mutex>

#include "native_common.h"

namespace {

py::object& rotary_module() {
  static py::object* m = new py::object(py::module_::import("jvp_flash_attention_b200.rotary"));  // lives as long as the process
  return *m;
}

py::object& gated_module() {
  static py::object* m = new py::object(py::module_::import("jvp_flash_attention_b200.gated"));
  return *m;
}
py::object or_none(const Tensor& t) { return t.defined() ? py::cast(t) : py::object(py::none()); }

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
// The tensor in memory: torch keeps some zeros as a shape alone.
Tensor in_memory(const Tensor& t) {
  if (!t.defined() || !t._is_zerotensor()) return t;
  NoFunctorch nf;
  return at::zeros(t.sizes(), t.options().requires_grad(false));
}
// The tangent in its value's type, and in memory.
Tensor as_tangent(const Tensor& t, const Tensor& x) {
  if (!t.defined()) return t;
  const Tensor y = in_memory(t);
  NoFunctorch nf;
  return y.scalar_type() == x.scalar_type() ? y : y.to(x.scalar_type());
}

// ---- rotary --------------------------------------------------------------------------------------------------------------
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
        ys[i] = launch(primal_of(xs[i]), freq, or_none(positions), turn.offset, turn.interleaved,
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
    Tensor x = xs[i] = in_memory(xs[i]);
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
            out[j] = turned(grads[j], f, or_none(p), back.offset, back.interleaved,
                            back.amplitude, back.transposed).cast<Tensor>();
        return out;
      }
      plain[i] = g;
    }
    variable_list out = turned_again(plain, f, p, back);
    // A cotangent that is dual, inside a forward-AD level: so is its gradient.
    std::vector<Tensor> tangents(grads.size());
    for (size_t i = 0; i < grads.size(); ++i)
      if (plain[i].defined()) tangents[i] = as_tangent(grads[i]._fw_grad(0), plain[i]);
    tangents = turned_again(tangents, f, p, back);
    for (size_t i = 0; i < out.size(); ++i)
      if (tangents[i].defined()) out[i]._set_fw_grad(tangents[i], /*level=*/0, /*is_inplace_op=*/false);
    return out;
  }
  // xs turned, with a node behind those that need one.
  std::vector<Tensor> turned_again(const std::vector<Tensor>& xs, const Tensor& f, const Tensor& p, const Turn& back) const {
    std::vector<Tensor> out = launch_rotary(xs, orders, f, p, back);
    std::vector<int> again;
    for (size_t i = 0; i < out.size(); ++i)
      if (out[i].defined() && torch::autograd::compute_requires_grad(xs[i])) again.push_back((int)i);
    connect(xs, out, again, f, p, back, orders);
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
  for (const Tensor* t : {&q, &k})
    for (int64_t d = 0; t->defined() && d < t->dim(); ++d)
      if (t->size(d) > INT32_MAX) return false;
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
  // (Inside a forward-AD level the primals stay dual: the kernels read their memory, the graph has their edges.)
  for (Tensor& x : xs) x = at_level_below(x, level);
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

// ---- gated projection ----------------------------------------------------------------------------------------------------
struct GatedOut {
  Tensor h, th, kept;  // kept: what a backward reads (jvpfa_gated_fwd_args)
};
struct GatedGrads {
  Tensor dx, dtx, dwg, dwu;
};

Tensor from_python(const py::handle& o) { return o.is_none() ? Tensor() : o.cast<Tensor>(); }

// (rows, K) with contiguous columns.
Tensor as_rows(const Tensor& x_) {
  const Tensor x = in_memory(x_);
  if (!x.defined() || (x.dim() == 2 && x.stride(1) == 1)) return x;
  NoFunctorch nf;
  at::AutoDispatchBelowADInplaceOrView below;
  const int64_t K = x.size(-1);
  Tensor r = x.dim() == 2 ? x : x.reshape({x.numel() / K, K});
  return r.stride(1) == 1 ? r : r.contiguous();
}
// Row-major, on a 16-byte boundary, of the type of `like`.
Tensor as_dense(const Tensor& x_, const Tensor& like) {
  const Tensor x = in_memory(x_);
  if (!x.defined()) return x;
  const bool aligned = (reinterpret_cast<uintptr_t>(x.const_data_ptr()) & 15u) == 0;
  if (x.is_contiguous() && aligned && x.scalar_type() == like.scalar_type()) return x;
  NoFunctorch nf;
  at::AutoDispatchBelowADInplaceOrView below;
  return at::empty_like(x, x.options().dtype(like.scalar_type()), at::MemoryFormat::Contiguous).copy_(x);
}
Tensor workspace_for(int64_t bytes, const Tensor& x) { return bytes > 0 ? empty({bytes}, at::kByte, x.device()) : Tensor(); }

// h, with tx also th, and with `keep` what a backward reads.
GatedOut launch_gated_fwd(const Tensor& x, const Tensor& tx, const Tensor& wg, const Tensor& wu, int activation, bool keep) {
  GatedOut r;
  if (!x.is_cuda()) {
    py::gil_scoped_acquire gil;
    NoFunctorch nf;
    at::AutoGradMode no_grad(false);
    py::tuple out = gated_module().attr("_launch_fwd")(primal_of(x), or_none(tx), wg, wu, activation, keep);
    r.h = from_python(out[0]), r.th = from_python(out[1]), r.kept = from_python(out[2]);
    return r;
  }
  c10::cuda::OptionalCUDAGuard guard;
  if (x.get_device() != c10::cuda::current_device()) guard.set_index(x.get_device());
  std::vector<int64_t> sizes = x.sizes().vec();
  sizes.back() = wg.size(0);
  const int64_t rows = x.numel() / wg.size(1);
  r.h = empty(sizes, x.scalar_type(), x.device());
  if (tx.defined()) r.th = empty(sizes, x.scalar_type(), x.device());
  if (keep)
    r.kept = empty({jvpfa_gated_kept_bytes(dtype_of(x, false), (int)rows, (int)wg.size(0), tx.defined())}, at::kByte, x.device());
  if (rows == 0) return r;
  const Tensor x2 = as_rows(x), tx2 = as_rows(tx), wg2 = as_rows(wg), wu2 = as_rows(wu);
  jvpfa_gated_fwd_args a{};
  a.struct_size = sizeof(a);
  a.dtype = dtype_of(x, false);
  a.M = (int)x2.size(0), a.K = (int)x2.size(1), a.F = (int)wg.size(0);
  a.activation = activation;
  a.x = data(x2), a.tx = data(tx2), a.wg = data(wg2), a.wu = data(wu2);
  a.x_stride = x2.stride(0), a.tx_stride = tx2.defined() ? tx2.stride(0) : 0, a.wg_stride = wg2.stride(0), a.wu_stride = wu2.stride(0);
  a.h = r.h.data_ptr(), a.th = r.th.defined() ? r.th.data_ptr() : nullptr;
  if (keep) a.kept = r.kept.data_ptr();
  const Tensor workspace = workspace_for(jvpfa_gated_fwd_workspace(&a), x);
  if (workspace.defined()) a.workspace = workspace.data_ptr(), a.workspace_bytes = workspace.numel();
  check_status(jvpfa_gated_fwd(&a, c10::cuda::getCurrentCUDAStream(x.get_device()).stream()), "jvpfa_gated_fwd");
  return r;
}

// Gradients of <gh, h> + <gth, th>; tx as in the forward that left `kept`.
GatedGrads launch_gated_bwd(const Tensor& x, const Tensor& tx, const Tensor& wg, const Tensor& wu, const Tensor& kept, Tensor gh, Tensor gth,
                            int activation, bool need_x, bool need_tx, bool need_w) {
  GatedGrads r;
  need_tx = need_tx && gth.defined();
  if (!need_x && !need_tx && !need_w) return r;
  if (!x.is_cuda()) {
    py::gil_scoped_acquire gil;
    NoFunctorch nf;
    at::AutoGradMode no_grad(false);
    py::tuple out = gated_module().attr("_launch_bwd")(x, or_none(tx), wg, wu, kept, or_none(gh), or_none(gth), activation, need_x,
                                                       need_tx, need_w);
    Tensor* to[] = {&r.dx, &r.dtx, &r.dwg, &r.dwu};
    for (int i = 0; i < 4; ++i) *to[i] = from_python(out[i]);
    return r;
  }
  c10::cuda::OptionalCUDAGuard guard;
  if (x.get_device() != c10::cuda::current_device()) guard.set_index(x.get_device());
  if (x.numel() == 0) {
    NoFunctorch nf;
    at::AutoDispatchBelowADInplaceOrView below;
    if (need_x) r.dx = at::zeros_like(x);
    if (need_tx) r.dtx = at::zeros_like(x);
    if (need_w) r.dwg = at::zeros_like(wg), r.dwu = at::zeros_like(wu);
    return r;
  }
  gh = as_dense(gh, x), gth = as_dense(gth, x);
  const bool dual = gth.defined();
  if (need_x) r.dx = empty(x.sizes(), x.scalar_type(), x.device());
  if (need_tx) r.dtx = empty(x.sizes(), x.scalar_type(), x.device());
  if (need_w) r.dwg = empty(wg.sizes(), x.scalar_type(), x.device()), r.dwu = empty(wu.sizes(), x.scalar_type(), x.device());
  const Tensor x2 = as_rows(x), tx2 = dual ? as_rows(tx) : Tensor(), wg2 = as_rows(wg), wu2 = as_rows(wu);
  jvpfa_gated_bwd_args a{};
  a.struct_size = sizeof(a);
  a.dtype = dtype_of(x, false);
  a.M = (int)x2.size(0), a.K = (int)x2.size(1), a.F = (int)wg.size(0);
  a.activation = activation;
  a.x = data(x2), a.tx = data(tx2), a.wg = data(wg2), a.wu = data(wu2);
  a.x_stride = x2.stride(0), a.tx_stride = dual ? tx2.stride(0) : 0, a.wg_stride = wg2.stride(0), a.wu_stride = wu2.stride(0);
  a.kept = data(kept), a.kept_tangent = tx.defined();
  a.gh = data(gh), a.gth = data(gth);
  if (need_x) a.dx = r.dx.data_ptr();
  if (need_tx) a.dtx = r.dtx.data_ptr();
  if (need_w) a.dwg = r.dwg.data_ptr(), a.dwu = r.dwu.data_ptr();
  const Tensor workspace = workspace_for(jvpfa_gated_bwd_workspace(&a), x);
  if (workspace.defined()) a.workspace = workspace.data_ptr(), a.workspace_bytes = workspace.numel();
  check_status(jvpfa_gated_bwd(&a, c10::cuda::getCurrentCUDAStream(x.get_device()).stream()), "jvpfa_gated_bwd");
  return r;
}

constexpr const char* kThird = "gated_linear cannot be differentiated a third time";
constexpr const char* kThroughTangent = "the gradient through the tangent output of gated_linear cannot be differentiated a second time";

// Inside a forward-AD level: a tensor's tangent, if it has one, and one put on a gradient.
Tensor tangent_of(const Tensor& t) { return t.defined() ? t._fw_grad(0) : Tensor(); }
void set_tangent(Tensor& t, const Tensor& tangent) {
  if (!t.defined() || !tangent.defined()) return;
  if (t.is_view()) t = t.clone(at::MemoryFormat::Contiguous);  // (a view's would have to be one of its base's)
  t._set_fw_grad(tangent, /*level=*/0, /*is_inplace_op=*/false);
}
// In place of a tangent that takes a third derivative, which there is no formula for: NaN, since none would be read as zero.  (The gradient
// itself is right, and who does not ask for its tangent loses nothing.)
Tensor unknown_like(const Tensor& t) {
  if (!t.defined()) return t;
  at::AutoDispatchBelowADInplaceOrView below;
  at::AutoGradMode no_grad(false);
  return at::full_like(t, std::numeric_limits<double>::quiet_NaN());
}

// (dx, dwg, dwu) of <gh, h> as a node that can be differentiated once more: with v the incoming gradients,
//   d<(dx, dwg, dwu), v>/d(x, wg, wu) = d<th(x, wg, wu; v), gh>/d(x, wg, wu)   and   d<(dx, dwg, dwu), v>/d(gh) = th(x, wg, wu; v),
// one value-and-tangent forward and one backward through the tangent (of operands side by side, which the Python module makes, where the
// weights' gradients are differentiated).
struct GatedGradNode : public Node {
  int activation;
  SavedVariable x, wg, wu, gh;

  // One behind e's gradients.
  static void connect(GatedGrads& e, int activation, const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& gh) {
    auto node = std::shared_ptr<GatedGradNode>(new GatedGradNode(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x, wg, wu, gh));
    node->activation = activation;
    node->x = SavedVariable(x, false);
    node->wg = SavedVariable(wg, false);
    node->wu = SavedVariable(wu, false);
    node->gh = SavedVariable(gh, false);
    for (Tensor* t : {&e.dx, &e.dwg, &e.dwu}) {
      if (t->defined())
        torch::autograd::set_history(*t, node);
      else
        node->add_input_metadata(Node::undefined_input());
    }
  }

  variable_list apply(variable_list&& v) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list out(4);
    if (!v[0].defined() && !v[1].defined() && !v[2].defined()) return out;
    for (const Tensor& t : v)
      if (t.defined() && is_wrapped(t)) throw std::runtime_error("gated_linear cannot be differentiated a second time under a functorch transform");
    const Tensor x_ = x.unpack(), wg_ = wg.unpack(), wu_ = wu.unpack(), gh_ = gh.unpack();
    variable_list plain, tangents;
    for (const Tensor& t : v) plain.push_back(primal_of(t)), tangents.push_back(as_tangent(tangent_of(t), t));
    out = along(plain, x_, wg_, wu_, gh_);
    // Inside a forward-AD level: linear in v, and a third derivative where the operands move.
    const bool moves = tangent_of(x_).defined() || tangent_of(gh_).defined();
    if (moves) {
      for (Tensor& t : out) set_tangent(t, unknown_like(t));
    } else if (tangents[0].defined() || tangents[1].defined() || tangents[2].defined()) {
      const variable_list t = along(tangents, x_, wg_, wu_, gh_);
      for (int i = 0; i < 4; ++i) set_tangent(out[i], t[i]);
    }
    return out;
  }
  variable_list along(const variable_list& v, const Tensor& x_, const Tensor& wg_, const Tensor& wu_, const Tensor& gh_) {
    variable_list out(4);
    const Tensor xp = unwrap(primal_of(x_)), wgp = unwrap(wg_), wup = unwrap(wu_), ghp = unwrap(primal_of(gh_));
    const bool need_x = task_should_compute_output(0), need_w = task_should_compute_output(1) || task_should_compute_output(2);
    if (v[1].defined() || v[2].defined()) {
      py::gil_scoped_acquire gil;
      NoFunctorch nf;
      at::AutoGradMode no_grad(false);
      py::tuple h = gated_module().attr("_second")(xp, wgp, wup, ghp, or_none(v[0]), or_none(v[1]), or_none(v[2]), activation);
      for (int i = 0; i < 4; ++i)
        if (task_should_compute_output(i)) out[i] = from_python(h[i]);
    } else {
      const GatedOut f = launch_gated_fwd(xp, v[0], wgp, wup, activation, need_x || need_w);
      if (need_x || need_w) {
        const GatedGrads g = launch_gated_bwd(xp, v[0], wgp, wup, f.kept, Tensor(), ghp, activation, need_x, false, need_w);
        out[0] = g.dx, out[1] = g.dwg, out[2] = g.dwu;
      }
      if (task_should_compute_output(3)) out[3] = f.th;
    }
    if (at::GradMode::is_enabled())
      attach_refusal(kThird, {&out[0], &out[1], &out[2], &out[3]}, x_, wg_, wu_, gh_, v[0], v[1], v[2]);
    return out;
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* s : {&x, &wg, &wu, &gh}) s->reset_data();
  }
  std::string name() const override { return "GatedLinearBackwardBackward"; }
};

// The node of a call: outputs h (0) and, with a tangent, th (1); edges to x, wg, wu and, with a tangent, tx.
struct GatedNode : public Node {
  int activation;
  bool side_by_side;  // operands of twice the width, [x | 0], [tx | x] and [w | tw] (the Python module's, for tangents of the weights)
  SavedVariable x, tx, wg, wu, kept;

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list out(num_outputs());
    const Tensor gh = primal_of(grads[0]), gth = grads.size() > 1 ? primal_of(grads[1]) : Tensor();
    if (!gh.defined() && !gth.defined()) return out;
    for (const Tensor& g : grads)
      TORCH_CHECK_NOT_IMPLEMENTED(!g.defined() || !g.key_set().has(c10::DispatchKey::Batched),
                                  "gated_linear has no rule for torch.autograd.grad(is_grads_batched=True)");
    const Tensor x_dual = x.unpack(), x_ = primal_of(x_dual), wg_ = primal_of(wg.unpack()), wu_ = primal_of(wu.unpack());
    const Tensor xp = unwrap(x_), wgp = unwrap(wg_), wup = unwrap(wu_);
    const Tensor tx_ = num_outputs() > 3 ? tx.unpack() : Tensor(), txp = unwrap(tx_), kept_ = unwrap(kept.unpack());
    const bool need_x = task_should_compute_output(0), need_w = task_should_compute_output(1) || task_should_compute_output(2);
    const bool need_tx = num_outputs() > 3 && task_should_compute_output(3);
    if ((gh.defined() && is_wrapped(gh)) || (gth.defined() && is_wrapped(gth))) {
      // the cotangents belong to a functorch transform, which differentiates Functions (and takes their tangents along)
      if (side_by_side && tangent_of(x_dual).defined())
        throw std::runtime_error("inside a forward-AD level where gated_linear's weights have tangents, its gradient cannot be transformed");
      py::gil_scoped_acquire gil;
      py::tuple d = gated_module().attr("_backward_under_functorch")(x_dual, or_none(tx_), wg_, wu_, kept_, or_none(grads[0]),
                                                                     or_none(grads.size() > 1 ? grads[1] : Tensor()), activation);
      const int at[] = {0, 3, 1, 2};  // of (dx, dtx, dwg, dwu) among the edges
      for (int i = 0; i < 4; ++i)
        if (at[i] < (int)out.size()) out[at[i]] = from_python(d[i]);
      return out;
    }
    // Under create_graph the part through h stays a node of its own, which can be differentiated again.
    const bool again = at::GradMode::is_enabled() && torch::autograd::compute_requires_grad(x_, wg_, wu_, tx_, gh, gth);
    GatedGrads d;
    if (gth.defined()) {
      d = launch_gated_bwd(xp, txp, wgp, wup, kept_, again ? Tensor() : gh, gth, activation, need_x, need_tx, need_w);
      if (again) attach_refusal(kThroughTangent, {&d.dx, &d.dtx, &d.dwg, &d.dwu}, x_, wg_, wu_, tx_, gth);
    }
    if (gh.defined() && (again || !gth.defined())) {
      GatedGrads e = launch_gated_bwd(xp, txp, wgp, wup, kept_, gh, Tensor(), activation, need_x, false, need_w);
      if (again) GatedGradNode::connect(e, activation, x_dual, wg_, wu_, grads[0]);
      auto add = [](Tensor& to, const Tensor& t) {
        if (t.defined()) to = to.defined() ? to + t : t;
      };
      add(d.dx, e.dx), add(d.dwg, e.dwg), add(d.dwu, e.dwu);
    }
    // Inside a forward-AD level gradients are dual.
    const Tensor tgh = tangent_of(grads[0]), tgth = grads.size() > 1 ? tangent_of(grads[1]) : Tensor();
    const bool along = tangent_of(x_dual).defined();  // x moves along tx
    if (along || tgh.defined() || tgth.defined()) {
      GatedGrads t;
      if (along && gth.defined()) {
        t = {unknown_like(d.dx), unknown_like(d.dtx), unknown_like(d.dwg), unknown_like(d.dwu)};
      } else if (along) {
        t = along_tx(xp, txp, wgp, wup, kept_, gh, as_tangent(tgh, gh), need_x, need_w);
        if (again) attach_refusal(kThird, {&t.dx, &t.dwg, &t.dwu}, x_, wg_, wu_, tx_, gh, tgh);
      } else {  // linear in the cotangents
        const Tensor ch = as_tangent(tgh, gh), cth = as_tangent(tgth, gth);
        t = launch_gated_bwd(xp, txp, wgp, wup, kept_, ch, cth, activation, need_x, need_tx, need_w);
        if (again && cth.defined())
          attach_refusal(kThroughTangent, {&t.dx, &t.dtx, &t.dwg, &t.dwu}, x_, wg_, wu_, tx_, ch, cth);
        else if (again)
          GatedGradNode::connect(t, activation, x_, wg_, wu_, ch);
      }
      set_tangent(d.dx, t.dx), set_tangent(d.dtx, t.dtx), set_tangent(d.dwg, t.dwg), set_tangent(d.dwu, t.dwu);
    }
    out[0] = d.dx;
    if (task_should_compute_output(1)) out[1] = d.dwg;
    if (task_should_compute_output(2)) out[2] = d.dwu;
    if (need_tx) out[3] = d.dtx;
    return out;
  }
  // The tangents of the gradients (dx, dwg, dwu) of <gh, h>, x moving along tx and gh along tgh: by the symmetry of second derivatives the
  // gradients of <tgh, h> + <gh, th>, from the projections that the forward kept.
  GatedGrads along_tx(const Tensor& xp, const Tensor& txp, const Tensor& wgp, const Tensor& wup, const Tensor& kept_, const Tensor& gh,
                      const Tensor& tgh, bool need_x, bool need_w) const {
    GatedGrads t = launch_gated_bwd(xp, txp, wgp, wup, kept_, tgh, gh, activation, need_x, need_x && side_by_side, need_w);
    if (!side_by_side) return t;
    // Operands side by side: what is wanted of x is both halves' sum (the weights move as well), and h does not depend on what stands for
    // the tangents.
    at::AutoDispatchBelowADInplaceOrView below;
    at::AutoGradMode no_grad(false);
    const int64_t K = xp.size(-1) / 2;
    auto with_zeros = [](const Tensor& y) { return at::cat({y, at::zeros_like(y)}, -1); };
    if (need_x) t.dx = with_zeros(t.dx.narrow(-1, 0, K) + t.dtx.narrow(-1, K, K)), t.dtx = Tensor();
    if (need_w) t.dwg = with_zeros(t.dwg.narrow(-1, 0, K)), t.dwu = with_zeros(t.dwu.narrow(-1, 0, K));
    return t;
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* s : {&x, &tx, &wg, &wu, &kept}) s->reset_data();
  }
  std::string name() const override { return "GatedLinearBackward"; }
};

bool gated_acceptable(const Tensor& x, const Tensor& wg, const Tensor& wu) {
  if (x.dim() < 1 || wg.dim() != 2 || wu.sizes() != wg.sizes() || x.size(-1) != wg.size(1)) return false;
  if (wg.size(0) < 1 || wg.size(1) < 1) return false;
  for (const Tensor* t : {&x, &wg, &wu})
    if (t->layout() != at::kStrided || t->scalar_type() != x.scalar_type() || t->device() != x.device()) return false;
  const int64_t K = wg.size(1), F = wg.size(0);
  if (x.numel() / K > INT32_MAX || K > INT32_MAX || F > INT32_MAX) return false;
  return !x.is_cuda() || dtype_of(x, false) >= 0;
}

// None: not a case for this path; the caller takes its general route.
py::object gated(const Tensor& x_in, const Tensor& wg_in, const Tensor& wu_in, int activation, bool side_by_side) {
  const int64_t level = jvp_level();
  if (level == -2 || wg_in._fw_grad(0).defined() || wu_in._fw_grad(0).defined()) return py::none();
  Tensor x = x_in, tx = x._fw_grad(0);
  if (level >= 0 && !tx.defined()) return py::none();
  // (inside torch.func.jvp the function may use the weights as they are, or wrapped at its level without a tangent)
  x = at_level_below(x, level), tx = at_level_below(tx, level);
  const Tensor wg = at_level_below(wg_in, level), wu = at_level_below(wu_in, level);
  for (const Tensor* t : std::initializer_list<const Tensor*>{&x, &tx, &wg, &wu})
    if (t->defined() && is_wrapped(*t)) return py::none();
  if (!gated_acceptable(x, wg, wu)) return py::none();
  if (tx.defined()) {
    if (tx.sizes() != x.sizes() || tx.device() != x.device()) return py::none();
    tx = as_tangent(tx, x);
  }
  const bool grad_h = torch::autograd::compute_requires_grad(x, wg, wu), grad = grad_h || torch::autograd::compute_requires_grad(tx);
  GatedOut r;
  {
    std::optional<py::gil_scoped_release> no_gil;
    if (x.is_cuda()) no_gil.emplace();
    r = launch_gated_fwd(x, tx, wg, wu, activation, grad);
  }
  if (grad) {
    auto node = std::shared_ptr<GatedNode>(new GatedNode(), torch::autograd::deleteNode);
    node->set_next_edges(tx.defined() ? torch::autograd::collect_next_edges(x, wg, wu, tx) : torch::autograd::collect_next_edges(x, wg, wu));
    node->activation = activation;
    node->side_by_side = side_by_side;
    node->x = SavedVariable(x, false);
    node->wg = SavedVariable(wg, false);
    node->wu = SavedVariable(wu, false);
    node->kept = SavedVariable(r.kept, false);
    if (grad_h)
      torch::autograd::set_history(r.h, node);
    else
      node->add_input_metadata(Node::undefined_input());
    if (tx.defined()) {
      node->tx = SavedVariable(tx, false);
      torch::autograd::set_history(r.th, node);
    }
  }
  return dual(r.h, r.th, level);
}

}  // namespace

void bind_block(py::module_& m) {
  m.def("rotary", &rotary, py::arg("q"), py::arg("k").none(true), py::arg("inv_freq"), py::arg("positions").none(true), py::arg("offset"),
        py::arg("interleaved"), py::arg("amplitude"));
  m.def("gated", &gated, py::arg("x"), py::arg("w_gate"), py::arg("w_up"), py::arg("activation"), py::arg("side_by_side") = false);
}
