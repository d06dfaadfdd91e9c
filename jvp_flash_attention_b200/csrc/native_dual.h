// Operators of several inputs and outputs as graph nodes, with tangents travelling along: one node for values and tangents, one for
// gradients that are differentiated once more.  An operator brings its two launches; everything else follows from what holds for all of them:
//   d<grads(g), v>/dx = d<ty(x; v), g>/dx,   d<grads(g), v>/dg = ty(x; v),   and the gradients' tangents along (tx, tg) are the gradients of
//   <tg, y> + <g, ty>.
// Third derivatives are refused, and where a tangent would be one it is NaN, since none would be read as zero.
#pragma once
#include <limits>
#include <mutex>

#include "native_common.h"

namespace {

using Tensors = std::vector<Tensor>;

struct DualOut {
  Tensors y, ty;
  Tensor kept;  // what a backward reads
};

struct DualOp {
  const char* name;
  int outputs;
  Tensors extras;  // tensors without gradients, as the launches take them
  virtual ~DualOp() = default;
  // y, with any tangent ty too, and with `keep` what a backward reads.
  virtual DualOut forward(const Tensors& x, const Tensors& tx, const Tensors& extras, bool keep) const = 0;
  // Gradients of <g, y> + <gt, ty> with respect to x (first half) and tx (second half), as far as wanted; tx as in the forward.
  virtual Tensors backward(const Tensors& x, const Tensors& tx, const Tensors& extras, const Tensor& kept, const Tensors& g, const Tensors& gt,
                           const std::vector<bool>& want) const = 0;
  // The same for cotangents that belong to a functorch transform, by the Python module's Functions.
  virtual Tensors backward_under_functorch(const Tensors& x, const Tensors& tx, const Tensors& extras, const Tensor& kept, const Tensors& g,
                                           const Tensors& gt) const = 0;
  std::string message(const char* what) const { return std::string(what) + name; }
};

inline bool any_defined(const Tensors& ts) {
  for (const Tensor& t : ts)
    if (t.defined()) return true;
  return false;
}
inline bool any_requires_grad(const Tensors& ts) {
  for (const Tensor& t : ts)
    if (t.defined() && torch::autograd::compute_requires_grad(t)) return true;
  return false;
}
inline Tensor dual_tangent_of(const Tensor& t) { return t.defined() ? t._fw_grad(0) : Tensor(); }
inline Tensors map_tensors(const Tensors& ts, Tensor (*f)(const Tensor&)) {
  Tensors r;
  for (const Tensor& t : ts) r.push_back(t.defined() ? f(t) : Tensor());
  return r;
}
inline Tensor plain_of(const Tensor& t) { return unwrap(primal_of(t)); }
inline Tensor memory_of(const Tensor& t) {  // torch keeps some zeros as a shape alone
  if (!t._is_zerotensor()) return t;
  NoFunctorch nf;
  return at::zeros(t.sizes(), t.options().requires_grad(false));
}
// The tangent in its value's type, and in memory.
inline Tensor tangent_like(const Tensor& t, const Tensor& x) {
  if (!t.defined()) return t;
  const Tensor y = memory_of(t);
  NoFunctorch nf;
  return y.scalar_type() == x.scalar_type() ? y : y.to(x.scalar_type());
}
inline void put_tangent(Tensor& t, const Tensor& tangent) {
  if (!t.defined() || !tangent.defined()) return;
  if (t.is_view()) t = t.clone(at::MemoryFormat::Contiguous);  // (a view's would have to be one of its base's)
  t._set_fw_grad(tangent, /*level=*/0, /*is_inplace_op=*/false);
}
inline Tensor nan_like(const Tensor& t) {
  if (!t.defined()) return t;
  at::AutoDispatchBelowADInplaceOrView below;
  at::AutoGradMode no_grad(false);
  return at::full_like(t, std::numeric_limits<double>::quiet_NaN());
}
inline void refuse_through(const std::string& message, Tensors& outs, const Tensors& inputs) {
  if (!any_requires_grad(inputs)) return;
  auto node = std::shared_ptr<Refuse>(new Refuse(message), torch::autograd::deleteNode);
  torch::autograd::edge_list edges;
  for (const Tensor& t : inputs)
    if (t.defined()) edges.push_back(torch::autograd::impl::gradient_edge(t));
  node->set_next_edges(std::move(edges));
  for (Tensor& t : outs)
    if (t.defined()) torch::autograd::set_history(t, node);
}
inline torch::autograd::Edge edge_of(const Tensor& t) { return t.defined() ? torch::autograd::impl::gradient_edge(t) : torch::autograd::Edge(); }
inline std::vector<SavedVariable> saved(const Tensors& ts) {
  std::vector<SavedVariable> r;
  for (const Tensor& t : ts) r.emplace_back(t, false);
  return r;
}
inline Tensors unpacked(const std::vector<SavedVariable>& ss, std::shared_ptr<Node> = nullptr) {
  Tensors r;
  for (const SavedVariable& s : ss) r.push_back(s.unpack());
  return r;
}
inline Tensors joined(Tensors a, const Tensors& b) {
  a.insert(a.end(), b.begin(), b.end());
  return a;
}

// The gradients (of <g, y>) as a node that can be differentiated once more; edges to x and g.
struct DualGradNode : public Node {
  std::shared_ptr<const DualOp> op;
  std::vector<SavedVariable> x, g, extras;

  static void connect(Tensors& d, const std::shared_ptr<const DualOp>& op, const Tensors& x, const Tensors& g, const Tensors& extras) {
    if (!any_requires_grad(x) && !any_requires_grad(g)) return;
    auto node = std::shared_ptr<DualGradNode>(new DualGradNode(), torch::autograd::deleteNode);
    torch::autograd::edge_list edges;
    for (const Tensor& t : x) edges.push_back(edge_of(t));
    for (const Tensor& t : g) edges.push_back(edge_of(t));
    node->set_next_edges(std::move(edges));
    node->op = op, node->x = saved(x), node->g = saved(g), node->extras = saved(extras);
    for (Tensor& t : d) {
      if (t.defined())
        torch::autograd::set_history(t, node);
      else
        node->add_input_metadata(Node::undefined_input());
    }
  }
  variable_list apply(variable_list&& v) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list out(num_outputs());
    if (!any_defined(v)) return out;
    for (const Tensor& t : v)
      if (t.defined() && is_wrapped(t))
        throw std::runtime_error(op->message("under a functorch transform there is no second derivative of the graph of a call of "));
    const Tensors x_ = unpacked(x), g_ = unpacked(g), e_ = unpacked(extras);
    Tensors plain, tangents;
    for (const Tensor& t : v) plain.push_back(t.defined() ? primal_of(t) : t), tangents.push_back(t.defined() ? tangent_like(t._fw_grad(0), t) : t);
    out = along(plain, x_, g_, e_);
    // Inside a forward-AD level: linear in v, and a third derivative where the operands move.
    bool moves = false;
    for (const Tensors* ts : {&x_, &g_})
      for (const Tensor& t : *ts) moves = moves || dual_tangent_of(t).defined();
    if (moves) {
      for (Tensor& t : out) put_tangent(t, nan_like(t));
    } else if (any_defined(tangents)) {
      const variable_list t = along(tangents, x_, g_, e_);
      for (size_t i = 0; i < out.size(); ++i) put_tangent(out[i], t[i]);
    }
    return out;
  }
  variable_list along(const Tensors& v, const Tensors& x_, const Tensors& g_, const Tensors& e_) {
    const size_t n = x.size(), m = g.size();
    const Tensors xp = map_tensors(x_, plain_of), gp = map_tensors(g_, plain_of), ep = map_tensors(e_, unwrap_of);
    std::vector<bool> want(2 * n, false);
    bool any = false;
    for (size_t i = 0; i < n; ++i) want[i] = xp[i].defined() && task_should_compute_output(i), any = any || want[i];
    const DualOut f = op->forward(xp, v, ep, any);
    Tensors out(n + m);
    if (any) {
      const Tensors d = op->backward(xp, v, ep, f.kept, Tensors(m), gp, want);
      for (size_t i = 0; i < n; ++i) out[i] = d[i];
    }
    for (size_t j = 0; j < m; ++j)
      if (gp[j].defined() && task_should_compute_output(n + j)) out[n + j] = f.ty[j];
    if (at::GradMode::is_enabled()) refuse_through(op->message("there is no third derivative of "), out, joined(joined(x_, g_), v));
    return out;
  }
  static Tensor unwrap_of(const Tensor& t) { return unwrap(t); }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (auto* ss : {&x, &g, &extras})
      for (SavedVariable& s : *ss) s.reset_data();
  }
  std::string name() const override { return "DualBackwardBackward"; }
};

// The node of a call: outputs y and, with tangents, ty; edges to x and, with tangents, tx.
struct DualNode : public Node {
  std::shared_ptr<const DualOp> op;
  bool dual;
  std::vector<SavedVariable> x, tx, extras;
  SavedVariable kept;

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    const size_t n = x.size(), m = op->outputs;
    variable_list out(num_outputs());
    if (!any_defined(grads)) return out;
    Tensors g(m), gt(m), dual_g(grads.begin(), grads.begin() + m);
    bool wrapped = false;
    for (size_t j = 0; j < grads.size(); ++j) {
      if (!grads[j].defined()) continue;
      TORCH_CHECK_NOT_IMPLEMENTED(!grads[j].key_set().has(c10::DispatchKey::Batched), op->name,
                                  " has no rule for torch.autograd.grad(is_grads_batched=True)");
      (j < m ? g[j] : gt[j - m]) = primal_of(grads[j]);
      wrapped = wrapped || is_wrapped(primal_of(grads[j]));
    }
    const Tensors x_dual = unpacked(x), tx_ = unpacked(tx), e_ = unpacked(extras);
    const Tensors x_ = map_tensors(x_dual, primal_of), xp = map_tensors(x_dual, plain_of), txp = map_tensors(tx_, plain_of);
    const Tensors ep = map_tensors(e_, DualGradNode::unwrap_of);
    const Tensor kept_ = unwrap(kept.unpack());
    if (wrapped) {
      const Tensors d = op->backward_under_functorch(x_dual, tx_, e_, kept_, Tensors(grads.begin(), grads.begin() + m), dual ? Tensors(grads.begin() + m, grads.end()) : Tensors(m));
      for (size_t i = 0; i < out.size(); ++i)
        if (task_should_compute_output(i)) out[i] = d[i];
      return out;
    }
    std::vector<bool> want(2 * n, false);
    for (size_t i = 0; i < out.size(); ++i) want[i] = (i < n ? xp[i] : txp[i - n]).defined() && task_should_compute_output(i);
    // Under create_graph the part through y stays a node of its own, which can be differentiated again.
    const bool again = at::GradMode::is_enabled() && any_requires_grad(joined(joined(x_, tx_), Tensors(grads.begin(), grads.end())));
    const bool through = any_defined(gt);
    Tensors d(2 * n);
    if (through) {
      d = op->backward(xp, txp, ep, kept_, again ? Tensors(m) : g, gt, want);
      if (again) refuse_through(op->message("there is no second derivative through the tangent outputs of "), d, joined(joined(x_, tx_), gt));
    }
    if (any_defined(g) && (again || !through)) {
      std::vector<bool> want_x(want);
      for (size_t i = n; i < 2 * n; ++i) want_x[i] = false;
      Tensors e = op->backward(xp, txp, ep, kept_, g, Tensors(m), want_x);
      e.resize(n);
      if (again) DualGradNode::connect(e, op, x_dual, dual_g, e_);
      for (size_t i = 0; i < n; ++i)
        if (e[i].defined()) d[i] = d[i].defined() ? d[i] + e[i] : e[i];
    }
    // Inside a forward-AD level gradients are dual.
    Tensors tg(m), tgt(m);
    bool along = false;
    for (size_t j = 0; j < grads.size(); ++j)
      if (grads[j].defined()) (j < m ? tg[j] : tgt[j - m]) = tangent_like(grads[j]._fw_grad(0), grads[j]);
    for (const Tensor& t : x_dual) along = along || dual_tangent_of(t).defined();
    if (along || any_defined(tg) || any_defined(tgt)) {
      Tensors t(2 * n);
      if (along && through) {
        for (size_t i = 0; i < 2 * n; ++i) t[i] = nan_like(d[i]);
      } else if (along) {
        std::vector<bool> want_x(want);
        for (size_t i = n; i < 2 * n; ++i) want_x[i] = false;
        t = op->backward(xp, txp, ep, kept_, tg, g, want_x);
        if (again) refuse_through(op->message("there is no third derivative of "), t, joined(joined(x_, tx_), joined(g, tg)));
      } else {  // linear in the cotangents
        t = op->backward(xp, txp, ep, kept_, tg, tgt, want);
        if (again && any_defined(tgt)) {
          refuse_through(op->message("there is no second derivative through the tangent outputs of "), t, joined(joined(x_, tx_), joined(tg, tgt)));
        } else if (again) {
          Tensors first(t.begin(), t.begin() + n);
          DualGradNode::connect(first, op, x_, tg, e_);
          std::copy(first.begin(), first.end(), t.begin());
        }
      }
      for (size_t i = 0; i < 2 * n; ++i) put_tangent(d[i], t[i]);
    }
    for (size_t i = 0; i < out.size(); ++i)
      if (want[i]) out[i] = d[i];
    return out;
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (auto* ss : {&x, &tx, &extras})
      for (SavedVariable& s : *ss) s.reset_data();
    kept.reset_data();
  }
  std::string name() const override { return std::string("Backward of ") + op->name; }
};

// The level of the lone torch.func.jvp that is active, -1 without any transform, -2 under others.
inline int64_t lone_jvp_level() {
  const auto& stack = at::functorch::getDynamicLayerStack();
  if (stack.empty()) return -1;
  return stack.size() == 1 && stack.back().key() == at::functorch::TransformType::Jvp ? stack.back().layerId() : -2;
}
inline Tensor below_level(const Tensor& x, int64_t level) {
  auto* w = x.defined() && level >= 0 ? at::functorch::maybeGetTensorWrapper(x) : nullptr;
  return w && w->level() == level ? Tensor(w->value()) : x;
}

// Operands as the caller gave them, taken off a lone torch.func.jvp's wrappers.
struct DualOperands {
  int64_t level;
  Tensors x, tx, extras;
  bool ok = false;  // else: not a case for this path
  DualOperands(const std::vector<std::optional<Tensor>>& in, const Tensors& extras_in) : level(lone_jvp_level()) {
    if (level == -2) return;
    for (const auto& t : in) {
      const Tensor v = t ? *t : Tensor(), tangent = dual_tangent_of(v);
      x.push_back(below_level(v, level));
      tx.push_back(below_level(tangent, level));
    }
    for (const Tensor& t : extras_in) extras.push_back(unwrap(t));
    if (level >= 0 && !any_defined(tx)) return;
    for (size_t i = 0; i < x.size(); ++i) {
      if (!x[i].defined()) continue;
      if (is_wrapped(x[i]) || x[i].layout() != at::kStrided) return;
      if (!tx[i].defined()) continue;
      if (is_wrapped(tx[i]) || tx[i].sizes() != x[i].sizes() || tx[i].device() != x[i].device()) return;
      tx[i] = tangent_like(tx[i], x[i]);
    }
    ok = true;
  }
};

// The operator applied: values (with their tangents), and the graph.
inline std::vector<py::object> apply_dual(const std::shared_ptr<DualOp>& op, const DualOperands& in) {
  const bool dual = any_defined(in.tx), grad_y = any_requires_grad(in.x), grad = grad_y || any_requires_grad(in.tx);
  DualOut r;
  {
    std::optional<py::gil_scoped_release> no_gil;
    if (in.x[0].is_cuda()) no_gil.emplace();
    r = op->forward(in.x, in.tx, in.extras, grad);
  }
  if (grad) {
    auto node = std::shared_ptr<DualNode>(new DualNode(), torch::autograd::deleteNode);
    torch::autograd::edge_list edges;
    for (const Tensor& t : in.x) edges.push_back(edge_of(t));
    if (dual)
      for (const Tensor& t : in.tx) edges.push_back(edge_of(t));
    node->set_next_edges(std::move(edges));
    node->op = op, node->dual = dual;
    node->x = saved(in.x), node->tx = saved(in.tx), node->extras = saved(in.extras);
    node->kept = SavedVariable(r.kept, false);
    for (Tensor& t : r.y) {
      if (grad_y && t.defined())
        torch::autograd::set_history(t, node);
      else
        node->add_input_metadata(Node::undefined_input());
    }
    if (dual)
      for (Tensor& t : r.ty) {
        if (t.defined())
          torch::autograd::set_history(t, node);
        else
          node->add_input_metadata(Node::undefined_input());
      }
  }
  std::vector<py::object> out;
  for (size_t j = 0; j < r.y.size(); ++j) {
    Tensor value = r.y[j], tangent = dual ? r.ty[j] : Tensor();
    if (!value.defined()) {
      out.push_back(py::none());
      continue;
    }
    if (tangent.defined()) {
      if (in.level >= 0) {
        value = at::functorch::makeTensorWrapper(value, in.level);
        tangent = at::functorch::makeTensorWrapper(tangent, in.level);
      }
      value._set_fw_grad(tangent, /*level=*/0, /*is_inplace_op=*/false);
    }
    out.push_back(py::cast(value));
  }
  return out;
}

inline py::object none_or(const Tensor& t) { return t.defined() ? py::cast(t) : py::object(py::none()); }
inline py::list list_of(const Tensors& ts) {
  py::list r;
  for (const Tensor& t : ts) r.append(none_or(t));
  return r;
}
inline Tensor tensor_of(const py::handle& o) { return o.is_none() ? Tensor() : o.cast<Tensor>(); }
inline Tensors tensors_of(const py::handle& o) {
  Tensors r;
  for (const py::handle& t : o) r.push_back(tensor_of(t));
  return r;
}

// An operator whose launches on other than CUDA tensors are those of a Python module (the CPU suite puts its formulas there):
//   _launch_fwd(x, tx, extras, options, keep) -> (y, ty or None, kept)
//   _launch_bwd(x, tx, extras, kept, g, gt, options, want) -> d
// and whose Functions are that module's _backward_under_functorch(x, tx, extras, kept, g, gt, options) -> d.
struct ModuleOp : DualOp {
  const char* module;
  // The Python module's form of what the operator was called with (made when it is needed: a graph holds nothing of Python's).
  virtual py::tuple options() const = 0;
  py::object function(const char* name) const { return py::module_::import(module).attr(name); }
  DualOut python_forward(const Tensors& x, const Tensors& tx, const Tensors& extras, bool keep) const {
    py::gil_scoped_acquire gil;
    NoFunctorch nf;
    at::AutoGradMode no_grad(false);
    py::tuple r = function("_launch_fwd")(list_of(map_tensors(x, primal_of)), list_of(tx), list_of(extras), options(), keep);
    return {tensors_of(r[0]), r[1].is_none() ? Tensors(outputs) : tensors_of(r[1]), tensor_of(r[2])};
  }
  Tensors python_backward(const Tensors& x, const Tensors& tx, const Tensors& extras, const Tensor& kept, const Tensors& g, const Tensors& gt,
                          const std::vector<bool>& want) const {
    py::gil_scoped_acquire gil;
    NoFunctorch nf;
    at::AutoGradMode no_grad(false);
    return tensors_of(function("_launch_bwd")(list_of(x), list_of(tx), list_of(extras), none_or(kept), list_of(g), list_of(gt), options(), want));
  }
  Tensors backward_under_functorch(const Tensors& x, const Tensors& tx, const Tensors& extras, const Tensor& kept, const Tensors& g,
                                   const Tensors& gt) const override {
    py::gil_scoped_acquire gil;
    return tensors_of(function("_backward_under_functorch")(list_of(x), list_of(tx), list_of(extras), none_or(kept), list_of(g), list_of(gt), options()));
  }
};

}  // namespace
