// Host side of linear_attention and linear_attention_step: argument checks, allocation, launches; the graph is native_dual.h's.  What this
// layer declines returns None and is served by the Python module.
#include <cmath>

#include "native_dual.h"

namespace {

constexpr int kQ = 0, kK = 1, kV = 2, kState = 3, kOperands = 4;

bool any_of(const std::vector<bool>& v) { return std::find(v.begin(), v.end(), true) != v.end(); }

struct LinearOp : ModuleOp {
  double scale;
  bool want_state;
  py::tuple options() const override { return py::make_tuple(scale, want_state, name); }

  struct Call {
    jvpfa_linear_args a{};
    Tensors alive;
  };
  static Tensor rows(const Tensor& x_, at::ScalarType type) {  // with contiguous entries
    const Tensor x = memory_of(x_);
    if ((x.stride(3) == 1 || x.size(3) == 1) && x.scalar_type() == type) return x;
    NoFunctorch nf;
    at::AutoDispatchBelowADInplaceOrView below;
    return x.to(type).contiguous();
  }
  static Tensor whole(const Tensor& x_) {  // a state, row-major
    const Tensor x = memory_of(x_);
    if (x.is_contiguous()) return x;
    NoFunctorch nf;
    at::AutoDispatchBelowADInplaceOrView below;
    return x.contiguous();
  }
  static void put(jvpfa_linear_tensor& to, const Tensor& x) {
    to.p = x.const_data_ptr();
    for (int d = 0; d < 3; ++d) to.stride[d] = x.stride(d);
  }
  void describe(Call& c, const Tensors& x, const Tensors& tx, const Tensors& extras, bool dual) const {
    jvpfa_linear_args& a = c.a;
    c.alive.reserve(16);
    a.struct_size = sizeof(a);
    a.dtype = dtype_of(x[kQ], false);
    a.B = (int)x[kQ].size(0), a.H = (int)x[kQ].size(1), a.L = (int)x[kQ].size(2), a.D = (int)x[kQ].size(3), a.E = (int)x[kV].size(3);
    a.scale = (float)scale, a.dual = dual;
    if (extras[0].defined()) a.log_decay = static_cast<const float*>(extras[0].const_data_ptr());
    if (extras[1].defined()) a.lengths = static_cast<const int32_t*>(extras[1].const_data_ptr());
    jvpfa_linear_tensor* to[6] = {&a.q, &a.k, &a.v, &a.tq, &a.tk, &a.tv};
    for (int i = 0; i < 6; ++i) operand(c, *to[i], i < 3 ? x[i] : dual ? tx[i - 3] : Tensor(), x[kQ]);
    a.state = state(c, x[kState]), a.tstate = dual ? state(c, tx[kState]) : nullptr;
  }
  static void operand(Call& c, jvpfa_linear_tensor& to, const Tensor& t, const Tensor& like) {
    if (t.defined()) put(to, c.alive.emplace_back(rows(t, like.scalar_type())));
  }
  static const float* state(Call& c, const Tensor& t) {
    return t.defined() ? static_cast<const float*>(c.alive.emplace_back(whole(t)).const_data_ptr()) : nullptr;
  }
  static float* out(const Tensor& t) { return t.defined() ? static_cast<float*>(t.data_ptr()) : nullptr; }
  static Tensor workspace(Call& c, int64_t bytes, const Tensor& like) {
    Tensor w;
    if (bytes > 0) w = empty({bytes}, at::kByte, like.device()), c.a.workspace = w.data_ptr(), c.a.workspace_bytes = bytes;
    return w;
  }

  DualOut forward(const Tensors& x, const Tensors& tx, const Tensors& extras, bool want_kept) const override {
    if (!x[kQ].is_cuda()) return python_forward(x, tx, extras, want_kept);
    const Tensor& q = x[kQ];
    c10::cuda::OptionalCUDAGuard guard;
    if (q.get_device() != c10::cuda::current_device()) guard.set_index(q.get_device());
    const bool dual = any_defined(tx);
    DualOut r;
    r.y.resize(2), r.ty.resize(2);
    const std::vector<int64_t> states{q.size(0), q.size(1), q.size(3), x[kV].size(3)};
    for (int side = 0; side < (dual ? 2 : 1); ++side) {
      Tensors& y = side ? r.ty : r.y;
      y[0] = empty_in_order(x[kV].sizes(), order_of(x[kV]), q.scalar_type(), q.device());
      if (want_state) y[1] = empty(states, at::kFloat, q.device());
    }
    if (q.size(0) * q.size(1) * q.size(2) == 0) {  // no rows: the state stays
      NoFunctorch nf;
      at::AutoDispatchBelowADInplaceOrView below;
      for (int side = 0; side < (dual ? 2 : 1); ++side) {
        Tensor& y = (side ? r.ty : r.y)[1];
        const Tensor& from = (side ? tx : x)[kState];
        if (y.defined()) from.defined() ? y.copy_(memory_of(from)) : y.zero_();
      }
      return r;
    }
    Call c;
    describe(c, x, tx, extras, dual);
    put(c.a.o, r.y[0]);
    c.a.state_out = out(r.y[1]);
    if (dual) put(c.a.to, r.ty[0]), c.a.tstate_out = out(r.ty[1]);
    if (want_kept) {
      const int64_t bytes = jvpfa_linear_kept_bytes(&c.a);
      r.kept = empty({bytes}, at::kByte, q.device());
      if (bytes > 0) c.a.kept = r.kept.data_ptr();
    }
    const Tensor w = workspace(c, jvpfa_linear_fwd_workspace(&c.a), q);
    check_status(jvpfa_linear_fwd(&c.a, c10::cuda::getCurrentCUDAStream(q.get_device()).stream()), "jvpfa_linear_fwd");
    return r;
  }
  Tensors backward(const Tensors& x, const Tensors& tx, const Tensors& extras, const Tensor& kept, const Tensors& g, const Tensors& gt,
                   const std::vector<bool>& want) const override {
    Tensors d(2 * kOperands);
    if (!any_of(want)) return d;
    if (!x[kQ].is_cuda()) return python_backward(x, tx, extras, kept, g, gt, want);
    const Tensor& q = x[kQ];
    c10::cuda::OptionalCUDAGuard guard;
    if (q.get_device() != c10::cuda::current_device()) guard.set_index(q.get_device());
    const bool dual = any_defined(gt), nothing = q.size(0) * q.size(1) * q.size(2) == 0;
    for (int i = 0; i < 2 * kOperands; ++i) {
      const Tensor& of = x[i % kOperands];
      if (!want[i] || !of.defined()) continue;
      if (nothing || (i >= kOperands && !dual)) {
        NoFunctorch nf;
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor c = i == kState ? g[1] : i == kOperands + kState ? gt[1] : Tensor();
        d[i] = nothing && c.defined() ? memory_of(c).clone() : at::zeros(of.sizes(), of.options().requires_grad(false));
      } else {
        d[i] = i % kOperands == kState ? empty(of.sizes(), at::kFloat, of.device()) : empty_in_order(of.sizes(), order_of(of), of.scalar_type(), of.device());
      }
    }
    if (nothing) return d;
    Call c;
    describe(c, x, tx, extras, dual);
    operand(c, c.a.go, g[0], q);
    c.a.gstate = state(c, g[1]);
    if (dual) operand(c, c.a.gto, gt[0], q), c.a.gtstate = state(c, gt[1]);
    jvpfa_linear_tensor* to[6] = {&c.a.dq, &c.a.dk, &c.a.dv, &c.a.dtq, &c.a.dtk, &c.a.dtv};
    for (int i = 0; i < 6; ++i) {
      const Tensor& t = d[i < 3 ? i : kOperands + i - 3];
      if (t.defined() && (i < 3 || dual)) put(*to[i], t);
    }
    if (kept.defined() && kept.numel() > 0) c.a.kept = const_cast<void*>(kept.const_data_ptr()), c.a.kept_dual = any_defined(tx);
    c.a.dstate = out(d[kState]);
    if (dual) c.a.dtstate = out(d[kOperands + kState]);
    const Tensor w = workspace(c, jvpfa_linear_bwd_workspace(&c.a), q);
    check_status(jvpfa_linear_bwd(&c.a, c10::cuda::getCurrentCUDAStream(q.get_device()).stream()), "jvpfa_linear_bwd");
    return d;
  }
};

bool decays_acceptable(const Tensor& w, const Tensor& like, int64_t heads) {
  return !w.defined() || (w.dim() == 1 && w.size(0) == heads && w.scalar_type() == at::kFloat && w.is_contiguous() && w.device() == like.device() &&
                          !(w.requires_grad() && at::GradMode::is_enabled()) && !w._fw_grad(0).defined() && !is_wrapped(w));
}

bool linear_acceptable(const Tensors& x, const Tensors& extras) {
  const Tensor &q = x[kQ], &k = x[kK], &v = x[kV], &state = x[kState];
  for (const Tensor* t : {&q, &k, &v})
    if (!t->defined() || t->dim() != 4 || t->scalar_type() != q.scalar_type() || t->device() != q.device()) return false;
  if (k.sizes() != q.sizes()) return false;
  for (int d = 0; d < 3; ++d)
    if (v.size(d) != q.size(d)) return false;
  const int64_t B = q.size(0), H = q.size(1), D = q.size(3), E = v.size(3);
  if (D < 1 || E < 1 || D > 128 || E > 128 || q.size(2) > (1 << 30) || B * H > (1 << 24)) return false;
  if (q.is_cuda() && dtype_of(q, false) < 0) return false;
  if (state.defined() && (state.dim() != 4 || state.size(0) != B || state.size(1) != H || state.size(2) != D || state.size(3) != E ||
                          (q.is_cuda() && state.scalar_type() != at::kFloat) || state.device() != q.device()))
    return false;
  if (!decays_acceptable(extras[0], q, H)) return false;
  const Tensor& n = extras[1];
  return !n.defined() || (n.dim() == 1 && n.size(0) == B && n.scalar_type() == at::kInt && n.is_contiguous() && n.device() == q.device());
}

std::shared_ptr<LinearOp> operator_of(const py::tuple& options) {
  auto op = std::make_shared<LinearOp>();
  op->name = "linear_attention", op->outputs = 2, op->module = "jvp_flash_attention_b200.linear_attention";
  op->scale = options[0].cast<double>(), op->want_state = options[1].cast<bool>();
  return op;
}

// (o, state), None where there is none; None for all: not a case for this path.
py::object linear(const std::vector<std::optional<Tensor>>& operands, const std::optional<Tensor>& log_decay, const std::optional<Tensor>& lengths,
                  const py::tuple& options) {
  const Tensor w = log_decay ? *log_decay : Tensor();
  if (w.defined() && w._fw_grad(0).defined()) return py::none();
  const DualOperands in(operands, {w, lengths ? *lengths : Tensor()});
  if (!in.ok || in.x.size() != kOperands || !linear_acceptable(in.x, in.extras)) return py::none();
  const std::vector<py::object> r = apply_dual(operator_of(options), in);
  return py::make_tuple(r[0], r[1]);
}

py::tuple launch_fwd(const py::list& x, const py::list& tx, const py::list& extras, const py::tuple& options, bool keep) {
  const DualOut r = operator_of(options)->forward(tensors_of(x), tensors_of(tx), tensors_of(extras), keep);
  return py::make_tuple(list_of(r.y), list_of(r.ty), none_or(r.kept));
}
py::list launch_bwd(const py::list& x, const py::list& tx, const py::list& extras, const py::object& kept, const py::list& g, const py::list& gt,
                    const py::tuple& options, const std::vector<bool>& want) {
  return list_of(operator_of(options)->backward(tensors_of(x), tensors_of(tx), tensors_of(extras), tensor_of(kept), tensors_of(g), tensors_of(gt), want));
}

// o of one more token, `state` updated; None: bad arguments, which the Python module names.
py::object step(const Tensor& q_, const Tensor& k_, const Tensor& v_, const std::optional<Tensor>& log_decay, const Tensor& state, double scale) {
  if (!at::functorch::getDynamicLayerStack().empty()) return py::none();
  const Tensor w = log_decay ? *log_decay : Tensor();
  for (const Tensor* t : {&q_, &k_, &v_, &state})
    if (!t->is_cuda() || t->layout() != at::kStrided || t->device() != q_.device() || t->_fw_grad(0).defined() ||
        (at::GradMode::is_enabled() && t->requires_grad()))
      return py::none();
  if (q_.dim() != 3 || k_.sizes() != q_.sizes() || v_.dim() != 3 || v_.size(0) != q_.size(0) || v_.size(1) != q_.size(1) || state.dim() != 4) return py::none();
  const int64_t B = q_.size(0), H = q_.size(1), D = q_.size(2), E = v_.size(2);
  if (dtype_of(q_, false) < 0 || k_.scalar_type() != q_.scalar_type() || v_.scalar_type() != q_.scalar_type() || D < 1 || E < 1 || D > 128 || E > 128 ||
      B * H > (1 << 24))
    return py::none();
  if (state.scalar_type() != at::kFloat || state.size(0) != B || state.size(1) != H || state.size(2) != D || state.size(3) != E || !decays_acceptable(w, q_, H))
    return py::none();
  if ((D > 1 && state.stride(2) != E) || (E > 1 && state.stride(3) != 1)) return py::none();
  c10::cuda::OptionalCUDAGuard guard;
  if (q_.get_device() != c10::cuda::current_device()) guard.set_index(q_.get_device());
  auto entries = [](const Tensor& t) { return t.stride(2) == 1 || t.size(2) == 1 ? t : t.contiguous(); };
  at::AutoDispatchBelowADInplaceOrView below;
  const Tensor q = entries(memory_of(q_)), k = entries(memory_of(k_)), v = entries(memory_of(v_));
  const Tensor o = empty({B, H, E}, q.scalar_type(), q.device());
  if (B * H == 0) return py::cast(o);
  jvpfa_linear_step_args a{};
  a.struct_size = sizeof(a);
  a.dtype = dtype_of(q, false);
  a.B = (int)B, a.H = (int)H, a.D = (int)D, a.E = (int)E, a.scale = (float)scale;
  if (w.defined()) a.log_decay = static_cast<const float*>(w.const_data_ptr());
  a.q = q.const_data_ptr(), a.k = k.const_data_ptr(), a.v = v.const_data_ptr(), a.o = o.data_ptr();
  for (int d = 0; d < 2; ++d)
    a.q_stride[d] = q.stride(d), a.k_stride[d] = k.stride(d), a.v_stride[d] = v.stride(d), a.state_stride[d] = state.stride(d);
  a.state = static_cast<float*>(state.data_ptr());
  state.unsafeGetTensorImpl()->bump_version();  // (refuses what must not be written)
  const int rc = jvpfa_linear_step(&a, c10::cuda::getCurrentCUDAStream(q.get_device()).stream());
  if (rc == JVPFA_ERR_SHAPE) return py::none();  // states that share memory
  check_status(rc, "jvpfa_linear_step");
  return py::cast(o);
}

}  // namespace

void bind_linear(py::module_& m) {
  m.def("linear", &linear, py::arg("operands"), py::arg("log_decay").none(true), py::arg("lengths").none(true), py::arg("options"));
  m.def("linear_launch_fwd", &launch_fwd);
  m.def("linear_launch_bwd", &launch_bwd);
  m.def("linear_step", &step, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("log_decay").none(true), py::arg("state"), py::arg("scale"));
}
