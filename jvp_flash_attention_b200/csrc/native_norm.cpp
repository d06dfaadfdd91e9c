// Host side of norm, residual and residual_norm: argument checks, allocation, launches; the graph is native_dual.h's.  What this layer
// declines returns None and is served by the Python module.
#include <algorithm>

#include "native_dual.h"

namespace {

constexpr int kX = 0, kY = 1, kVectors = 2;  // places of the operands; the vectors in the order of jvpfa_norm_vector
constexpr int kOperands = 8;

struct NormOp : ModuleOp {
  int kind, post;
  double alpha, eps;
  py::tuple options() const override { return py::make_tuple(kind, post, alpha, eps, name); }

  // Rows of a group, 0 where the vectors cannot be laid out so: their dimensions are x's from the first up to some, and 1 from there on.
  static int64_t group_rows(const Tensors& x, bool grouped[6]) {
    const Tensor& t = x[kX];
    const int64_t C = t.size(-1), M = C ? t.numel() / C : 0;
    int64_t groups = 1;
    for (int i = 0; i < 6; ++i) {
      const Tensor& v = x[kVectors + i];
      grouped[i] = false;
      if (!v.defined()) continue;
      if (v.dim() < 1 || v.dim() > t.dim() || v.size(-1) != C) return 0;
      if (v.numel() == C && v.dim() < t.dim()) continue;
      if (v.dim() != t.dim()) return 0;
      bool one = false;
      int64_t n = 1;
      for (int64_t d = 0; d + 1 < t.dim(); ++d) {
        if (v.size(d) == t.size(d) && !one) {
          n *= v.size(d);
        } else if (v.size(d) == 1) {
          one = one || t.size(d) != 1;
        } else {
          return 0;
        }
      }
      if (n == 1) continue;
      if (groups != 1 && n != groups) return 0;
      groups = n, grouped[i] = true;
    }
    return M ? M / groups : 1;
  }
  static Tensor rows(const Tensor& x_) {  // (M, C) with contiguous columns
    const Tensor x = memory_of(x_);
    if (x.dim() == 2 && x.stride(1) == 1) return x;
    NoFunctorch nf;
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor r = x.reshape({-1, x.size(-1)});
    return r.stride(1) == 1 || r.size(1) == 1 ? r : r.contiguous();
  }
  static Tensor vector(const Tensor& v_, bool grouped) {  // (groups, C) or (C) with contiguous entries
    const Tensor v = memory_of(v_);
    NoFunctorch nf;
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor r = v.reshape(grouped ? std::vector<int64_t>{-1, v.size(-1)} : std::vector<int64_t>{v.size(-1)});
    return r.stride(-1) == 1 || r.size(-1) == 1 ? r : r.contiguous();
  }
  static Tensor dense(const Tensor& g_, const Tensor& like) {
    const Tensor g = memory_of(g_);
    if (g.is_contiguous() && g.scalar_type() == like.scalar_type()) return g;
    NoFunctorch nf;
    at::AutoDispatchBelowADInplaceOrView below;
    return at::empty_like(g, g.options().dtype(like.scalar_type()), at::MemoryFormat::Contiguous).copy_(g);
  }
  static at::ScalarType vector_type(const Tensors& x) {
    for (int i = 0; i < 6; ++i)
      if (x[kVectors + i].defined()) return x[kVectors + i].scalar_type();
    return x[kX].scalar_type();
  }
  void describe(jvpfa_norm_args& a, const Tensors& x, const Tensors& tx, bool dual, Tensors& alive) const {
    bool grouped[6];
    a.struct_size = sizeof(a);
    a.dtype = dtype_of(x[kX], false);
    a.vec_dtype = vector_type(x) == at::kFloat ? JVPFA_FP32 : a.dtype;
    a.C = (int)x[kX].size(-1), a.M = (int)(x[kX].numel() / a.C);
    a.group_rows = (int)group_rows(x, grouped);
    a.kind = kind, a.post = post, a.alpha = (float)alpha, a.eps = (float)eps;
    a.dual = dual;
    auto keep = [&](const Tensor& t) -> const Tensor& { return alive.emplace_back(t); };
    auto operand = [&](const Tensor& t, const void** p, int64_t* stride) {
      if (!t.defined()) return;
      const Tensor& r = keep(rows(t));
      *p = r.const_data_ptr(), *stride = r.size(0) > 1 ? r.stride(0) : 0;
    };
    operand(x[kX], &a.x, &a.x_stride), operand(x[kY], &a.y, &a.y_stride);
    if (dual) operand(tx[kX], &a.tx, &a.tx_stride), operand(tx[kY], &a.ty, &a.ty_stride);
    for (int i = 0; i < 6; ++i) {
      if (!x[kVectors + i].defined()) continue;
      const Tensor& v = keep(vector(x[kVectors + i], grouped[i]));
      a.vec[i].grouped = grouped[i];
      a.vec[i].v = v.const_data_ptr(), a.vec[i].stride = grouped[i] ? v.stride(0) : 0;
      if (!dual || !tx[kVectors + i].defined()) continue;
      const Tensor& t = keep(vector(tx[kVectors + i], grouped[i]));
      a.vec[i].tv = t.const_data_ptr(), a.vec[i].tv_stride = grouped[i] ? t.stride(0) : 0;
    }
  }
  DualOut forward(const Tensors& x, const Tensors& tx, const Tensors& extras, bool want_kept) const override {
    if (!x[kX].is_cuda()) return python_forward(x, tx, extras, want_kept);
    const Tensor& t = x[kX];
    c10::cuda::OptionalCUDAGuard guard;
    if (t.get_device() != c10::cuda::current_device()) guard.set_index(t.get_device());
    const bool dual = any_defined(tx), sum = x[kY].defined(), norm = kind != JVPFA_NORM_NONE;
    DualOut r;
    r.y.resize(2), r.ty.resize(2);
    auto make = [&](bool wanted) { return wanted ? empty(t.sizes(), t.scalar_type(), t.device()) : Tensor(); };
    r.y[0] = make(sum), r.y[1] = make(norm), r.ty[0] = make(sum && dual), r.ty[1] = make(norm && dual);
    const int64_t M = t.numel() / std::max<int64_t>(t.size(-1), 1);
    if (want_kept) r.kept = empty({M, 8}, at::kFloat, t.device());
    if (t.numel() == 0) return r;
    jvpfa_norm_args a{};
    Tensors alive;
    alive.reserve(16);
    describe(a, x, tx, dual, alive);
    auto at = [](const Tensor& o) { return o.defined() ? o.data_ptr() : nullptr; };
    a.r = at(r.y[0]), a.n = at(r.y[1]), a.tr = at(r.ty[0]), a.tn = at(r.ty[1]);
    if (want_kept) a.stats = static_cast<float*>(r.kept.data_ptr());
    check_status(jvpfa_norm_fwd(&a, c10::cuda::getCurrentCUDAStream(t.get_device()).stream()), "jvpfa_norm_fwd");
    return r;
  }
  Tensors backward(const Tensors& x, const Tensors& tx, const Tensors& extras, const Tensor& kept, const Tensors& g, const Tensors& gt,
                   const std::vector<bool>& want) const override {
    Tensors d(2 * kOperands);
    if (std::find(want.begin(), want.end(), true) == want.end()) return d;
    if (!x[kX].is_cuda()) return python_backward(x, tx, extras, kept, g, gt, want);
    const Tensor& t = x[kX];
    c10::cuda::OptionalCUDAGuard guard;
    if (t.get_device() != c10::cuda::current_device()) guard.set_index(t.get_device());
    const bool dual = any_defined(gt);
    for (int i = 0; i < 2 * kOperands; ++i) {
      const Tensor& of = x[i % kOperands];
      if (!want[i] || !of.defined()) continue;
      const bool nothing = t.numel() == 0 || (i >= kOperands && !dual);
      if (nothing) {
        NoFunctorch nf;
        at::AutoDispatchBelowADInplaceOrView below;
        d[i] = at::zeros(of.sizes(), of.options().requires_grad(false));
      } else {
        d[i] = empty(of.sizes(), of.scalar_type(), of.device());
      }
    }
    if (t.numel() == 0) return d;
    jvpfa_norm_args a{};
    Tensors alive;
    alive.reserve(24);
    describe(a, x, tx, dual, alive);
    a.stats = static_cast<float*>(const_cast<void*>(kept.const_data_ptr()));
    auto cotangent = [&](const Tensor& c) -> const void* { return c.defined() ? alive.emplace_back(dense(c, t)).const_data_ptr() : nullptr; };
    a.gr = cotangent(g[0]), a.gn = cotangent(g[1]);
    if (dual) a.gtr = cotangent(gt[0]), a.gtn = cotangent(gt[1]);
    auto at = [&](int i) { return d[i].defined() && (i < kOperands || dual) ? d[i].data_ptr() : nullptr; };
    a.dx = at(kX), a.dy = at(kY), a.dtx = at(kOperands + kX), a.dty = at(kOperands + kY);
    for (int i = 0; i < 6; ++i) a.d[i] = at(kVectors + i), a.dt[i] = at(kOperands + kVectors + i);
    const int64_t bytes = jvpfa_norm_bwd_workspace(&a);
    const Tensor workspace = bytes > 0 ? empty({bytes}, at::kByte, t.device()) : Tensor();
    if (bytes > 0) a.workspace = workspace.data_ptr(), a.workspace_bytes = bytes;
    check_status(jvpfa_norm_bwd(&a, c10::cuda::getCurrentCUDAStream(t.get_device()).stream()), "jvpfa_norm_bwd");
    return d;
  }
};

// (r, n), None where there is none; None for all: not a case for this path.
py::object norm(const std::vector<std::optional<Tensor>>& operands, int kind, int post, double alpha, double eps, const char* name) {
  const DualOperands in(operands, {});
  if (!in.ok || in.x.size() != kOperands) return py::none();
  const Tensor& x = in.x[kX];
  if (!x.defined() || x.dim() < 1 || (x.is_cuda() && dtype_of(x, false) < 0) || x.size(-1) < 1 || x.size(-1) > JVPFA_NORM_MAX_WIDTH ||
      x.numel() / x.size(-1) > (1 << 30))
    return py::none();
  const Tensor& y = in.x[kY];
  if (y.defined() && (y.sizes() != x.sizes() || y.scalar_type() != x.scalar_type() || y.device() != x.device())) return py::none();
  const at::ScalarType vec = NormOp::vector_type(in.x);
  if (vec != x.scalar_type() && vec != at::kFloat) return py::none();
  for (int i = 0; i < 6; ++i) {
    const Tensor& v = in.x[kVectors + i];
    if (v.defined() && (v.scalar_type() != vec || v.device() != x.device())) return py::none();
  }
  bool grouped[6];
  if (!NormOp::group_rows(in.x, grouped)) return py::none();
  auto op = std::make_shared<NormOp>();
  const std::string which = name;
  op->name = which == "norm" ? "norm" : which == "residual" ? "residual" : "residual_norm";  // (it outlives the caller's text)
  op->outputs = 2, op->module = "jvp_flash_attention_b200.norms";
  op->kind = kind, op->post = post, op->alpha = alpha, op->eps = eps;
  std::vector<py::object> r = apply_dual(op, in);
  return py::make_tuple(r[0], r[1]);
}

std::shared_ptr<NormOp> operator_of(const py::tuple& options) {
  auto op = std::make_shared<NormOp>();
  op->name = "norm", op->outputs = 2, op->module = "jvp_flash_attention_b200.norms";
  op->kind = options[0].cast<int>(), op->post = options[1].cast<int>(), op->alpha = options[2].cast<double>(), op->eps = options[3].cast<double>();
  return op;
}

// The launches as the Python module's Functions make them.
py::tuple launch_fwd(const py::list& x, const py::list& tx, const py::tuple& options, bool keep) {
  const DualOut r = operator_of(options)->forward(tensors_of(x), tensors_of(tx), {}, keep);
  return py::make_tuple(list_of(r.y), list_of(r.ty), none_or(r.kept));
}
py::list launch_bwd(const py::list& x, const py::list& tx, const Tensor& kept, const py::list& g, const py::list& gt, const py::tuple& options,
                    const std::vector<bool>& want) {
  return list_of(operator_of(options)->backward(tensors_of(x), tensors_of(tx), {}, kept, tensors_of(g), tensors_of(gt), want));
}

}  // namespace

void bind_norm(py::module_& m) {
  m.def("norm", &norm, py::arg("operands"), py::arg("kind"), py::arg("post"), py::arg("alpha"), py::arg("eps"), py::arg("name"));
  m.def("norm_launch_fwd", &launch_fwd);
  m.def("norm_launch_bwd", &launch_bwd);
}
