"""CPU tests of norm, residual and residual_norm: graph, tangents, levels and refusals.  Launches go to the formulas (tests/_norm_formulas.py)."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwAD

import jvp_flash_attention_b200.norms as norms
from jvp_flash_attention_b200 import _lib
from tests import _norm_formulas as formulas

B, L, C = 2, 3, 6
SHAPES = {"x": (B, L, C), "y": (B, L, C), "weight": (C,), "bias": (C,), "scale": (B, 1, C), "shift": (B, 1, C), "gate": (B, 1, C), "post_weight": (C,)}


@pytest.fixture()
def cpu(monkeypatch):
    calls = []

    def forward(x, tx, *args):
        calls.append("dual" if any(t is not None for t in tx) else "value")
        return formulas.stub_fwd(x, tx, *args)

    monkeypatch.setattr(norms, "_launch_fwd", forward)
    monkeypatch.setattr(norms, "_launch_bwd", formulas.stub_bwd)
    monkeypatch.setattr(norms, "_require_cuda", lambda *a: None)
    return calls


def _operands(seed, std=1.0, grad=False):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g, dtype=torch.float64) * std).requires_grad_(grad) for s in SHAPES.values()]


def _own(x, y, w, b, sc, sh, gate, pw):
    return norms.residual_norm(x, y, w, b, scale=sc, shift=sh, gate=gate, post="rms", post_weight=pw, alpha=0.5, kind="layer")


def _exact(*x):
    return formulas._value(x, 2, 1, 0.5, 1e-6)


def _close(a, b):
    for s, t in zip(a, b, strict=True):
        torch.testing.assert_close(s, t)


@pytest.mark.parametrize("route", ["func", "fwad"])
def test_values_tangents_and_gradients(cpu, route):
    x, tx, cots = _operands(1, grad=True), _operands(2, 0.3, True), [_operands(3)[0] for _ in range(2)] + [_operands(4)[0] for _ in range(2)]
    results = []
    for f in (_own, _exact):
        cpu.clear()
        if route == "func" or f is _exact:
            y, ty = torch.func.jvp(f, tuple(x), tuple(tx))
        else:
            with fwAD.dual_level():
                y, ty = zip(*(fwAD.unpack_dual(o) for o in f(*map(fwAD.make_dual, x, tx))))
        assert f is _exact or cpu == ["dual"]  # one launch for values and tangents
        results.append((*y, *ty, *torch.autograd.grad((*y, *ty), (*x, *tx), cots)))
    _close(*results)


@pytest.mark.parametrize("present", [("x",), ("x", "weight"), ("x", "bias", "shift"), ("x", "scale"), ("x", "y"), ("x", "y", "gate"), ("x", "y", "post_weight")])
@pytest.mark.parametrize("kind,post", [("rms", None), ("layer", "layer"), (None, "rms")])
def test_absent_operands_against_differences(cpu, present, kind, post):
    if kind is None and ("y" not in present or set(present) & {"weight", "bias", "scale", "shift"}):
        pytest.skip("no norm of x alone")
    x = [t for n, t in zip(SHAPES, _operands(5, grad=True)) if n in present]

    def f(*xs):
        p = dict(zip(present, xs))
        if "y" not in p:
            return norms.norm(kind=kind, **p)
        return norms.residual(post=post, **p) if kind is None else norms.residual_norm(kind=kind, post=post, **p)

    torch.autograd.gradcheck(f, x, check_forward_ad=True)
    torch.autograd.gradgradcheck(f, x)


def test_only_what_is_asked_for(cpu):
    x = _operands(6)
    x[2].requires_grad_()
    r, n = _own(*x)
    assert n.requires_grad and torch.autograd.grad(n.sum(), x[2])[0].shape == (C,)
    with torch.no_grad():
        assert not _own(*x)[1].requires_grad
    t = torch.randn(B, L, C, dtype=torch.float64)
    _, tn = torch.func.jvp(lambda a: _exact(a, *x[1:])[1], (x[0].detach(),), (t,))
    with fwAD.dual_level():  # a tangent of one operand alone
        r, n = _own(fwAD.make_dual(x[0].detach(), t), *(v.detach() for v in x[1:]))
        torch.testing.assert_close(fwAD.unpack_dual(n).tangent, tn.detach())


def test_nested_transforms(cpu):
    x, v = [t.detach() for t in _operands(7)], [t.detach() for t in _operands(8)]
    results = []
    for f in (_own, _exact):
        loss = lambda *a: sum((o**3).sum() for o in f(*a))  # noqa: B023, E731
        grad = torch.func.grad(loss, argnums=tuple(range(8)))
        g, hv = torch.func.jvp(grad, tuple(x), tuple(v))
        rr = torch.func.grad(lambda *a: sum((s * t).sum() for s, t in zip(grad(*a), v)), argnums=tuple(range(8)))(*x)
        vj = torch.func.vjp(f, *x)[1](tuple(f(*x)))
        results.append((*g, *hv, *rr, *vj))
    _close(*results)


def test_gradients_inside_a_level_are_dual(cpu):
    """Forward over reverse; the gradient of the value can then be differentiated, its tangent is a further backward."""
    x, tx = _operands(9, grad=True), [t.detach() for t in _operands(10)]
    results = []
    for f in (_own, _exact):
        with fwAD.dual_level():
            out = f(*map(fwAD.make_dual, x, tx))
            g = torch.autograd.grad(sum((fwAD.unpack_dual(o).primal ** 1 * o).sum() for o in out), x)
            results.append([t for d in g for t in fwAD.unpack_dual(d)])
    _close(*results)


def test_a_transform_of_the_cotangent(cpu):
    x, c, u = _operands(11, grad=True), _operands(12)[0].detach(), [t.detach() for t in _operands(13)]
    results = []
    for f in (_own, _exact):
        out = f(*x)
        vjp = lambda a: torch.autograd.grad(out[1], x, a, retain_graph=True, create_graph=True, materialize_grads=True)  # noqa: B023, E731
        results.append([torch.func.grad(lambda a: sum((d * w).sum() for d, w in zip(vjp(a), u)))(c)])  # noqa: B023
    _close(*results)


def test_what_is_refused(cpu):
    x = _operands(14, grad=True)
    plain = [t.detach() for t in x]
    r, n = _own(*x)
    d = torch.autograd.grad((n**2).sum(), x[0], create_graph=True)[0]
    d2 = torch.autograd.grad((d**2).sum(), x[0], create_graph=True)[0]
    with pytest.raises(RuntimeError, match="no third derivative"):
        torch.autograd.grad(d2.sum(), x[0])
    _, ty = torch.func.jvp(_own, tuple(x), tuple(plain))
    d = torch.autograd.grad(ty[1].sum(), x[0], create_graph=True)[0]
    with pytest.raises(RuntimeError, match="no second derivative through the tangent"):
        torch.autograd.grad(d.sum(), x[0])
    with pytest.raises(RuntimeError, match="further forward"):
        torch.func.jvp(lambda a: torch.func.jvp(norms.norm, (a,), (a,))[1], (plain[0],), (plain[0],))
    with pytest.raises(NotImplementedError, match="no rule for"):
        torch.func.vmap(lambda a: norms.norm(a, plain[2]))(plain[0])
    with pytest.raises(NotImplementedError, match="no rule for"):
        torch.autograd.grad(n, x[0], torch.ones(2, B, L, C, dtype=torch.float64), is_grads_batched=True)


def test_bad_arguments(cpu):
    x, y, w, b, sc, sh, gate, pw = _operands(15)
    for error, f in [
        (ValueError, lambda: norms.norm(x, kind="mean")), (ValueError, lambda: norms.norm(x, kind=None)), (ValueError, lambda: norms.residual_norm(x, y, kind=None)),
        (ValueError, lambda: norms.residual(x, y[:1])), (TypeError, lambda: norms.residual(x, y.float())), (ValueError, lambda: norms.norm(x, w[:3])),
        (ValueError, lambda: norms.norm(x, scale=torch.ones(1, L, C, dtype=torch.float64))), (ValueError, lambda: norms.norm(x, scale=torch.ones(B, C, dtype=torch.float64))),
        (ValueError, lambda: norms.norm(x, scale=sc, shift=torch.ones(B, L, C, dtype=torch.float64))), (TypeError, lambda: norms.norm(x, w, b.float())),
        (TypeError, lambda: norms.norm(x, w.half())), (ValueError, lambda: norms.norm(x[..., :0])), (ValueError, lambda: norms.norm(torch.ones((), dtype=torch.float64))),
        (ValueError, lambda: norms.residual(x, y, post="x")), (ValueError, lambda: norms.norm(torch.ones(1, norms.MAX_WIDTH + 1))),
    ]:
        with pytest.raises(error):
            f()


def test_no_cpu_fallback():
    with pytest.raises(RuntimeError, match="runs only on CUDA tensors"):
        norms.norm(torch.ones(2, 3))


def test_the_c_entries_refuse():
    lib = _lib.load()

    def call(entry, **kw):
        a = _lib.NormArgs()
        a.struct_size = ctypes.sizeof(a)
        a.M, a.C, a.group_rows, a.kind, a.x, a.x_stride = 4, 8, 2, 1, 64, 8
        a.n, a.stats = 64, 64
        for key, v in kw.items():
            if key == "vec":
                for i, (p, t) in v.items():
                    a.vec[i].v, a.vec[i].tv = p, t
            elif key in ("d", "dt"):
                getattr(a, key)[v] = 64
            else:
                setattr(a, key, v)
        return entry(ctypes.byref(a), None) if entry is not lib.jvpfa_norm_bwd_workspace else entry(ctypes.byref(a))

    both = [(-7, dict(struct_size=8)), (-3, dict(dtype=3)), (-3, dict(vec_dtype=1)), (-2, dict(M=0)), (-2, dict(C=0)), (-2, dict(C=16385)), (-10, dict(M=1 << 30 | 2)), (-2, dict(group_rows=3)),
            (-9, dict(kind=3)), (-9, dict(kind=0)), (-9, dict(post=1)), (-9, dict(ty=64)), (-1, dict(x=None)), (-1, dict(tx=64)), (-2, dict(x_stride=-8)),
            (-1, dict(vec={0: (None, 64)})), (-1, dict(vec={0: (64, 64)})), (-9, dict(vec={4: (64, None)})), (-8, dict(x=65)), (-8, dict(vec={1: (63, None)})), (-8, dict(stats=68))]
    forward = [(-1, dict(n=None)), (-1, dict(r=64)), (-1, dict(dual=1)), (-1, dict(y=64))]
    backward = [(-1, dict(stats=None)), (-1, dict(dy=64)), (-1, dict(gtn=64)), (-1, dict(dtx=64)), (-1, dict(d=0)), (-1, dict(vec={0: (64, None)}, dt=0)), (-8, dict(gn=63)),
                (-1, dict(vec={0: (64, None)}, d=0))]  # (the last: a workspace is needed)
    for entry, cases in ((lib.jvpfa_norm_fwd, both + forward), (lib.jvpfa_norm_bwd, both + backward)):
        assert entry(None, None) == -1
        for want, kw in cases:
            assert call(entry, **kw) == want, kw
    assert call(lib.jvpfa_norm_bwd_workspace, vec={0: (64, None)}, d=0) > 0 and call(lib.jvpfa_norm_bwd_workspace) == 0
    assert call(lib.jvpfa_norm_bwd_workspace, M=0) == 0
