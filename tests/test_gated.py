"""CPU tests of gated_linear: graph, tangents, second derivatives and refusals.  Launches go to the formulas (tests/_block_formulas.py),
which are themselves held against torch's differentiation."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwAD

import jvp_flash_attention_b200.gated as gated
from jvp_flash_attention_b200 import _lib
from jvp_flash_attention_b200.gated import gated_linear
from tests import _block_formulas as formulas

F = torch.nn.functional
PLAIN = {"silu": F.silu, "sigmoid": torch.sigmoid, "gelu": F.gelu, "gelu_tanh": lambda g: F.gelu(g, approximate="tanh")}


@pytest.fixture()
def cpu_kernels(monkeypatch):
    calls = []
    monkeypatch.setattr(gated, "_launch_fwd", lambda *a: (calls.append(("fwd", a[1] is not None, a[5])), formulas.launch_gated_fwd(*a))[1])
    monkeypatch.setattr(gated, "_launch_bwd", lambda *a: (calls.append(("bwd", *a[8:])), formulas.launch_gated_bwd(*a))[1])
    monkeypatch.setattr(gated, "_require_cuda", lambda *a: None)
    return calls


def _inputs(seed, rows=(2, 5), k=4, f=3):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    return r(*rows, k), r(*rows, k), r(f, k), r(f, k), r(*rows, f), r(*rows, f)


def _plain(name):
    return lambda x, wg, wu: PLAIN[name](x @ wg.T) * (x @ wu.T)


@pytest.mark.parametrize("route", ["func", "fwad"])
@pytest.mark.parametrize("name", list(PLAIN))
@pytest.mark.parametrize("through", ["h", "t", "both"])
def test_values_tangents_and_gradients(cpu_kernels, route, name, through):
    x, tx, wg, wu, gh, gth = _inputs(1)
    leaves = [t.requires_grad_() for t in (x, tx, wg, wu)]
    want = torch.func.jvp(lambda v: _plain(name)(v, wg, wu), (x,), (tx,))
    if route == "func":
        got = torch.func.jvp(lambda v: gated_linear(v, wg, wu, name), (x,), (tx,))
    else:
        with fwAD.dual_level():
            got = fwAD.unpack_dual(gated_linear(fwAD.make_dual(x, tx), wg, wu, name))
    pick = {"h": [0], "t": [1], "both": [0, 1]}[through]
    for a, b in zip(got, want):
        torch.testing.assert_close(a, b)
    args = [[o[i] for i in pick] for o in (got, want)]
    cots = [(gh, gth)[i] for i in pick]
    for a, b in zip(torch.autograd.grad(args[0], leaves, cots, allow_unused=True), torch.autograd.grad(args[1], leaves, cots, allow_unused=True)):
        assert (a is None) == (b is None) or not (a if b is None else b).any()
        if a is not None and b is not None:
            torch.testing.assert_close(a, b)


@pytest.mark.parametrize("name", list(PLAIN))
def test_gradients_against_differences(cpu_kernels, name):
    x, _, wg, wu, _, _ = _inputs(2)
    torch.autograd.gradcheck(lambda *a: gated_linear(*a, name), tuple(t.requires_grad_() for t in (x, wg, wu)))
    torch.autograd.gradgradcheck(lambda *a: gated_linear(*a, name), (x, wg, wu))


def test_a_gradient_penalty_reaches_the_weights(cpu_kernels):
    x, _, wg, wu, gh, v = _inputs(3)
    leaves = [t.requires_grad_() for t in (x, wg, wu)]
    gh.requires_grad_()
    out = []
    for f in (gated_linear, _plain("silu")):
        (dx,) = torch.autograd.grad(f(*leaves), x, gh, create_graph=True)
        out.append(torch.autograd.grad((dx**2).sum(), (*leaves, gh)))
    for a, b in zip(*out):
        torch.testing.assert_close(a, b)


@pytest.mark.parametrize("wanted", ["xg", "g", "u", "xgu"])
def test_second_derivatives_through_the_weights(cpu_kernels, wanted):
    """Hessian-vector products of a loss with respect to x and the weights, whichever of them the product's vector lies along."""
    x, tx, wg, wu, gh, _ = _inputs(3)
    leaves = [t.requires_grad_() for t in (x, wg, wu)]
    along = [t for t, name in zip(leaves, "xgu") if name in wanted]
    vectors = [torch.randn(t.shape, generator=torch.Generator().manual_seed(i), dtype=t.dtype) for i, t in enumerate(along)]
    out = []
    for f in (gated_linear, _plain("silu")):
        grads = torch.autograd.grad((f(*leaves) * gh).tanh().sum(), along, create_graph=True)
        out.append(torch.autograd.grad(grads, leaves, vectors))
    for a, b in zip(*out):
        torch.testing.assert_close(a, b)


def test_what_cannot_be_differentiated_says_so(cpu_kernels):
    x, tx, wg, wu, gh, gth = _inputs(4)
    leaves = [t.requires_grad_() for t in (x, wg, wu)]
    dx, dw = torch.autograd.grad(gated_linear(*leaves), (x, wg), gh, create_graph=True)
    (h,) = torch.autograd.grad((dw**2).sum() + (dx**2).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="third time"):
        torch.autograd.grad(h.sum(), x)
    h, th = torch.func.jvp(lambda v: gated_linear(v, wg, wu), (x,), (tx,))
    (dx,) = torch.autograd.grad(th, x, gth, create_graph=True, retain_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated a second time"):
        torch.autograd.grad(dx.sum(), x)
    # ... but the part through h can
    (dx,) = torch.autograd.grad(h, x, gh, create_graph=True)
    torch.autograd.grad(dx.sum(), x)


@pytest.mark.parametrize("route", ["func", "fwad", "nested"])
@pytest.mark.parametrize("given", ["g", "u", "xg", "xgu"])
def test_tangents_of_the_weights(cpu_kernels, route, given):
    x, _, wg, wu, gh, gth = _inputs(13)
    primals = [t.requires_grad_() for t in (x, wg, wu)]
    tangents = [torch.randn(t.shape, generator=torch.Generator().manual_seed(i), dtype=t.dtype).requires_grad_(n in given)
                for i, (t, n) in enumerate(zip(primals, "xgu"))]
    at = [i for i, n in enumerate("xgu") if n in given]
    leaves = primals + [tangents[i] for i in at]
    out = []
    for f in (gated_linear, _plain("silu")):
        def along(*some):
            args = list(primals)
            for i, t in zip(at, some):
                args[i] = t
            return f(*args)

        p, t = tuple(primals[i] for i in at), tuple(tangents[i] for i in at)
        if route == "nested":
            def value(*some):
                return torch.func.vjp(along, *some)[0]

            y, ty = torch.func.jvp(value, p, t)
        elif route == "func":
            y, ty = torch.func.jvp(along, p, t)
        else:
            with fwAD.dual_level():
                y, ty = fwAD.unpack_dual(along(*(fwAD.make_dual(a, b) for a, b in zip(p, t))))
        out.append((y, ty, *torch.autograd.grad((y, ty), leaves, (gh, gth))))
    for a, b in zip(*out):
        torch.testing.assert_close(a, b)


def test_nested_transforms_take_the_general_route(cpu_kernels):
    x, tx, wg, wu, gh, v = _inputs(5)
    f, plain = (lambda a: (gated_linear(a, wg, wu) * gh).sum()), (lambda a: (_plain("silu")(a, wg, wu) * gh).sum())
    torch.testing.assert_close(torch.func.grad(f)(x), torch.func.grad(plain)(x))
    torch.testing.assert_close(torch.func.grad(lambda w: (gated_linear(x, w, wu) * gh).sum())(wg),
                               torch.func.grad(lambda w: (_plain("silu")(x, w, wu) * gh).sum())(wg))
    torch.testing.assert_close(torch.func.grad(lambda a: (torch.func.grad(f)(a) * tx).sum())(x),
                               torch.func.grad(lambda a: (torch.func.grad(plain)(a) * tx).sum())(x))


@pytest.mark.parametrize("outputs", ["h", "both"])
def test_a_functorch_transform_of_the_cotangent(cpu_kernels, monkeypatch, outputs):
    """d/dc <dx(c), v> of a graph built outside the transform is th along v; through the tangent it is refused."""
    def plain(launch):
        def run(*args):
            with torch.no_grad(), _lib.native().NoFunctorch():
                return launch(*(gated._unwrap(t).detach() if isinstance(t, torch.Tensor) else t for t in args))
        return run

    monkeypatch.setattr(gated, "_launch_fwd", plain(formulas.launch_gated_fwd))
    monkeypatch.setattr(gated, "_launch_bwd", plain(formulas.launch_gated_bwd))
    x, tx, wg, wu, gh, gth = _inputs(11)
    v = _inputs(12)[0]
    x.requires_grad_()
    if outputs == "h":
        outs = (gated_linear(x, wg, wu),)
    else:
        outs = torch.func.jvp(lambda a: gated_linear(a, wg, wu), (x,), (tx,))
    grad = lambda cots: torch.autograd.grad(outs, x, cots, retain_graph=True, create_graph=True)[0]  # noqa: E731
    got = torch.func.grad(lambda c: (grad((c, gth)[:len(outs)]) * v).sum())(gh)
    torch.testing.assert_close(got, formulas.gated_fwd(x.detach(), v, wg, wu, 0)[1])
    if outputs == "both":
        with pytest.raises(RuntimeError, match="cannot be differentiated a second time"):
            torch.func.grad(lambda c: (grad((gh, c)) * v).sum())(gth)


def test_only_what_is_asked_for_is_computed(cpu_kernels):
    x, tx, wg, wu, gh, gth = _inputs(6)
    gated_linear(x, wg, wu)
    assert cpu_kernels == [("fwd", False, False)]  # nothing kept without a graph
    cpu_kernels.clear()
    h = gated_linear(x, wg.requires_grad_(), wu)
    torch.autograd.grad(h, wg, gh)
    assert cpu_kernels == [("fwd", False, True), ("bwd", False, False, True)]
    cpu_kernels.clear()
    wg.requires_grad_(False)
    _, th = torch.func.jvp(lambda v: gated_linear(v, wg, wu), (x,), (tx.requires_grad_(),))
    torch.autograd.grad(th, tx, gth)
    assert cpu_kernels == [("fwd", True, True), ("bwd", False, True, False)]


def test_a_run_of_operators_under_one_jvp(cpu_kernels):
    """A feed-forward block: the gated projection, the narrowing product and the residual."""
    x, tx, wg, wu, _, _ = _inputs(7)
    wd = _inputs(8, k=3, f=4)[2]
    leaves = [t.requires_grad_() for t in (x, wg, wu, wd)]
    block = lambda f: lambda v: v + F.linear(f(v, wg, wu), wd)  # noqa: E731
    out = []
    for f in (gated_linear, _plain("silu")):
        y, ty = torch.func.jvp(block(f), (x,), (tx,))
        out.append((y, ty, *torch.autograd.grad((y.sum() + (ty**2).sum()), leaves)))
    for a, b in zip(*out):
        torch.testing.assert_close(a, b)


def test_refusals(cpu_kernels):
    x, tx, wg, wu, _, _ = _inputs(9)
    for error, args in [(ValueError, (x, wg, wu, "relu")), (ValueError, (x, wg[0], wu[0])), (ValueError, (x, wg, wu[:2])),
                        (ValueError, (x[..., :3], wg, wu)), (ValueError, (x, wg[:0], wu[:0])), (TypeError, (x, wg.float(), wu)),
                        (ValueError, (x[..., 0:0], wg[:, :0], wu[:, :0]))]:
        with pytest.raises(error):
            gated_linear(*args)


def test_no_cpu_fallback():
    x, _, wg, wu, _, _ = (t.float() for t in _inputs(10))
    with pytest.raises(RuntimeError, match="runs only on CUDA tensors"):
        gated_linear(x, wg, wu)


def _fwd_args(**kw):
    a = _lib.GatedFwdArgs()
    a.struct_size = ctypes.sizeof(a)
    a.M = a.K = a.F = 64
    a.x = a.wg = a.wu = a.h = 256
    a.x_stride = a.wg_stride = a.wu_stride = 64
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _bwd_args(**kw):
    a = _lib.GatedBwdArgs()
    a.struct_size = ctypes.sizeof(a)
    a.M = a.K = a.F = 64
    a.x = a.wg = a.wu = a.kept = a.gh = a.dx = a.workspace = 256
    a.x_stride = a.wg_stride = a.wu_stride = 64
    a.workspace_bytes = 1 << 30
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_the_c_entries_refuse():
    lib = _lib.load()
    assert lib.jvpfa_gated_fwd(None, None) == -1 and lib.jvpfa_gated_bwd(None, None) == -1
    common = [(-7, dict(struct_size=4)), (-3, dict(dtype=3)), (-2, dict(M=0)), (-10, dict(M=2**31 - 1)), (-10, dict(F=2**31 - 4000)), (-2, dict(K=0)), (-2, dict(F=0)), (-9, dict(activation=4)),
              (-9, dict(activation=-1)), (-1, dict(x=None)), (-1, dict(wg=None)), (-1, dict(wu=None)), (-8, dict(x=257)), (-2, dict(x_stride=-8))]
    for want, kw in common + [(-1, dict(h=None)), (-8, dict(h=264)), (-1, dict(tx=256)), (-1, dict(th=256)), (-8, dict(kept=264)),
                              (-1, dict(x=258)), (-1, dict(dtype=2))]:  # the last two need a workspace
        assert lib.jvpfa_gated_fwd(ctypes.byref(_fwd_args(**kw)), None) == want, kw
    for want, kw in common + [(-1, dict(kept=None)), (-1, dict(gh=None)), (-1, dict(gth=256)), (-1, dict(gth=256, tx=256)), (-1, dict(dtx=256)), (-1, dict(dwg=256)), (-1, dict(dx=None)),
                              (-8, dict(dx=264)), (-8, dict(gh=258)), (-1, dict(workspace=None)), (-1, dict(workspace_bytes=16))]:
        assert lib.jvpfa_gated_bwd(ctypes.byref(_bwd_args(**kw)), None) == want, kw


def test_workspaces():
    lib = _lib.load()
    fwd = lambda **kw: lib.jvpfa_gated_fwd_workspace(ctypes.byref(_fwd_args(**kw)))  # noqa: E731
    assert fwd() == 0
    assert fwd(x=258) == 64 * 64 * 2  # rows that begin elsewhere are copied
    assert fwd(x_stride=65) == 64 * 64 * 2 and fwd(K=63, x_stride=63) == 64 * 64 * 2  # rows padded to 16 bytes; wg and wu have them
    assert fwd(x_stride=0) == 64 * 64 * 2  # one row for all
    assert fwd(dtype=2) == 3 * 64 * 64 * 2  # fp32: three parts, up to 128 rows of x alone
    assert fwd(dtype=2, M=256) == 3 * (256 + 2 * 64) * 64 * 2
    bwd = lambda **kw: lib.jvpfa_gated_bwd_workspace(ctypes.byref(_bwd_args(**kw)))  # noqa: E731
    assert bwd() == 2 * 64 * 64 * 2
    assert bwd(gth=256, tx=256, kept_tangent=1, tx_stride=64) == 2 * 2 * 64 * 64 * 2
    assert bwd(dtype=2) == 3 * 2 * 64 * 64 * 2 and bwd(dtype=2, M=256) == 3 * (2 * 256 * 64 + 2 * 64 * 64) * 2
    assert bwd(M=0) == 0
    # tiles whose depth is worth cutting: 2 x 28 672 of the contraction, two rows of 16 tiles, 2 pieces each of 256 x 256 sums
    assert bwd(M=300, K=4096, F=28672, x_stride=4096, wg_stride=4096, wu_stride=4096) == 2 * 300 * 28672 * 2 + 32 * 2 * 256 * 256 * 4
    assert bwd(M=2**26 + 64, dx=None, dwg=256, dwu=256) == 0 < bwd(M=2**26, dx=None, dwg=256, dwu=256)  # sums of more k-blocks than a wait lasts
    kept = lib.jvpfa_gated_kept_bytes
    assert kept(0, 1, 1, 0) == 2 * 1024 * 3 and kept(2, 33, 40, 1) == 4 * 4 * 1024 * 4 and kept(3, 1, 1, 0) == kept(0, 0, 1, 0) == 0
