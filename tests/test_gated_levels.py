"""CPU tests of gated_linear's gradients where forward mode goes over them: inside a forward-AD level and under functorch transforms.
Launches go to the formulas (tests/_block_formulas.py), and what they add up to is held against torch's differentiation of the plain form."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

import jvp_flash_attention_b200.gated as gated
from jvp_flash_attention_b200 import _lib
from jvp_flash_attention_b200.gated import ACTIVATIONS, gated_linear
from tests import _block_formulas as formulas


def _in_memory(launch):
    """The launch as the GPU's is: it reads what is in the tensors' memory, whatever transforms they belong to."""
    def run(*args):
        with torch.no_grad(), _lib.native().NoFunctorch():
            plain = [fwAD.unpack_dual(gated._unwrap(t)).primal.detach() if isinstance(t, torch.Tensor) else t for t in args]
            return launch(*(gated._in_memory(t) if isinstance(t, torch.Tensor) else t for t in plain))
    return run


@pytest.fixture(autouse=True)
def cpu_kernels(monkeypatch):
    monkeypatch.setattr(gated, "_launch_fwd", _in_memory(formulas.launch_gated_fwd))
    monkeypatch.setattr(gated, "_launch_bwd", _in_memory(formulas.launch_gated_bwd))
    monkeypatch.setattr(gated, "_require_cuda", lambda *a: None)


def _inputs(seed, k=4, f=3):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    return {"x": r(2, 5, k), "wg": r(f, k), "wu": r(f, k), "tx": r(2, 5, k), "tg": r(f, k), "tu": r(f, k), "gh": r(2, 5, f), "tgh": r(2, 5, f),
            "wd": r(k, f)}


def _plain(name):
    act = lambda g: formulas.activation(ACTIVATIONS[name], g)[0]  # noqa: E731  (elementary operations, which torch differentiates in any order)
    return lambda x, wg, wu: act(x @ wg.T) * (x @ wu.T)


def _forward_over_reverse(loss, primals, tangents):
    """(gradients, their tangents), by torch."""
    return torch.func.jvp(lambda *a: torch.func.grad(loss, argnums=tuple(range(len(primals))))(*a), tuple(primals), tuple(tangents))


@pytest.mark.parametrize("name", list(ACTIVATIONS))
@pytest.mark.parametrize("given", ["x", "g", "xgu"])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("create_graph", [False, True])
def test_gradients_inside_a_level_carry_their_tangents(name, given, residual, create_graph):
    i = _inputs(1)
    primals = [i[n].requires_grad_() for n in ("x", "wg", "wu")]
    tangents = [t if n in given else torch.zeros_like(t) for n, t in zip("xgu", (i["tx"], i["tg"], i["tu"]))]
    block = lambda f: lambda x, wg, wu: ((x + f(x, wg, wu) @ i["wd"].T if residual else f(x, wg, wu)) ** 3).sum()  # noqa: E731
    want, moving = _forward_over_reverse(block(_plain(name)), [p.detach() for p in primals], tangents)
    with fwAD.dual_level():
        duals = [fwAD.make_dual(p, t) if n in given else p for n, p, t in zip("xgu", primals, tangents)]
        y = block(lambda *a: gated_linear(*a, name))(*duals)
        grads = torch.autograd.grad(y, primals, create_graph=create_graph)
        for d, w, m in zip(grads, want, moving):
            d, t = fwAD.unpack_dual(d)
            torch.testing.assert_close(d, w)
            torch.testing.assert_close(t, m)


def test_a_cotangent_that_alone_is_dual():
    """The gradient is linear in it; with a graph, its tangent can be differentiated as the gradient can."""
    i = _inputs(2)
    leaves = [i[n].requires_grad_() for n in ("x", "wg", "wu", "gh", "tgh")]
    out = []
    for f in (gated_linear, _plain("silu")):
        y = f(*leaves[:3])
        with fwAD.dual_level():
            if f is gated_linear:
                grads = torch.autograd.grad(y, leaves[:3], fwAD.make_dual(leaves[3], leaves[4]), create_graph=True)
                pairs = [tuple(fwAD.unpack_dual(d)) for d in grads]
            else:
                pairs = list(zip(*(torch.autograd.grad(y, leaves[:3], c, create_graph=True) for c in leaves[3:])))
        flat = [t for p in pairs for t in p]
        out.append([*flat, *torch.autograd.grad(sum((t**2).sum() for t in flat), leaves)])
    for a, b in zip(*out):
        torch.testing.assert_close(a, b)


def test_dual_cotangents_of_a_graph_with_a_tangent():
    """A call under torch.func.jvp, whose graph is walked later with dual cotangents of both outputs."""
    i = _inputs(3)
    leaves = [i[n].requires_grad_() for n in ("x", "wg", "wu", "tx")]
    both = torch.func.jvp(lambda v: gated_linear(v, leaves[1], leaves[2]), (leaves[0],), (leaves[3],))
    cots, tangents = (i["gh"], i["tgh"]), (i["tgh"] * 2, i["gh"] - 1)
    want = [torch.autograd.grad(both, leaves, c, retain_graph=True) for c in (cots, tangents)]
    with fwAD.dual_level():
        got = torch.autograd.grad(both, leaves, [fwAD.make_dual(c, t) for c, t in zip(cots, tangents)], retain_graph=True)
        for d, w, t in zip(got, *want):
            d, td = fwAD.unpack_dual(d)
            torch.testing.assert_close(d, w)
            torch.testing.assert_close(td, t)


@pytest.mark.parametrize("through", ["t", "both"])
def test_a_third_derivative_is_nan_and_the_gradient_right(through):
    i = _inputs(4)
    leaves = [i[n].requires_grad_() for n in ("x", "wg", "wu")]
    cots = [i["gh"], i["tgh"]][through == "t":]
    out = []
    for inside in (False, True):
        with fwAD.dual_level():
            both = tuple(fwAD.unpack_dual(gated_linear(fwAD.make_dual(leaves[0], i["tx"]), *leaves[1:])))[through == "t":]
            if inside:
                duals = [fwAD.unpack_dual(d) for d in torch.autograd.grad(both, leaves, cots)]
                assert all(d.tangent.isnan().all() for d in duals)
                out.append([d.primal for d in duals])
        if not inside:
            out.append(torch.autograd.grad(both, leaves, cots))
    for a, b in zip(*out):
        torch.testing.assert_close(a, b)


def test_a_tangent_of_a_gradient_is_not_differentiated_again():
    i = _inputs(5)
    x = i["x"].requires_grad_()
    with fwAD.dual_level():
        (d,) = torch.autograd.grad((gated_linear(fwAD.make_dual(x, i["tx"]), i["wg"], i["wu"]) ** 2).sum(), x, create_graph=True)
        d, td = fwAD.unpack_dual(d)
        with pytest.raises(RuntimeError, match="third time"):
            torch.autograd.grad(td.sum(), x, retain_graph=True)
        torch.autograd.grad(d.sum(), x)


@pytest.mark.parametrize("wanted", ["x", "xgu"])
def test_second_derivatives_inside_a_level(wanted):
    """Linear in the vector they are taken along; a third derivative where the operands move, NaN beside what is right."""
    i = _inputs(6)
    leaves = [i[n].requires_grad_() for n in ("x", "wg", "wu", "gh")]
    at = [n for n, k in enumerate("xgu") if k in wanted]
    v, tv = [i[("tx", "tg", "tu")[k]] for k in at], [leaves[k].detach() for k in at]
    want = []
    for along in (v, tv):
        grads = torch.autograd.grad(_plain("silu")(*leaves[:3]), [leaves[k] for k in at], leaves[3], create_graph=True)
        want.append(torch.autograd.grad(grads, leaves, along))
    with fwAD.dual_level():
        grads = torch.autograd.grad(gated_linear(*leaves[:3]), [leaves[k] for k in at], leaves[3], create_graph=True)
        got = torch.autograd.grad(grads, leaves, [fwAD.make_dual(a, b) for a, b in zip(v, tv)])
        for d, w, m in zip(got, *want):
            d, t = fwAD.unpack_dual(d)
            torch.testing.assert_close(d, w)
            torch.testing.assert_close(t, m)
        moving = fwAD.make_dual(leaves[0], i["tx"])
        grads = torch.autograd.grad(gated_linear(moving, *leaves[1:3]), [leaves[k] for k in at], leaves[3], create_graph=True)
        got = torch.autograd.grad([fwAD.unpack_dual(d).primal for d in grads], leaves, v)
        for d, w in zip(got, want[0]):
            d, t = fwAD.unpack_dual(d)
            torch.testing.assert_close(d, w)
            assert t.isnan().all()


@pytest.mark.parametrize("given", ["x", "g", "xgu"])
@pytest.mark.parametrize("name", list(ACTIVATIONS))
def test_torch_func_jvp_of_torch_func_grad(name, given):
    i = _inputs(7)
    at = [n for n, k in enumerate("xgu") if k in given]
    primals, tangents = [i[n] for n in ("x", "wg", "wu")], [i[n] for n in ("tx", "tg", "tu")]

    def loss(f):
        def run(*some):
            args = list(primals)
            for k, t in zip(at, some):
                args[k] = t
            return ((args[0] + f(*args) @ i["wd"].T) ** 3).sum()
        return run

    got, want = (_forward_over_reverse(loss(f), [primals[k] for k in at], [tangents[k] for k in at])
                 for f in (lambda *a: gated_linear(*a, name), _plain(name)))
    for a, b in zip((*got[0], *got[1]), (*want[0], *want[1])):
        torch.testing.assert_close(a, b)


def test_torch_func_jvp_of_a_vjp():
    """The gradient is linear in the cotangent, whether the graph is torch.func's or an ordinary one."""
    i = _inputs(8)
    _, vjp = torch.func.vjp(lambda *a: gated_linear(*a), i["x"], i["wg"], i["wu"])
    want = [torch.func.vjp(_plain("silu"), i["x"], i["wg"], i["wu"])[1](c) for c in (i["gh"], i["tgh"])]
    for a, b in zip(torch.func.jvp(vjp, (i["gh"],), (i["tgh"],)), want):
        for d, w in zip(a, b):
            torch.testing.assert_close(d, w)


def test_torch_func_jvp_of_a_vjp_through_the_tangent():
    i = _inputs(12)
    along = lambda x, wg: torch.func.jvp(lambda v: gated_linear(v, wg, i["wu"]), (x,), (i["tx"],))  # noqa: E731
    _, vjp = torch.func.vjp(along, i["x"], i["wg"])
    cots, tangents = (i["gh"], i["tgh"]), (i["tgh"] - 1, i["gh"])
    for a, b in zip(torch.func.jvp(vjp, (cots,), (tangents,)), (vjp(cots), vjp(tangents))):
        for d, w in zip(a, b):
            torch.testing.assert_close(d, w)
    with pytest.raises(RuntimeError, match="cannot be differentiated a second time"):
        torch.func.grad(lambda x: torch.func.grad(lambda v: along(v, i["wg"])[1].sum())(x).sum())(i["x"])


@pytest.mark.parametrize("outputs", ["h", "t", "both"])
def test_torch_func_jvp_of_the_cotangents_of_an_ordinary_graph(outputs):
    i = _inputs(10)
    leaves = [i[n].requires_grad_() for n in ("x", "tx", "wg", "wu")]
    pick = {"h": [0], "t": [1], "both": [0, 1]}[outputs]
    graph = torch.func.jvp(lambda v: gated_linear(v, *leaves[2:]), tuple(leaves[:1]), tuple(leaves[1:2]))
    grads = lambda *c: torch.autograd.grad([graph[k] for k in pick], leaves[::2], c, retain_graph=True)  # noqa: E731
    cots, tangents = (tuple(([i["gh"], i["tgh"]] if n == 0 else [i["tgh"] - 1, i["gh"]])[k] for k in pick) for n in (0, 1))
    for a, b in zip(torch.func.jvp(grads, cots, tangents), (grads(*cots), grads(*tangents))):
        for d, w in zip(a, b):
            torch.testing.assert_close(d, w)


def test_torch_func_grad_of_dual_tensors():
    i = _inputs(11)
    loss = lambda f: lambda v: (f(v, i["wg"], i["wu"]) ** 3).sum()  # noqa: E731
    want = _forward_over_reverse(loss(_plain("silu")), [i["x"]], [i["tx"]])
    with fwAD.dual_level():
        got = fwAD.unpack_dual(torch.func.grad(loss(gated_linear))(fwAD.make_dual(i["x"], i["tx"])))
        for a, (b,) in zip(got, want):
            torch.testing.assert_close(a, b)


def test_its_tangent_cannot_be_differentiated_a_third_time():
    i = _inputs(9)
    hvp = lambda x: torch.func.jvp(torch.func.grad(lambda v: (gated_linear(v, i["wg"], i["wu"]) ** 2).sum()), (x,), (i["tx"],))[1].sum()  # noqa: E731
    with pytest.raises(RuntimeError, match="third time"):
        torch.func.grad(hvp)(i["x"])


def test_transforms_that_are_refused():
    i = _inputs(13)
    f = lambda x: gated_linear(x, i["wg"], i["wu"])  # noqa: E731
    along = lambda x: torch.func.jvp(f, (x,), (i["tx"],))[1]  # noqa: E731
    with pytest.raises(RuntimeError, match="by a further forward transform"):
        torch.func.jvp(along, (i["x"],), (i["tx"],))
    grad = torch.func.grad(lambda x: (f(x) ** 2).sum())
    with pytest.raises(RuntimeError, match="by a further forward transform|third time"):
        torch.func.jvp(lambda x: torch.func.jvp(grad, (x,), (i["tx"],))[1], (i["x"],), (i["tx"],))
    for call in (lambda: torch.func.vmap(f)(i["x"]), lambda: torch.func.vmap(grad)(i["x"]), lambda: torch.func.jacfwd(f)(i["x"]),
                 lambda: torch.func.jacrev(f)(i["x"]), lambda: torch.func.hessian(lambda x: f(x).sum())(i["x"]),
                 lambda: torch.func.vmap(lambda w: gated_linear(i["x"], w, i["wu"]))(torch.stack((i["wg"], i["wu"])))):
        with pytest.raises(NotImplementedError, match="gated_linear has no rule for torch.func.vmap"):
            call()
    x = i["x"].requires_grad_()
    h = f(x)
    with pytest.raises(NotImplementedError, match="gated_linear has no rule for torch.func.vmap"):  # an ordinary graph
        torch.func.vmap(lambda c: torch.autograd.grad(h, x, c, retain_graph=True)[0])(torch.stack((i["gh"], i["tgh"])))
    with pytest.raises(NotImplementedError, match="gated_linear has no rule for .*is_grads_batched"):
        torch.autograd.grad(h, x, torch.stack((i["gh"], i["tgh"])), is_grads_batched=True)


@pytest.mark.parametrize("linear", [False, True])
def test_a_third_derivative_under_torch_func_is_refused(linear):
    """Whichever way it is taken: not even the part of it that other operators make comes out alone."""
    i = _inputs(14)
    loss = lambda f: lambda v: (f(v, i["wg"], i["wu"]) * i["gh"]).sum() if linear else (f(v, i["wg"], i["wu"]) ** 2).sum()  # noqa: E731
    along = lambda f: lambda x: (f(x) * i["tx"]).sum()  # noqa: E731
    twice = lambda f: torch.func.grad(along(torch.func.grad(loss(f))))  # noqa: E731
    torch.testing.assert_close(twice(gated_linear)(i["x"]), twice(_plain("silu"))(i["x"]))
    for third in (lambda: torch.func.grad(along(twice(gated_linear)))(i["x"]), lambda: torch.func.jvp(twice(gated_linear), (i["x"],), (i["tx"],))):
        with pytest.raises(RuntimeError, match="third time"):
            third()
    # linear in the vector of a second derivative
    pulled = [torch.func.vjp(torch.func.grad(loss(f)), i["x"])[1] for f in (gated_linear, _plain("silu"))]
    for a, b in zip(*(torch.func.jvp(lambda v: p(v)[0], (i["tx"],), (i["x"],)) for p in pulled)):
        torch.testing.assert_close(a, b)
    with fwAD.dual_level():
        d, t = fwAD.unpack_dual(twice(gated_linear)(fwAD.make_dual(i["x"], i["tx"])))
        torch.testing.assert_close(d, twice(_plain("silu"))(i["x"]))
        assert t.isnan().all()


def test_reverse_over_forward_under_torch_func():
    i = _inputs(15)
    for loss in (lambda h: (h * i["gh"]).sum(), lambda h: (h**2).sum()):
        got, want = (torch.func.grad(lambda x: torch.func.jvp(lambda v: loss(f(v, i["wg"], i["wu"])), (x,), (i["tx"],))[1])(i["x"])
                     for f in (gated_linear, _plain("silu")))
        torch.testing.assert_close(got, want)
