"""GPU tests of gated_linear's gradients where forward mode goes over them, inside a forward-AD level and under functorch transforms.
Bounds as in test_gpu_gated.py: the launches are the same, with other cotangents."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from jvp_flash_attention_b200 import _lib
from jvp_flash_attention_b200.gated import ACTIVATIONS, gated_linear
from tests import _block_formulas as formulas
from tests.test_gpu_gated import _check, _inputs, _run

pytestmark = pytest.mark.gpu


def _plain(name):
    return lambda x, wg, wu: formulas.activation(ACTIVATIONS[name], x @ wg.T)[0] * (x @ wu.T)


@pytest.mark.parametrize("name", list(ACTIVATIONS))
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("M,K,F", [(90, 72, 136), (400, 128, 130)])
def test_gradients_inside_a_level_carry_their_tangents(name, dt, M, K, F):
    """By the symmetry of second derivatives the tangents are the gradients of <tgh, h> + <gh, th>."""
    x, tx, wg, wu, gh, tgh = _inputs(M, K, F, dt, 31)
    leaves = [t.requires_grad_() for t in (x, wg, wu)]
    with fwAD.dual_level():
        h = gated_linear(fwAD.make_dual(x, tx), wg, wu, name)
        pairs = [fwAD.unpack_dual(d) for d in torch.autograd.grad(h, leaves, fwAD.make_dual(gh, tgh))]
        first, second = (dict(zip(("dx", "dwg", "dwu"), ts)) for ts in zip(*pairs))
    _check({k: v.detach() for k, v in first.items()}, x, None, wg, wu, gh, None, ACTIVATIONS[name])
    _check({k: v.detach() for k, v in second.items()}, x, tx, wg, wu, tgh, gh, ACTIVATIONS[name])
    assert _lib.device_status() == 0


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("M", [90, 400])
def test_and_those_of_the_weights(dt, M):
    """Against torch in float64.  An entry of x's is the rounded sum of two that are rounded: two gradients' bounds of the norm."""
    x, tx, wg, wu, gh, tgh = _inputs(M, 72, 136, dt, 32)
    tg, tu = (torch.randn(w.shape, generator=torch.Generator(device=w.device).manual_seed(7), device=w.device).to(w.dtype) * 0.3 * 72**-0.5
              for w in (wg, wu))
    leaves = [t.requires_grad_() for t in (x, wg, wu)]
    with fwAD.dual_level():
        h = gated_linear(*(fwAD.make_dual(p, t) for p, t in zip(leaves, (tx, tg, tu))))
        pairs = [fwAD.unpack_dual(d) for d in torch.autograd.grad(h, leaves, fwAD.make_dual(gh, tgh))]
        got = [t.detach() for p in zip(*pairs) for t in p]
    gradient = lambda x, wg, wu, c: torch.func.vjp(_plain("silu"), x, wg, wu)[1](c)  # noqa: E731
    want = torch.func.jvp(gradient, tuple(t.detach().double() for t in (x, wg, wu, gh)), tuple(t.double() for t in (tx, tg, tu, tgh)))
    most = 2e-5 if dt == "fp32" else 8 * 2.0**-8
    for a, b in zip(got, [t for p in want for t in p]):
        assert (a.double() - b).norm() <= most * b.norm()


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_torch_func_jvp_of_a_vjp(dt):
    """Forward over reverse under functorch, x and the weights moving, and the cotangent alone."""
    x, tx, wg, wu, gh, tgh = _inputs(150, 72, 136, dt, 33)
    gradient = lambda x, c: torch.func.vjp(lambda v: gated_linear(v, wg, wu), x)[1](c)[0]  # noqa: E731
    dx, tdx = torch.func.jvp(gradient, (x, gh), (tx, tgh))
    _check({"dx": dx}, x, None, wg, wu, gh, None, 0)
    _check({"dx": tdx}, x, tx, wg, wu, tgh, gh, 0)
    _, tdx = torch.func.jvp(lambda c: gradient(x, c), (gh,), (tgh,))
    _check({"dx": tdx}, x, None, wg, wu, tgh, None, 0)
    moving = lambda f: torch.func.jvp(lambda w, c: torch.func.vjp(lambda v: f(x.to(w.dtype), v, wu.to(w.dtype)), w)[1](c)[0],  # noqa: E731
                                      *(tuple(t if f is gated_linear else t.double() for t in ts) for ts in ((wg, gh), (wu, tgh))))
    for a, b in zip(moving(gated_linear), moving(_plain("silu"))):
        assert (a.double() - b).norm() <= (2e-5 if dt == "fp32" else 8 * 2.0**-8) * b.norm()


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_cotangents_that_begin_between_16_byte_pieces(dt):
    """Of a loss that concatenates something in front of h, where rows of F = 37 end anywhere: torch.func.grad, and a second derivative through
    the weights, which reads the first one's cotangent."""
    x, _, wg, wu, gh, _ = _inputs(21, 72, 37, dt, 34)
    front = torch.randn(3, 37, device=x.device).to(x.dtype)
    c = torch.cat((front, gh)) * 2
    behind = lambda f: lambda v, w: torch.cat((front.to(v.dtype), f(v, w, wu.to(v.dtype))))  # noqa: E731
    got = torch.func.grad(lambda v, w: (behind(gated_linear)(v, w) * c).sum(), argnums=(0, 1))(x, wg)
    _check(dict(zip(("dx", "dwg"), got)), x, None, wg, wu, c[3:], None, 0)
    second = []
    for f in (gated_linear, _plain("silu")):
        leaves = [(t if f is gated_linear else t.double()).detach().requires_grad_() for t in (x, wg)]
        (dw,) = torch.autograd.grad(behind(f)(*leaves), leaves[1], c.to(leaves[0].dtype), create_graph=True)
        second.append(torch.autograd.grad(dw, leaves, wu.to(dw.dtype)))
    for a, b in zip(*second):
        assert (a.double() - b).norm() <= (2e-5 if dt == "fp32" else 8 * 2.0**-8) * b.norm()


@pytest.mark.parametrize("name", list(ACTIVATIONS))
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("M", [10, 200])
def test_second_derivatives_of_far_gates(name, dt, M):
    """Gates of 40.7 to 1e36 to either side, with u = 1, tg = 1, tu = 0 and gth = 1: the cotangents are dg = a'', du = dtg = a', dtu = a, whose sums over 64
    features or M rows are finite (the largest, in dwu, below 2 M 1e36), and a'' and a' have their limits, 0 and 0 or 1.

    They are off by no more than (2 + |g|) exp(-|g|), which falls: 42.7 exp(-40.7) = 9.1e-17 < 2^-53 for a' and a'', and with the factor |g| that dwg
    has from x, 3.7e-15 < 2^-47.  Next to 1 that is nothing; beside 0 the sums are off by 64 or M of it."""
    K, F = 8, 64
    x, _, wg, wu, _, gth = _inputs(M, K, F, dt, 35)
    far = 10.0 ** torch.linspace(1.61, 36, M // 2, device=x.device)
    with torch.no_grad():
        for t in (x, wg, wu):
            t.zero_()
        x[:, 0], x[:, 1], wg[:, 0], wu[:, 1] = torch.cat((far, -far)).to(x.dtype), 1, 1, 1
        tx = torch.zeros_like(x)
        tx[:, 0] = 1
    got = _run(x, tx, wg, wu, None, torch.ones_like(gth), name, "jvp_bwd_t")
    _check(got, x, tx, wg, wu, None, torch.ones_like(gth), ACTIVATIONS[name])
    up = (x[:, 0] > 0).to(x.dtype) * (name != "sigmoid")
    near = lambda y, limit, off: torch.testing.assert_close(y, limit, rtol=0, atol=off)  # noqa: E731
    near(got["th"], up[:, None].expand(M, F), 2.0**-53)
    near(got["dx"][:, 0], torch.zeros_like(up), 64 * 2.0**-53)
    near(got["dx"][:, 1], 64 * up, 64 * 2.0**-53)
    near(got["dtx"][:, 0], 64 * up, 64 * 2.0**-53)
    near(got["dwg"][:, 0], up.sum().expand(F), M * 2.0**-47)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_nested_reverse_transforms(dt):
    """torch.func.grad of torch.func.grad, against torch in float64: two gradients' bounds of the norm.  A third derivative is refused."""
    x, tx, wg, wu, gh, _ = _inputs(140, 72, 136, dt, 36)

    def hvp(f, x, tx, wg, wu, gh):
        first = torch.func.grad(lambda v: (f(v, wg, wu) * gh).sum())
        return torch.func.grad(lambda v: (first(v) * tx).sum())(x)

    want = hvp(_plain("silu"), *(t.double() for t in (x, tx, wg, wu, gh)))
    got = hvp(gated_linear, x, tx, wg, wu, gh)
    assert (got.double() - want).norm() <= (2e-5 if dt == "fp32" else 8 * 2.0**-8) * want.norm()
    with pytest.raises(RuntimeError, match="third time"):
        torch.func.grad(lambda v: (hvp(gated_linear, v, tx, wg, wu, gh) * tx).sum())(x)
