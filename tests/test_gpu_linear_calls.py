"""GPU tests of calls of linear attention besides whole training steps."""
import pytest
import torch

import jvp_flash_attention_b200.linear_attention as la
from tests import _linear_formulas as formulas
from tests.test_gpu_linear_attention import DEV, DT, _bits, _near

pytestmark = pytest.mark.gpu


def test_a_module_decodes_with_the_decay_it_learns():
    w = torch.nn.Parameter(torch.tensor([-0.1, -0.5], device=DEV))
    q, s = torch.randn(1, 2, 9, 16, device=DEV), torch.randn(1, 2, 16, 16, device=DEV)
    want = la.linear_attention(q, q, q, w.detach(), state=s, return_state=True)
    with torch.no_grad():
        got = la.linear_attention(q, q, q, w, state=s, return_state=True)
        step, other = s.clone(), s.clone()
        o = la.linear_attention_step(q[:, :, 0], q[:, :, 0], q[:, :, 0], w, step)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(o, la.linear_attention_step(q[:, :, 0], q[:, :, 0], q[:, :, 0], w.detach(), other)) and torch.equal(step, other)
    for call in (lambda: la.linear_attention(q, q, q, w), lambda: la.linear_attention_step(q[:, :, 0], q[:, :, 0], q[:, :, 0], w, other)):
        with pytest.raises(NotImplementedError, match="log_decay"):
            call()


def test_operands_without_dimensions_are_refused_as_such():
    x = torch.ones((), device=DEV)
    with pytest.raises(ValueError, match="shapes"):
        la.linear_attention(x, x, x)
    with pytest.raises(ValueError, match="shapes"):
        la.linear_attention_step(x, x, x, None, x)


@pytest.mark.parametrize("scale", [2.0**-64, -(2.0**-40), 2.0**64])
def test_scales_at_the_ends_of_their_range(scale):
    """With a cotangent of the last state, whose part of dk and dv the scale does not go with."""
    g = torch.Generator(device=DEV).manual_seed(1)
    x = [torch.randn(1, 2, 150, 32, generator=g, device=DEV).requires_grad_() for _ in range(3)]
    w = torch.tensor([-0.01, -0.2], device=DEV)
    go, gs = torch.randn(1, 2, 150, 32, generator=g, device=DEV), torch.randn(1, 2, 32, 32, generator=g, device=DEV)
    o, s = la.linear_attention(*x, w, sm_scale=scale, return_state=True)
    grads = torch.autograd.grad((o, s), x, (go / scale, gs))
    want, _, _ = formulas.launch_fwd([*x, None], [None] * 4, (w, None), (scale, True, ""), False)
    dwant = formulas.launch_bwd([*x, None], [None] * 4, (w, None), None, [go / scale, gs], [None, None], (scale, True, ""), [True] * 8)
    mag = [t.detach().abs() for t in x]
    dsize = formulas.launch_bwd([*mag, None], [None] * 4, (w, None), None, [go.abs() / abs(scale), gs.abs()], [None, None], (abs(scale), True, ""), [True] * 8)
    size, _, _ = formulas.launch_fwd([*mag, None], [None] * 4, (w, None), (abs(scale), True, ""), False)
    _near(o.detach(), want[0], size[0], _bits(150, 32), "o")
    for d, e, f in zip(grads, dwant, dsize):
        _near(d, e, f, _bits(150, 32))


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("L,lengths", [(40, None), (1400, (1400, 515))])
def test_tangents_without_their_gradient(L, lengths, dt):
    """A call with tangents whose gradient is taken through the values alone, or through the tangents alone: the states that the forward kept are those
    of a call with tangents."""
    B, H, D, E = 2, 2, 64, 32
    g = torch.Generator(device=DEV).manual_seed(L)
    make = lambda std: [(torch.randn(*s, generator=g, device=DEV) * std).to(DT[dt] if i < 3 else torch.float32).requires_grad_()  # noqa: E731
                        for i, s in enumerate([(B, H, L, D), (B, H, L, D), (B, H, L, E), (B, H, D, E)])]
    x, tx = make(1.0), make(0.3)
    w = torch.tensor([-0.001, -0.1], device=DEV)
    n = None if lengths is None else torch.tensor(lengths, device=DEV, dtype=torch.int32)
    cots = [torch.randn(B, H, L, E, generator=g, device=DEV).to(DT[dt]), torch.randn(B, H, D, E, generator=g, device=DEV)]
    mag = lambda ts: [None if t is None else t.detach().abs() for t in ts]  # noqa: E731
    bits = _bits(L, D)
    outs = bits if dt == "fp32" else bits + 2.0**-11
    for through in (0, 1):
        y, ty = torch.func.jvp(lambda *a: la.linear_attention(*a[:3], w, sm_scale=0.3, state=a[3], lengths=n, return_state=True), tuple(x), tuple(tx))
        grads = torch.autograd.grad(ty if through else y, (*x, *tx), cots, materialize_grads=True)
        pair = ([None, None], cots) if through else (cots, [None, None])
        args = ((w, n), None, *pair, (0.3, True, ""), [True] * 8)
        want = formulas.launch_bwd(x, tx, *args)
        size = formulas.launch_bwd(mag(x), mag(tx), (w, n), None, *map(mag, pair), (0.3, True, ""), [True] * 8)
        for i, (d, e, f) in enumerate(zip(grads, want, size)):
            _near(d, e, f, bits if i % 4 == 3 else outs, (through, i))
