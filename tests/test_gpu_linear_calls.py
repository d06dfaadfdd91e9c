"""GPU tests of calls of linear attention besides whole training steps."""
import pytest
import torch

import jvp_flash_attention_b200.linear_attention as la
from tests import _linear_formulas as formulas
from tests.test_gpu_linear_attention import DEV, _bits, _near

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
