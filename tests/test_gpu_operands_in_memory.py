"""GPU tests of operands without memory: zeros that torch keeps as a shape alone."""
import pytest
import torch

import jvp_flash_attention_b200.rotary as rot
from jvp_flash_attention_b200.gated import gated_linear

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_zero_tangents_and_cotangents_under_nested_transforms():
    x, wg, wu = torch.randn(20, 16, device=DEV), torch.randn(24, 16, device=DEV), torch.randn(24, 16, device=DEV)
    zero = lambda *s: torch._efficientzerotensor(s, device=DEV)  # noqa: E731
    h, th = torch.func.jvp(lambda a: torch.func.vjp(lambda b: gated_linear(b, wg, wu), a)[0], (x,), (zero(20, 16),))
    assert torch.equal(h, gated_linear(x, wg, wu)) and not th.any()
    x.requires_grad_()
    (dx,) = torch.autograd.grad(gated_linear(x, wg, wu), x, zero(20, 24))
    assert dx.shape == x.shape and not dx.any()
    q, w = torch.randn(1, 2, 3, 8, device=DEV), rot.rotary_frequencies(8, device=DEV)
    y, ty = torch.func.jvp(lambda a: torch.func.vjp(lambda b: rot.rotary(b, None, w), a)[0], (q,), (zero(1, 2, 3, 8),))
    assert torch.equal(y, rot.rotary(q, None, w)) and not ty.any()


def test_batched_cotangents_are_refused():
    x, wg, wu = (torch.randn(s, 16, device=DEV) for s in (20, 24, 24))
    h = gated_linear(x.requires_grad_(), wg, wu)
    with pytest.raises(NotImplementedError, match="no rule for"):
        torch.autograd.grad(h, x, torch.randn(3, 20, 24, device=DEV), is_grads_batched=True, retain_graph=True)
    with pytest.raises(NotImplementedError, match="no rule for"):
        torch.func.vmap(lambda c: torch.autograd.grad(h, x, c, retain_graph=True)[0])(torch.randn(3, 20, 24, device=DEV))
