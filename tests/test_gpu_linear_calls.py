"""GPU tests of calls of linear attention besides whole training steps."""
import pytest
import torch

import jvp_flash_attention_b200.linear_attention as la
from tests.test_gpu_linear_attention import DEV

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
