"""CPU tests of what rotary's and gated_linear's general route hands to the launches: the addresses of memory that holds the operands."""
import ctypes

import pytest
import torch

import jvp_flash_attention_b200.gated as gated
import jvp_flash_attention_b200.rotary as rot
from jvp_flash_attention_b200 import _lib


def _read(address, n):
    return list((ctypes.c_float * n).from_address(address)) if address else None


def _zero(*shape):
    return torch._efficientzerotensor(shape)


@pytest.fixture()
def launched(monkeypatch):
    """The operands that an entry would read, by name."""
    seen = {}

    def run(a, x, entry):
        n = {"x": a.K, "tx": a.K, "wg": a.K, "wu": a.K, "gh": a.M * a.F, "gth": a.M * a.F}
        seen.update({k: _read(getattr(a, k), n[k]) for k in n if hasattr(a, k)})

    monkeypatch.setattr(gated, "_run", run)
    monkeypatch.setattr(_lib, "_launch", lambda x, entry, a: seen.update(x=_read(a.t[0].x, a.D)) or 0)
    return seen


def test_zeros_without_memory(launched):
    x, w = torch.ones(2, 8), torch.ones(4, 8)
    gated._launch_fwd(x, _zero(2, 8), w, w, 0, False)
    assert launched["tx"] == [0.0] * 8
    gated._launch_bwd(x, None, w, w, torch.zeros(1), _zero(2, 4), None, 0, True, False, True)
    assert launched["gh"] == [0.0] * 8 and launched["gth"] is None
    rot._launch(_zero(1, 1, 1, 8), rot.rotary_frequencies(8), None, 0, False, 1.0, False)
    assert launched["x"] == [0.0] * 8


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("offset", [0, 1, 2, 3, 5, 8])
def test_cotangents_begin_on_a_16_byte_boundary(monkeypatch, dtype, offset):
    """The gradient of torch.cat is a slice of the cotangent, contiguous at any offset; the entry refuses one that 16 bytes do not divide."""
    seen = {}
    monkeypatch.setattr(gated, "_run", lambda a, x, entry: seen.update(gh=a.gh, gth=a.gth, rows=bytes((ctypes.c_char * x.element_size()).from_address(a.gh))))
    x, w = torch.ones(2, 8, dtype=dtype), torch.ones(3, 8, dtype=dtype)
    c = torch.arange(6.0 + offset).to(dtype)[offset:].view(2, 3)
    gated._launch_bwd(x, x, w, w, torch.zeros(1), c, c, 0, True, True, True)
    assert seen["gh"] % 16 == 0 and seen["gth"] % 16 == 0
    assert seen["rows"] == c.flatten()[:1].view(torch.uint8).numpy().tobytes()
