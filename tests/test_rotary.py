"""CPU tests of rotary: frequencies, graph, tangents and refusals.  Launches go to the formula (tests/_block_formulas.py)."""
import ctypes
import math

import pytest
import torch
import torch.autograd.forward_ad as fwAD

import jvp_flash_attention_b200.rotary as rot
from jvp_flash_attention_b200 import _lib
from tests import _block_formulas as formulas

B, H, HK, L, D = 2, 3, 1, 5, 8
W = rot.rotary_frequencies(6)


@pytest.fixture()
def cpu_turn(monkeypatch):
    calls = []

    def launch(x, *args):
        calls.append(tuple(x.shape))
        return formulas.turn(x, *args)

    monkeypatch.setattr(rot, "_launch", launch)
    monkeypatch.setattr(rot, "_require_cuda", lambda *a: None)
    return calls


def _qk(seed, n=2):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(B, h, L, D, generator=g, dtype=torch.float64) for h in (H, HK) * (n // 2)]


@pytest.mark.parametrize("route", ["func", "fwad"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_values_tangents_and_gradients(cpu_turn, route, interleaved):
    q, k, tq, tk, gq, gk, gtq, gtk = _qk(1, 8)
    leaves = [x.requires_grad_() for x in (q, k, tq, tk)]
    pos = torch.tensor([[3, -1, 7, 0, 100000], [1, 2, 3, 4, 5]])
    f = lambda a, b: rot.rotary(a, b, W, pos, interleaved=interleaved, amplitude=1.5)  # noqa: E731
    if route == "func":
        (yq, yk), (zq, zk) = torch.func.jvp(f, (q, k), (tq, tk))
    else:
        with fwAD.dual_level():
            (yq, zq), (yk, zk) = (fwAD.unpack_dual(o) for o in f(fwAD.make_dual(q, tq), fwAD.make_dual(k, tk)))
    grads = torch.autograd.grad((yq, yk, zq, zk), leaves, (gq, gk, gtq, gtk))
    for y, x in zip((yq, yk, zq, zk), leaves):
        torch.testing.assert_close(y, formulas.turn(x, W, pos, 0, interleaved, 1.5))
    for d, g in zip(grads, (gq, gk, gtq, gtk)):
        torch.testing.assert_close(d, formulas.turn(g, W, pos, 0, interleaved, 1.5, True))


def test_gradients_against_differences(cpu_turn):
    q, k = _qk(2)
    torch.autograd.gradcheck(lambda a, b: rot.rotary(a, b, W, offset=9), (q.requires_grad_(), k.requires_grad_()))
    torch.autograd.gradgradcheck(lambda a, b: rot.rotary(a, b, W, offset=9), (q, k))


def test_only_what_is_asked_for_is_turned_back(cpu_turn):
    q, k = _qk(3)
    yq, yk = rot.rotary(q.requires_grad_(), k, W)
    assert yq.requires_grad and not yk.requires_grad
    cpu_turn.clear()
    torch.autograd.grad(yq.sum(), q)
    assert cpu_turn == [(B, H, L, D)]


def test_a_tangent_of_one_alone(cpu_turn):
    q, k, tq, _ = _qk(4, 4)
    with fwAD.dual_level():
        yq, yk = rot.rotary(fwAD.make_dual(q, tq), k, W)
        assert fwAD.unpack_dual(yk).tangent is None
        torch.testing.assert_close(fwAD.unpack_dual(yq).tangent, formulas.turn(tq, W))
    y, t = torch.func.jvp(lambda a: rot.rotary(a, None, W), (q,), (tq,))
    torch.testing.assert_close(t, formulas.turn(tq, W))


def test_nested_transforms_take_the_general_route(cpu_turn):
    q, k, tq, gq = _qk(5, 4)[0], None, _qk(6)[0], _qk(7)[0]
    g = torch.func.grad(lambda x: (rot.rotary(x, k, W) * gq).sum())(q)
    torch.testing.assert_close(g, formulas.turn(gq, W, transposed=True))
    _, t = torch.func.jvp(torch.func.grad(lambda x: (rot.rotary(x, k, W) ** 3).sum()), (q,), (tq,))
    y, ty = formulas.turn(q, W), formulas.turn(tq, W)
    torch.testing.assert_close(t, formulas.turn(6 * y * ty, W, transposed=True))


def test_a_functorch_transform_of_the_cotangent(cpu_turn):
    """A graph built outside the transform: the gradient is linear in its cotangent."""
    q, k = _qk(11)
    g, v, u = _qk(12)[0], _qk(13)[0], _qk(14)[1]
    yq, yk = rot.rotary(q.requires_grad_(), k.requires_grad_(), W)
    vjp = lambda c: torch.autograd.grad((yq, yk), q, (c, u), retain_graph=True, create_graph=True)[0]  # noqa: E731
    torch.testing.assert_close(torch.func.grad(lambda c: (vjp(c) * v).sum())(g), formulas.turn(v, W))


def test_the_gradient_of_a_dual_cotangent_is_dual(cpu_turn):
    """Forward over reverse inside a forward-AD level; the gradient and its tangent can be differentiated in turn."""
    q, k, tq, tk = _qk(15, 4)
    v = _qk(16)[0]
    leaves = [x.requires_grad_() for x in (q, k, tq, tk)]
    out = []
    for f in (lambda a, b: rot.rotary(a, b, W, offset=3), lambda a, b: (formulas.turn(a, W, None, 3), formulas.turn(b, W, None, 3))):
        with fwAD.dual_level():
            yq, yk = f(fwAD.make_dual(q, tq), fwAD.make_dual(k, tk))
            (g,) = torch.autograd.grad((yq**3).sum() + (yk**2).sum(), q, create_graph=True)
            g, tg = fwAD.unpack_dual(g)
            out.append((g, tg, *torch.autograd.grad((g * v).sum() + (tg * v).sum(), (q, tq))))
    for a, b in zip(*out):
        torch.testing.assert_close(a, b)


def test_nothing_to_turn(cpu_turn):
    assert rot.rotary(_qk(8)[0], None, W[:0]).shape == (B, H, L, D)


@pytest.mark.parametrize("rd", [2, 32, 64, 128])
def test_frequencies(rd):
    w = rot.rotary_frequencies(rd)
    assert w.dtype == torch.float64 and w[0] == 1.0
    for i in range(rd // 2):
        assert math.isclose(w[i], 10000.0 ** (-2 * i / rd), rel_tol=1e-14)
    torch.testing.assert_close(rot.rotary_frequencies(rd, scaling="linear", factor=4.0), w / 4)
    if rd > 2:
        based = rot.rotary_frequencies(rd, scaling="base", factor=4.0)
        assert based[0] == 1.0 and math.isclose(based[-1], w[-1] / 4, rel_tol=1e-12)
    for kind in ("ramp", "bands"):
        s = rot.rotary_frequencies(rd, scaling=kind, factor=4.0, original_length=4096)
        turns = 4096 * w / (2 * math.pi)
        assert ((s <= w * (1 + 1e-15)) & (s >= w / 4 * (1 - 1e-15))).all() and (s[:-1] >= s[1:]).all()
        assert (s[turns < 0.5] == w[turns < 0.5] / 4).all() and (s[turns > 100] == w[turns > 100]).all()
    turns = 4096 * w / (2 * math.pi)
    keep = ((turns - 1) / 31).clamp(0, 1)
    torch.testing.assert_close(s, w * keep + w / 4 * (1 - keep))


@pytest.mark.parametrize("bad", [dict(rotary_dim=3), dict(rotary_dim=-2), dict(rotary_dim=8, base=0.0), dict(rotary_dim=8, factor=-1.0),
                                 dict(rotary_dim=8, scaling="other"), dict(rotary_dim=8, scaling="ramp", quick=1.0, slow=2.0),
                                 dict(rotary_dim=8, scaling="ramp", base=1.0)])
def test_frequencies_that_are_refused(bad):
    with pytest.raises(ValueError):
        rot.rotary_frequencies(**bad)


def test_refusals(cpu_turn):
    q, k = _qk(9)
    cases = [
        (ValueError, (q[0], k, W)), (ValueError, (q, k[:, :, :4], W)), (TypeError, (q, k.float(), W)), (TypeError, (q, k, W.float())),
        (TypeError, (q, k, W[None])), (ValueError, (q, k, rot.rotary_frequencies(10))), (ValueError, (q, k, W.repeat_interleave(2)[::2])),
        (NotImplementedError, (q, k, W.clone().requires_grad_())), (TypeError, (q, k, W, torch.zeros(L))),
        (ValueError, (q, k, W, torch.zeros(L + 1, dtype=torch.int64))), (ValueError, (q, k, W, torch.zeros(3, L, dtype=torch.int64))),
        (ValueError, (q, k, W, torch.zeros(B, 1, dtype=torch.int64))),
    ]
    for error, args in cases:
        with pytest.raises(error):
            rot.rotary(*args)


def test_no_cpu_fallback():
    q, k = (x.float() for x in _qk(10))
    with pytest.raises(RuntimeError, match="runs only on CUDA tensors"):
        rot.rotary(q, k, W)


def test_the_c_entry_refuses():
    lib = _lib.load()

    def call(**kw):
        a = _lib.RotaryArgs()
        a.struct_size = ctypes.sizeof(a)
        a.B = a.L = 1
        a.D, a.n_freq, a.n_tensors, a.freq, a.position_bits = 8, 4, 1, 64, 64
        for i in range(4):
            a.t[i].x, a.t[i].y, a.t[i].H = 64, 64, 1
        for key, v in kw.items():
            if key in ("x", "y", "H"):
                setattr(a.t[0], key, v)
            elif key == "stride":
                a.t[0].x_stride[0] = v
            else:
                setattr(a, key, v)
        return lib.jvpfa_rotary(ctypes.byref(a), None)

    assert lib.jvpfa_rotary(None, None) == -1
    for want, kw in [(-7, dict(struct_size=8)), (-3, dict(dtype=3)), (-3, dict(dtype=-1)), (-2, dict(B=0)), (-2, dict(L=0)), (-2, dict(D=0)),
                     (-2, dict(n_freq=5)), (-2, dict(n_freq=-1)), (-2, dict(n_tensors=0)), (-2, dict(n_tensors=5)), (-1, dict(freq=None)),
                     (-3, dict(positions=64, position_bits=16)), (-1, dict(x=None)), (-1, dict(y=None)), (-2, dict(H=0)),
                     (-8, dict(x=65)), (-8, dict(dtype=2, y=66)), (-2, dict(stride=-8))]:
        assert call(**kw) == want, kw
