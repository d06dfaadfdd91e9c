"""CPU tests of linear attention: graph, tangents, levels and refusals.  Launches go to the formulas (tests/_linear_formulas.py), which are held
against the recurrence."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwAD

import jvp_flash_attention_b200.linear_attention as la
from jvp_flash_attention_b200 import _lib
from tests import _linear_formulas as formulas

B, H, L, D, E = 2, 3, 5, 4, 3
DECAY = torch.tensor([0.0, -0.3, -2.0])
LENGTHS = torch.tensor([5, 3], dtype=torch.int32)


@pytest.fixture()
def cpu(monkeypatch):
    calls = []

    def forward(x, tx, *args):
        calls.append("dual" if any(t is not None for t in tx) else "value")
        return formulas.launch_fwd(x, tx, *args)

    monkeypatch.setattr(la, "_launch_fwd", forward)
    monkeypatch.setattr(la, "_launch_bwd", formulas.launch_bwd)
    monkeypatch.setattr(la, "_require_cuda", lambda *a: None)
    return calls


def _operands(seed, std=1.0, grad=False):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g, dtype=torch.float64) * std).requires_grad_(grad) for s in ((B, H, L, D), (B, H, L, D), (B, H, L, E), (B, H, D, E))]


def _own(q, k, v, s):
    return la.linear_attention(q, k, v, DECAY, state=s, lengths=LENGTHS, return_state=True)


def _recurrence(q, k, v, s):
    """Row by row."""
    decay, out = torch.exp(DECAY.double())[None, :, None, None], []
    for t in range(L):
        live = (t < LENGTHS)[:, None, None, None]
        s = torch.where(live, decay * s + k[:, :, t, :, None] * v[:, :, t, None, :], s)
        out.append(torch.where(live[..., 0], (q[:, :, t, None, :] @ s)[..., 0, :] * D**-0.5, 0.0))
    return torch.stack(out, 2), s


def _close(a, b):
    for s, t in zip(a, b, strict=True):
        torch.testing.assert_close(s, t)


@pytest.mark.parametrize("route", ["func", "fwad"])
def test_values_tangents_and_gradients(cpu, route):
    x, tx, cots = _operands(1, grad=True), _operands(2, 0.3, True), [_operands(3)[i] for i in (2, 3)] + [_operands(4)[i] for i in (2, 3)]
    results = []
    for f in (_own, _recurrence):
        cpu.clear()
        if route == "func" or f is _recurrence:
            y, ty = torch.func.jvp(f, tuple(x), tuple(tx))
        else:
            with fwAD.dual_level():
                y, ty = zip(*(fwAD.unpack_dual(o) for o in f(*map(fwAD.make_dual, x, tx))))
        assert f is _recurrence or cpu == ["dual"]
        results.append((*y, *ty, *torch.autograd.grad((*y, *ty), (*x, *tx), cots)))
    _close(*results)


def test_without_a_state(cpu):
    q, k, v, _ = _operands(5, grad=True)
    f = lambda *a: la.linear_attention(*a, DECAY)  # noqa: E731
    torch.autograd.gradcheck(f, (q, k, v), check_forward_ad=True)
    torch.autograd.gradgradcheck(f, (q, k, v))
    o, s = la.linear_attention(q, k, v, return_state=True)
    torch.testing.assert_close(o, ((q @ k.transpose(-1, -2)).tril() @ v) * D**-0.5)
    torch.testing.assert_close(s, k.transpose(-1, -2) @ v)
    (dq,) = torch.autograd.grad(s.sum(), q, allow_unused=True, materialize_grads=True)
    assert not dq.any()


def test_sequences_in_pieces_and_token_by_token(cpu):
    q, k, v, s = _operands(6)
    o, last = la.linear_attention(q, k, v, DECAY, state=s, return_state=True)
    a, s1 = la.linear_attention(q[:, :, :2], k[:, :, :2], v[:, :, :2], DECAY, state=s, return_state=True)
    b, s2 = la.linear_attention(q[:, :, 2:], k[:, :, 2:], v[:, :, 2:], DECAY, state=s1, return_state=True)
    torch.testing.assert_close(torch.cat((a, b), 2), o)
    torch.testing.assert_close(s2, last)


def test_nested_transforms(cpu):
    x, v = [t.detach() for t in _operands(7)], [t.detach() for t in _operands(8)]
    results = []
    for f in (_own, _recurrence):
        loss = lambda *a: sum((o**3).sum() for o in f(*a))  # noqa: B023, E731
        grad = torch.func.grad(loss, argnums=(0, 1, 2, 3))
        g, hv = torch.func.jvp(grad, tuple(x), tuple(v))
        rr = torch.func.grad(lambda *a: sum((s * t).sum() for s, t in zip(grad(*a), v)), argnums=(0, 1, 2, 3))(*x)
        results.append((*g, *hv, *rr, *torch.func.vjp(f, *x)[1](tuple(f(*x)))))
    _close(*results)


def test_gradients_inside_a_level_are_dual(cpu):
    x, tx = _operands(9, grad=True), [t.detach() for t in _operands(10)]
    results = []
    for f in (_own, _recurrence):
        with fwAD.dual_level():
            out = f(*map(fwAD.make_dual, x, tx))
            results.append([t for d in torch.autograd.grad(sum((o**2).sum() for o in out), x) for t in fwAD.unpack_dual(d)])
    _close(*results)


def test_what_is_refused(cpu):
    x = _operands(11, grad=True)
    plain = [t.detach() for t in x]
    o, s = _own(*x)
    d = torch.autograd.grad((o**2).sum(), x[0], create_graph=True)[0]
    d2 = torch.autograd.grad((d**2).sum(), x[0], create_graph=True)[0]
    with pytest.raises(RuntimeError, match="no third derivative"):
        torch.autograd.grad(d2.sum(), x[0])
    _, ty = torch.func.jvp(_own, tuple(x), tuple(plain))
    d = torch.autograd.grad(ty[0].sum(), x[1], create_graph=True)[0]
    with pytest.raises(RuntimeError, match="no second derivative through the tangent"):
        torch.autograd.grad(d.sum(), x[1])
    with pytest.raises(NotImplementedError, match="no rule for"):
        torch.func.vmap(la.linear_attention)(*(t[:, None] for t in plain[:3]))
    with pytest.raises(RuntimeError, match="further forward"):
        torch.func.jvp(lambda a: torch.func.jvp(lambda b: la.linear_attention(b, *plain[1:3]), (a,), (a,))[1], (plain[0],), (plain[0],))


def test_bad_arguments(cpu):
    q, k, v, s = _operands(12)
    f = la.linear_attention
    for error, call in [
        (ValueError, lambda: f(q, k[:, :, :4], v)), (ValueError, lambda: f(q, k, v[:, :2])), (ValueError, lambda: f(q[0], k[0], v[0])), (TypeError, lambda: f(q, k.float(), v)),
        (TypeError, lambda: f(q, k, v, DECAY.double())), (TypeError, lambda: f(q, k, v, DECAY[:2])), (NotImplementedError, lambda: f(q, k, v, DECAY.clone().requires_grad_())),
        (ValueError, lambda: f(q, k, v, state=s[:1])), (TypeError, lambda: f(q, k, v, lengths=LENGTHS.long())), (TypeError, lambda: f(q, k, v, lengths=LENGTHS[:1])),
        (ValueError, lambda: f(q, k, v, sm_scale=0.0)), (ValueError, lambda: f(q, k, v, sm_scale=float("nan"))), (ValueError, lambda: f(q[..., :0], k[..., :0], v)),
        (ValueError, lambda: f(*(torch.ones(1, 1, 1, 129),) * 3)), (ValueError, lambda: f(q, k, v, torch.zeros(2 * H)[::2])),
    ]:
        with pytest.raises(error):
            call()
    step, t = la.linear_attention_step, [x[:, :, 0] for x in (q, k, v)]
    for error, call in [
        (ValueError, lambda: step(q, k, v, DECAY, s)), (ValueError, lambda: step(*t, DECAY, s[:1])), (TypeError, lambda: step(t[0], t[1].float(), t[2], DECAY, s)),
        (NotImplementedError, lambda: step(t[0].requires_grad_(), *t[1:], DECAY, s)), (ValueError, lambda: step(*t, DECAY, s, sm_scale=0.0)),
    ]:
        with pytest.raises(error):
            call()


def test_a_decay_that_is_a_parameter(cpu):
    """Refused where a gradient would be lost, and only there."""
    q, k, v, s = _operands(13)
    w = DECAY.clone().requires_grad_()
    want = la.linear_attention(q, k, v, DECAY, state=s, return_state=True)
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            _close(la.linear_attention(q, k, v, w, state=s, return_state=True), want)
            la._check_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], w, 1.0, s)
    for call in (lambda: la.linear_attention(q, k, v, w), lambda: la.linear_attention_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], w, s)):
        with pytest.raises(NotImplementedError, match="log_decay"):
            call()
    with torch.no_grad(), fwAD.dual_level(), pytest.raises(NotImplementedError, match="log_decay"):
        la.linear_attention(q, k, v, fwAD.make_dual(DECAY, DECAY))


def test_rows_are_counted_in_32_bits():
    x = torch.ones(1, 1, 1, 1).expand(1, 1, 2**30 + 1, 1)
    with pytest.raises(ValueError, match="at most 2\\*\\*30 rows"):
        la.linear_attention(x, x, x)


def test_no_cpu_fallback():
    x = torch.ones(1, 2, 3, 4)
    with pytest.raises(RuntimeError, match="runs only on CUDA tensors"):
        la.linear_attention(x, x, x)
    with pytest.raises(RuntimeError, match="runs only on CUDA tensors"):
        la.linear_attention_step(x[:, :, 0], x[:, :, 0], x[:, :, 0], None, torch.ones(1, 2, 4, 4))


def test_the_c_entries_refuse():
    lib = _lib.load()

    def call(entry, **kw):
        a = _lib.LinearArgs()
        a.struct_size = ctypes.sizeof(a)
        a.B = a.H = 1
        a.L, a.D, a.E, a.scale = 4, 8, 8, 1.0
        a.q.p = a.k.p = a.v.p = a.o.p = 64
        for key, v in kw.items():
            if isinstance(getattr(a, key), _lib.LinearTensor):
                getattr(a, key).p = v
            elif key == "stride":
                a.q.stride[0] = v
            else:
                setattr(a, key, v)
        return entry(ctypes.byref(a), None)

    both = [(-7, dict(struct_size=8)), (-3, dict(dtype=3)), (-2, dict(B=0)), (-2, dict(L=0)), (-2, dict(D=129)), (-2, dict(E=0)), (-10, dict(B=1 << 20, H=17)), (-10, dict(L=2**30 + 1)),
            (-9, dict(scale=float("nan"))), (-1, dict(q=None)), (-1, dict(tq=64)), (-1, dict(tstate=64)), (-8, dict(k=65)), (-8, dict(state=66)), (-8, dict(lengths=66)),
            (-1, dict(L=4096))]
    for entry, more in ((lib.jvpfa_linear_fwd, [(-1, dict(o=None)), (-1, dict(dual=1))]), (lib.jvpfa_linear_bwd, [(-1, dict(dstate=64)), (-9, dict(scale=0.0, gstate=64))])):
        assert entry(None, None) == -1
        for want, kw in both + more:
            assert call(entry, **kw) == want, kw

    def step(**kw):
        a = _lib.LinearStepArgs()
        a.struct_size = ctypes.sizeof(a)
        a.B = a.H = 2
        a.D = a.E = 4
        a.scale, a.q, a.k, a.v, a.o, a.state = 1.0, 64, 64, 64, 64, 64
        a.state_stride[0], a.state_stride[1] = kw.pop("state_stride", (32, 16))
        for key, v in kw.items():
            setattr(a, key, v)
        return lib.jvpfa_linear_step(ctypes.byref(a), None)

    assert lib.jvpfa_linear_step(None, None) == -1
    for want, kw in [(-7, dict(struct_size=8)), (-3, dict(dtype=9)), (-2, dict(D=0)), (-2, dict(E=129)), (-1, dict(o=None)), (-8, dict(q=65)), (-8, dict(state=66)),
                     (-2, dict(state_stride=(0, 16))), (-2, dict(state_stride=(16, 16))), (-2, dict(state_stride=(24, 16))), (-2, dict(state_stride=(16, 8)))]:
        assert step(**kw) == want, kw


def test_sequences_are_cut_into_rounds_that_fit():
    """float32 of 64 columns with tangents: shared memory has room for one CTA of an SM, so 148 at once (the cut shows in what a forward keeps)."""
    a = _lib.LinearArgs()
    a.struct_size = ctypes.sizeof(a)
    a.dtype, a.B, a.H, a.L, a.D, a.E, a.dual = 2, 3, 8, 1023, 64, 64, 1
    segments = _lib.load().jvpfa_linear_kept_bytes(ctypes.byref(a)) / (2 * 4 * a.B * a.H * a.D * a.E)
    assert segments > 1 and a.B * a.H * segments <= 148


def test_scales_beyond_32_bits_are_refused(cpu):
    """Backwards a last state's cotangent is divided by the scale, in 32 bits."""
    q, k, v, s = _operands(14)
    for scale in (1e-50, 1e-40, 1e-30, -1e-30, 1e30, 1e50):
        for call in (lambda: la.linear_attention(q, k, v, sm_scale=scale), lambda: la.linear_attention_step(q[:, :, 0], k[:, :, 0], v[:, :, 0], None, s, sm_scale=scale)):  # noqa: B023
            with pytest.raises(ValueError, match="sm_scale"):
                call()
    o, last = la.linear_attention(q, k, v, sm_scale=2.0**-64, return_state=True)
    torch.testing.assert_close(o, ((q @ k.transpose(-1, -2)).tril() @ v) * 2.0**-64, rtol=1e-6, atol=0)
    lib = _lib.load()
    for scale, gstate, want in ((2.0**-65, 64, -9), (2.0**65, None, -9), (float("inf"), None, -9), (2.0**-65, None, 0)):
        a = _lib.LinearArgs()
        a.struct_size = ctypes.sizeof(a)
        a.B = a.H = 1
        a.L, a.D, a.E, a.scale = 4, 8, 8, scale
        a.q.p = a.k.p = a.v.p = 64
        a.gstate = gstate
        got = lib.jvpfa_linear_bwd(ctypes.byref(a), None)
        assert got == want if want else got != -9
