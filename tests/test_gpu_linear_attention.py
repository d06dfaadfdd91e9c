"""GPU tests of linear attention against its definition in float64.

Bound of an entry: half a step of its type; 2^-11 of the sum of the magnitudes that it is made of for 16-bit types, whose weighted products of
queries and keys, states and weighted values may have 11 bits (half a step of each, 2^-12, and two of them stand one behind the other); and for sums in 32 bits, which the tensor cores truncate (2^-23 a step): at most three instructions
for every 8 rows or entries and 22 bits of each operand, (3 (L / 8 + D / 8 + 8) + 8) 2^-22 of that sum.  A gradient is such a map too; one through
tangents is a sum of three."""
import pytest
import torch

import jvp_flash_attention_b200.linear_attention as la
import jvp_flash_attention_b200.rotary as rot
from jvp_flash_attention_b200 import norms
from jvp_flash_attention_b200.gated import gated_linear
from tests import _linear_formulas as formulas

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _bits(L, D):
    return (3 * (L / 8 + D / 8 + 8) + 8) * 2.0**-22


def _near(got, want, size, rel, what=""):
    step = torch.finfo(got.dtype).eps / 2
    smallest = torch.finfo(got.dtype).smallest_normal * step * 2
    bound = step * want.abs() + (1 + step) * rel * size + smallest
    off = (got.double() - want).abs()
    assert got.shape == want.shape and (off <= bound).all(), (what, (off / bound).max().item())


def _make(B, H, L, W, dtype, layout, g, std=1.0):
    if layout == "blhd":
        return (torch.randn(B, L, H, W, generator=g, device=DEV) * std).to(dtype).transpose(1, 2)
    if layout == "odd":  # rows that begin anywhere
        return (torch.randn(B, H, L, W + 1, generator=g, device=DEV) * std).to(dtype)[..., 1:]
    if layout == "columns":  # not contiguous in the head dimension
        return (torch.randn(B, H, W, L, generator=g, device=DEV) * std).to(dtype).transpose(2, 3)
    return (torch.randn(B, H, L, W, generator=g, device=DEV) * std).to(dtype)


CASES = [
    # B, H, L, D, E, layout, decay, state, lengths
    (1, 1, 1, 64, 64, "bhld", "slow", False, None),
    (2, 3, 1, 32, 32, "bhld", None, True, None),
    (1, 2, 63, 64, 64, "blhd", "slow", True, None),
    (2, 2, 64, 128, 128, "bhld", "slow", False, None),
    (1, 3, 65, 64, 64, "bhld", "fast", True, None),
    (2, 1, 130, 32, 64, "blhd", "slow", True, (130, 7)),
    (3, 2, 200, 64, 32, "bhld", "slow", True, (0, 200, 65)),
    (1, 2, 97, 1, 1, "bhld", "slow", True, None),
    (1, 2, 77, 33, 7, "odd", "slow", True, None),
    (2, 2, 70, 100, 128, "odd", "mixed", False, (70, 1)),
    (1, 2, 90, 64, 64, "columns", "mixed", False, None),
    (1, 1, 1330, 64, 64, "blhd", "slow", True, None),
    (2, 2, 1030, 128, 128, "bhld", "mixed", True, (1030, 300)),
    (1, 2, 2048, 40, 24, "blhd", None, False, None),
    (1, 2, 769, 128, 64, "blhd", "fast", True, (640,)),
    (2, 2, 1400, 33, 7, "odd", "slow", True, (1400, 515)),
    (1, 3, 2500, 5, 3, "bhld", "mixed", True, None),
    (3, 4, 24, 32, 128, "blhd", "mixed", True, (3, 24, 10)),  # little is left of a given state
    (2, 4, 6, 103, 107, "blhd", "mixed", True, (3, 6)),
]


def _decay(kind, H):
    if kind is None:
        return None
    slow = torch.log1p(-torch.exp2(-5 - 7 * torch.arange(H, device=DEV) / max(H - 1, 1)))
    return {"slow": slow, "fast": slow * 40, "mixed": torch.tensor([0.0, -float("inf"), -3.0, -0.01][:H], device=DEV)}[kind]


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("dual", [False, True])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_values_tangents_and_gradients(case, dual, dt):
    B, H, L, D, E, layout, decay, has_state, lengths = CASES[case]
    g = torch.Generator(device=DEV).manual_seed(case)
    make = lambda std: [_make(B, H, L, W, DT[dt], layout, g, std).detach().requires_grad_() for W in (D, D, E)] + (  # noqa: E731
        [(3 * std * torch.randn(B, H, D, E, generator=g, device=DEV)).requires_grad_()] if has_state else [])
    x, tx = make(1.0), make(0.3) if dual else []
    w = _decay(decay, H)
    n = None if lengths is None else torch.tensor(lengths, device=DEV, dtype=torch.int32)
    scale = 0.3

    def f(q, k, v, s=None):
        return la.linear_attention(q, k, v, w, sm_scale=scale, state=s, lengths=n, return_state=True)

    y, ty = torch.func.jvp(f, tuple(x), tuple(tx)) if dual else (f(*x), ())
    cots = [_make(B, H, L, E, DT[dt], layout, g), torch.randn(B, H, D, E, generator=g, device=DEV)]
    tcots = [_make(B, H, L, E, DT[dt], layout, g), torch.randn(B, H, D, E, generator=g, device=DEV)] if dual else [None, None]
    grads = torch.autograd.grad((*y, *ty), (*x, *tx), [c for c in (*cots, *tcots) if c is not None], materialize_grads=True)
    full = lambda ts: list(ts) + [None] * (4 - len(ts))  # noqa: E731
    opts, extras = (scale, True, ""), (w, n)
    want, twant, _ = formulas.launch_fwd(full(x), full(tx), extras, opts, False)
    dwant = formulas.launch_bwd(full(x), full(tx), extras, None, cots, tcots, opts, [True] * 8)
    mag = lambda ts: [None if t is None else t.detach().abs() for t in full(ts)]  # noqa: E731
    size, tsize, _ = formulas.launch_fwd(mag(x), mag(tx), extras, opts, False)
    dsize = formulas.launch_bwd(mag(x), mag(tx), extras, None, [c.abs() for c in cots], [None if c is None else c.abs() for c in tcots], opts, [True] * 8)
    bits = _bits(L, max(D, E))
    outs = bits if dt == "fp32" else bits + 2.0**-11
    _near(y[0].detach(), want[0], size[0], outs, "o")
    _near(y[1].detach(), want[1], size[1], bits, "state")
    if dual:
        _near(ty[0].detach(), twant[0], tsize[0], outs, "to")
        _near(ty[1].detach(), twant[1], tsize[1], bits, "tstate")
    m = len(x)
    for i, d in enumerate(grads):
        at = i if i < m else 4 + i - m
        _near(d, dwant[at], dsize[at], bits if at % 4 == 3 else outs, f"gradient {at}")
    if n is not None:  # what stands behind the sequences is not read
        with torch.no_grad():
            bad = [t.detach().clone() for t in x]
            for t in bad[:3]:
                for b, m in enumerate(lengths):
                    t[b, :, m:] = float("nan")
            # (in the same form: with tangents the order of some sums is another one)
            o, s = torch.func.jvp(f, tuple(bad), tuple(tx))[0] if dual else f(*bad)
        assert torch.equal(o, y[0]) and torch.equal(s, y[1])


def test_what_is_left_keeps_its_digits():
    """Of a state alone, decayed row by row, over a whole sequence and over several segments of one."""
    w = torch.tensor([-3.0, -9.0, -0.02, -1e-4], device=DEV)
    s = torch.randn(1, 4, 64, 64, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV)
    for dt in DT.values():
        zero = torch.zeros(1, 4, 1000, 64, device=DEV, dtype=dt)
        token = s.clone()
        la.linear_attention_step(zero[:, :, 0], zero[:, :, 0], zero[:, :, 0], w, token)
        for n, got in [(1, token)] + [(n, la.linear_attention(zero[:, :, :n], zero[:, :, :n], zero[:, :, :n], w, state=s, return_state=True)[1]) for n in (1, 3, 9, 1000)]:
            want = s.double() * (w.double() * n).exp()[:, None, None]
            # an exponent's rounding and its function's, and a rounding for each of up to 16 chunks and 8 segments, all of them taken twice
            rel = 2 * ((w.double() * n).abs()[:, None, None] + 2 + 2 * 24) * 2.0**-24
            assert ((got.double() - want).abs() <= rel * want.abs() + 2.0**-126).all(), (dt, n)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_far_rows(dt):
    """A slow decay over a long sequence: states keep their digits, and pieces give what the whole gives."""
    B, H, L, D = 1, 2, 8192, 64
    g = torch.Generator(device=DEV).manual_seed(1)
    q, k, v = (_make(B, H, L, D, DT[dt], "blhd", g) for _ in range(3))
    w = torch.tensor([-(2.0**-12), 0.0], device=DEV)
    o, s = la.linear_attention(q, k, v, w, return_state=True)
    want, _, _ = formulas.launch_fwd([q, k, v, None], [None] * 4, (w, None), (D**-0.5, True, ""), False)
    assert (s.double() - want[1]).norm() <= 1e-6 * want[1].norm()
    assert (o.double() - want[0]).norm() <= (4e-3 if dt == "bf16" else 1e-6) * want[0].norm()  # (a bf16 rounding is 2^-8 / sqrt(12) on average)
    a, s1 = la.linear_attention(q[:, :, :5000], k[:, :, :5000], v[:, :, :5000], w, return_state=True)
    b, s2 = la.linear_attention(q[:, :, 5000:], k[:, :, 5000:], v[:, :, 5000:], w, state=s1, return_state=True)
    assert (s2 - s).norm() <= 2e-6 * s.norm()
    assert (torch.cat((a, b), 2).double() - want[0]).norm() <= (4e-3 if dt == "bf16" else 2e-6) * want[0].norm()


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("B,H,D,E,decay", [(1, 1, 64, 64, "slow"), (4, 16, 64, 64, "slow"), (3, 2, 128, 128, "mixed"), (2, 3, 33, 7, "slow"), (2, 2, 1, 1, None), (40, 8, 32, 100, "fast"),
                                           (2, 2, 128, 30, "slow")])
def test_tokens(B, H, D, E, decay, dt):
    """Token by token against whole sequences of the definition, with the state in a store of more matrices."""
    g = torch.Generator(device=DEV).manual_seed(2)
    n = 5
    x = torch.randn(n, B, H, 2 * D + E, generator=g, device=DEV).to(DT[dt])
    q, k, v = x[..., :D], x[..., D:2 * D], x[..., 2 * D:]
    store = torch.randn(B + 1, H + 2, D, E, generator=g, device=DEV)
    state = store[1:, 1:-1]
    before, w = store.clone(), _decay(decay, H)
    version = store._version
    o = torch.stack([la.linear_attention_step(q[i], k[i], v[i], w, state, sm_scale=0.5) for i in range(n)], 2)
    assert store._version == version + n
    full = [t.permute(1, 2, 0, 3) for t in (q, k, v)]
    args = ((w, None), (0.5, True, ""), False)
    want, _, _ = formulas.launch_fwd([*full, before[1:, 1:-1]], [None] * 4, *args)
    size, _, _ = formulas.launch_fwd([*(t.abs() for t in full), before[1:, 1:-1].abs()], [None] * 4, *args)
    # a token's sum has D terms in 32 bits, of a state that was rounded n times: (D + n + 8) 2^-24
    _near(o, want[0], size[0], (D + 16) * 2.0**-24)
    _near(state, want[1], size[1], 16 * 2.0**-24)
    store[1:, 1:-1] = before[1:, 1:-1]
    assert torch.equal(store, before)


def test_tokens_continue_prompts():
    B, H, L, D = 3, 4, 100, 64
    g = torch.Generator(device=DEV).manual_seed(3)
    q, k, v = (_make(B, H, L + 3, D, torch.bfloat16, "blhd", g) for _ in range(3))
    w = _decay("slow", H)
    want, want_s = la.linear_attention(q, k, v, w, return_state=True)
    o, s = la.linear_attention(q[:, :, :L], k[:, :, :L], v[:, :, :L], w, return_state=True)
    for i in range(L, L + 3):
        o = la.linear_attention_step(q[:, :, i], k[:, :, i], v[:, :, i], w, s)
        # both are off by roundings of bf16 and of the products to 11 bits
        assert (o - want[:, :, i]).norm() <= 1e-2 * want[:, :, i].norm()
    assert (s - want_s).norm() <= 2e-6 * want_s.norm()


def test_steps_that_are_refused():
    q = torch.randn(2, 3, 8, device=DEV)
    s = torch.randn(2, 3, 8, 8, device=DEV)
    for error, args in [(ValueError, (q, q, q, None, s[:1].expand(2, 3, 8, 8))), (ValueError, (q, q, q, None, s.transpose(2, 3))), (TypeError, (q, q, q, None, s.half())),
                        (ValueError, (q, q, q, None, s.cpu())), (TypeError, (q.double(),) * 3 + (None, s)), (NotImplementedError, (q, q, q, None, s.clone().requires_grad_()))]:
        with pytest.raises(error):
            la.linear_attention_step(*args)
    with torch.no_grad():
        la.linear_attention_step(q, q, q, None, s.clone().requires_grad_())
    with torch.inference_mode():
        kept, other = s.clone(), s.clone()
        o = la.linear_attention_step(q, q, q, None, kept)
    assert torch.equal(o, la.linear_attention_step(q, q, q, None, other.clone())) and not torch.equal(kept, s)
    before = kept.clone()
    with pytest.raises(RuntimeError, match="[Ii]nference"):
        la.linear_attention_step(q, q, q, None, kept)
    assert torch.equal(kept, before)


def test_a_decay_that_is_not_a_number_shows():
    q = torch.randn(1, 2, 70, 16, device=DEV)
    o = la.linear_attention(q, q, q, torch.tensor([float("nan"), -1.0], device=DEV))
    assert not o[0, 0, 1:].isfinite().any() and o[0, 1].isfinite().all()


@pytest.mark.parametrize("shape", [(0, 2, 5, 16), (2, 2, 0, 16), (2, 0, 5, 16)])
def test_empty(shape):
    q = torch.randn(shape, device=DEV, requires_grad=True)
    s = torch.randn(shape[0], shape[1], 16, 16, device=DEV, requires_grad=True)
    o, last = la.linear_attention(q, q, q, state=s, return_state=True)
    assert o.shape == q.shape and torch.equal(last, s)
    c = torch.randn_like(s)
    dq, ds = torch.autograd.grad((o.sum(), last), (q, s), (torch.ones((), device=DEV), c))
    assert dq.shape == q.shape and torch.equal(ds, c)


def test_streams_graphs_and_determinism():
    g = torch.Generator(device=DEV).manual_seed(4)
    q, k, v = (_make(2, 3, 1100, 64, torch.bfloat16, "blhd", g).detach().requires_grad_() for _ in range(3))
    w, n = _decay("slow", 3), torch.tensor([1100, 900], device=DEV, dtype=torch.int32)
    c = _make(2, 3, 1100, 64, torch.bfloat16, "bhld", g)

    def step():
        o, s = la.linear_attention(q, k, v, w, lengths=n, return_state=True)
        return (o.detach(), s.detach(), *torch.autograd.grad((o, s), (q, k, v), (c, torch.ones_like(s))))

    want = step()
    assert all(torch.equal(a, b) for a, b in zip(step(), want))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = step()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.no_grad():
        q.mul_(2), n.sub_(100)  # operands and lengths are read when the graph runs
    want = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
def test_powers_of_two_go_through(dt):
    """Operands and tangents times powers of two give results times powers of two, bit by bit, as long as nothing leaves the type's range."""
    big = 1 if dt == "fp16" else 5
    g = torch.Generator(device=DEV).manual_seed(8)
    x = [_make(1, 3, 150, 64, DT[dt], "bhld", g).clamp_(-4, 4) for _ in range(3)]
    tx = [_make(1, 3, 150, 64, DT[dt], "bhld", g, 0.25).clamp_(-1, 1) for _ in range(3)]
    x, tx = ([torch.where(t.abs() < 2.0**-6, 0, t) for t in ts] for ts in (x, tx))  # (nothing subnormal below)
    w = _decay("slow", 3)
    f = lambda *a: la.linear_attention(*a, w, return_state=True)  # noqa: E731
    y, ty = torch.func.jvp(f, tuple(x), tuple(tx))
    a, b, c, d = 2.0 ** (-4 * big), 2.0 ** (3 * big), 2.0 ** (2 * big), 2.0 ** (-2 * big)
    z, tz = torch.func.jvp(f, (x[0] * a, x[1] * b, x[2] * c), tuple(t * s * d for t, s in zip(tx, (a, b, c))))
    assert torch.equal(z[1], y[1] * (b * c)) and torch.equal(tz[1], ty[1] * (b * c * d))
    if dt != "fp16":  # (its small results are subnormal)
        assert torch.equal(z[0], y[0] * (a * b * c)) and torch.equal(tz[0], ty[0] * (a * b * c * d))
    else:
        assert (z[0] - y[0] * (a * b * c)).abs().max() <= 2.0**-10 * y[0].abs().max() * (a * b * c)


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_rows_of_very_different_size(dt):
    """A few rows 2^12 times the others, in one tile with them; values from 2^-20 on in a column."""
    B, H, L, D = 1, 2, 200, 64
    g = torch.Generator(device=DEV).manual_seed(9)
    q, k, v = (_make(B, H, L, D, DT[dt], "bhld", g) for _ in range(3))
    q[:, :, 37], k[:, :, 70:72], v[..., 5] = q[:, :, 37] * 2.0**8, k[:, :, 70:72] * 2.0**-12, v[..., 5] * 2.0**-12
    args = ((_decay("slow", H), None), (D**-0.5, True, ""), False)
    o, s = la.linear_attention(q, k, v, args[0][0], return_state=True)
    want, _, _ = formulas.launch_fwd([q, k, v, None], [None] * 4, *args)
    size, _, _ = formulas.launch_fwd([q.abs(), k.abs(), v.abs(), None], [None] * 4, *args)
    _near(o, want[0], size[0], _bits(L, D) + 2.0**-11, "o")
    _near(s, want[1], size[1], _bits(L, D), "state")


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("bad_value", [float("nan"), float("inf")])
def test_nonfinite_entries_stay_in_their_head_and_column(bad_value, dt):
    q, k, v = (torch.randn(2, 2, 200, 32, device=DEV).to(DT[dt]) for _ in range(3))
    want = la.linear_attention(q, k, v)
    v[1, 0, 150, 3] = bad_value
    o = la.linear_attention(q, k, v)
    bad = ~o.isfinite()
    assert bad[1, 0, 150:, 3].all() and not bad[1, 0, :128].any() and not bad[0].any() and not bad[1, 1].any() and not bad[..., :3].any() and not bad[..., 4:].any()
    assert torch.equal(o[~bad], want[~bad])


def test_second_derivatives():
    g = torch.Generator(device=DEV).manual_seed(5)
    a = [_make(1, 2, 70, 16, torch.float32, "bhld", g) for _ in range(3)]
    v = [_make(1, 2, 70, 16, torch.float32, "bhld", g) for _ in range(3)]
    w = _decay("slow", 2)
    results = []
    for kind in (torch.float32, torch.float64):
        def f(*x):
            if kind == torch.float32:  # noqa: B023
                return la.linear_attention(*x, w)
            return formulas.value(*x, None, formulas.Weights(x[0], (w, None)), 0.25)[0]
        x = [t.to(kind).requires_grad_() for t in a]
        u = [t.to(kind) for t in v]
        grads = torch.autograd.grad((f(*x) ** 3).sum(), x, create_graph=True)
        hv = torch.autograd.grad(sum((d * t).sum() for d, t in zip(grads, u)), x)
        p = [t.detach() for t in x]
        fr = torch.func.jvp(torch.func.grad(lambda *y: (f(*y) ** 3).sum(), argnums=(0, 1, 2)), tuple(p), tuple(u))  # noqa: B023
        results.append((*grads, *hv, *fr[0], *fr[1]))
    for got, want in zip(*results):
        # some hundred terms of either sign in 32 bits, several times over: 2^-24 * 256, of the largest entry
        assert (got.double() - want).abs().max() <= 2.0**-14 * want.abs().max()


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
def test_a_block_of_them(dt):
    """A transformer block with a linear mixer, conditioned norms and a gated projection under one torch.func.jvp, and its gradients,
    against the same formulas in float64."""
    B, H, L, D = 2, 4, 130, 32
    C, F = H * D, 200
    g = torch.Generator(device=DEV).manual_seed(6)
    randn = lambda *s, std=1.0: (torch.randn(*s, generator=g, device=DEV) * std).to(DT[dt])  # noqa: E731
    w_qkv, w_o, w_g, w_u, w_d = randn(3 * C, C, std=C**-0.5), randn(C, C, std=C**-0.5), randn(F, C, std=C**-0.5), randn(F, C, std=C**-0.5), randn(C, F, std=F**-0.5)
    weight = 1 + randn(C, std=0.1)
    x, cond = randn(B, L, C), [randn(B, 1, C, std=0.3) for _ in range(6)]
    tx, tcond = randn(B, L, C, std=0.1), [randn(B, 1, C, std=0.1) for _ in range(6)]
    decay, freq = _decay("slow", H), rot.rotary_frequencies(D, device=DEV)
    linear = torch.nn.functional.linear

    def own(x, sc1, sh1, g1, sc2, sh2, g2, ws):
        w_qkv, w_o, w_g, w_u, w_d, weight = ws
        n = norms.norm(x, scale=sc1, shift=sh1, kind="layer")
        q, k, v = linear(n, w_qkv).view(B, L, 3 * H, D).transpose(1, 2).split(H, 1)
        q, k = rot.rotary(q, k, freq)
        o = la.linear_attention(q, k, v, decay)
        y = linear(norms.norm(o.transpose(1, 2), kind="rms").reshape(B, L, C), w_o)
        r, n = norms.residual_norm(x, y, weight, gate=g1, scale=sc2, shift=sh2)
        return norms.residual(r, linear(gated_linear(n, w_g, w_u), w_d), gate=g2, post="rms", alpha=0.5)

    def exact(x, sc1, sh1, g1, sc2, sh2, g2, ws):
        w_qkv, w_o, w_g, w_u, w_d, weight = ws
        rms = lambda t: t * (t.square().mean(-1, keepdim=True) + 1e-6).rsqrt()  # noqa: E731
        center = lambda t: t - t.mean(-1, keepdim=True)  # noqa: E731
        n = rms(center(x)) * (1 + sc1) + sh1
        q, k, v = linear(n, w_qkv).view(B, L, 3 * H, D).transpose(1, 2).split(H, 1)
        p = (torch.arange(L, device=DEV).double()[:, None] * freq)

        def turn(t):
            a, b = t[..., :D // 2], t[..., D // 2:]
            return torch.cat((a * p.cos() - b * p.sin(), a * p.sin() + b * p.cos()), -1)

        o = formulas.value(turn(q), turn(k), v, None, formulas.Weights(q, (decay, None)), D**-0.5)[0]
        r = x + g1 * linear(rms(o.transpose(1, 2)).reshape(B, L, C), w_o)
        n = rms(r) * weight * (1 + sc2) + sh2
        h = torch.nn.functional.silu(linear(n, w_g)) * linear(n, w_u)
        return r + 0.5 * g2 * rms(linear(h, w_d))

    c1, c2 = randn(B, L, C), randn(B, L, C)
    results = []
    for f, kind in ((own, DT[dt]), (exact, torch.float64)):
        leaf = lambda t: t.to(kind).requires_grad_()  # noqa: B023, E731
        ws = tuple(map(leaf, (w_qkv, w_o, w_g, w_u, w_d, weight)))
        p, t = tuple(map(leaf, (x, *cond))), tuple(map(leaf, (tx, *tcond)))
        y, ty = torch.func.jvp(lambda *a: f(*a, ws), p, t)  # noqa: B023
        results.append((y, ty, *torch.autograd.grad((y, ty), (*p, *t, *ws), (c1.to(kind), c2.to(kind)))))
    for got, want in zip(*results):
        # about a dozen operators one behind another, each off by a few steps of its type on average, as torch's own products are: 32 half steps
        assert (got.double() - want).norm() <= 32 * torch.finfo(DT[dt]).eps / 2 * want.norm() * (4 if dt == "fp32" else 1)
