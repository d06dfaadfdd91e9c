"""GPU tests of gated_linear against its formulas in float64, from the very inputs.

Entrywise bounds, propagated through the formulas.  e: half a step of the type (2^-8 bf16, 2^-11 fp16, 2^-24 fp32).  A sum of n products that
the tensor cores form is off by at most 17 n / 16 * 2^-23 of the sum of the products' magnitudes (every instruction of 16 rounds 17
numbers towards zero), fp32 ones, which are taken up every 1024, by as much for n = 1024, 2^-24 for each of these pieces and 2^-21 for the
parts left out (where the parts are cut: mid < 2^-7, lo < 2^-15 of the leading bit's, two products of one of each and lo lo).  An activation and its derivatives are off by eta (1 + |g|): 2^-17 by the fast exponential and division, 2^-20 for fp32.
Projections and their cotangents are rounded to the type on the way to the gradients.  |a'''| <= 2 for each activation.

Those bounds are the worst case.  Random inputs' errors add up as random numbers do, so the norm of an output's error is held to e (a
value: one rounding, at most 1 / sqrt(3) of e, and the sums) and 4 e (a gradient: at most six roundings in a row) of the output's norm, and fp32 to
1e-5, the library's bound."""
import pytest
import torch

import jvp_flash_attention_b200.rotary as rot
from jvp_flash_attention_b200 import _lib
from jvp_flash_attention_b200.gated import ACTIVATIONS, gated_linear
from jvp_flash_attention_b200.jvp_attention import JVPAttn
from tests import _block_formulas as formulas

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _sum_error(n, dtype):
    if dtype == torch.float32:
        return 17 * min(n, 1024) / 16 * 2.0**-23 + (n // 1024 + 2) * 2.0**-24 + 2.0**-21
    return 17 * n / 16 * 2.0**-23 + 2.0**-23


def _check(got, x, tx, wg, wu, gh, gth, kind):
    """got: dict of outputs by name."""
    dtype = x.dtype
    e = torch.finfo(dtype).eps / 2
    eta = 2.0**-20 if dtype == torch.float32 else 2.0**-17
    flat = lambda t: None if t is None else t.detach().double().reshape(-1, t.shape[-1])  # noqa: E731
    x, tx, wg, wu, gh, gth = (flat(t) for t in (x, tx, wg, wu, gh, gth))
    h, th, g, u, tg, tu = formulas.gated_fwd(x, tx, wg, wu, kind)
    a, a1, a2 = (t.abs() for t in formulas.activation(kind, g))
    dx, dtx, dwg, dwu = formulas.gated_bwd(x, tx, wg, wu, g, u, tg, tu, gh, gth, kind) if gh is not None or gth is not None else (None,) * 4
    k = _sum_error(x.shape[1], dtype)
    tiny = torch.finfo(dtype).smallest_normal * e  # half the spacing of the smallest numbers, which cotangents of fp16 reach
    zero = torch.zeros_like(g)
    Eg, Eu = k * (x.abs() @ wg.abs().T), k * (x.abs() @ wu.abs().T)
    act = eta * (1 + g.abs())
    want = {"h": h, "th": th, "dx": dx, "dtx": dtx, "dwg": dwg, "dwu": dwu}
    # the bounds do without signs
    G, U = g.abs(), u.abs()
    bounds = {"h": a1 * U * Eg + a * Eu + act * U}
    if tx is not None:
        TG, TU = tg.abs(), tu.abs()
        Etg, Etu = k * (tx.abs() @ wg.abs().T), k * (tx.abs() @ wu.abs().T)
        bounds["th"] = a1 * U * Etg + a * Etu + (a2 * TG * U + a1 * TU) * Eg + a1 * TG * Eu + act * (TG * U + TU)
        Etg, Etu = Etg + e * TG, Etu + e * TU
    if dx is not None:
        Eg, Eu = Eg + e * G, Eu + e * U
        GH, GTH = (zero if t is None else t.abs() for t in (gh, gth))
        Edg, Edu = GH * (a2 * U * Eg + a1 * Eu + act * U), GH * (a1 * Eg + act)
        mdg, mdu = GH * a1 * U, GH * a  # magnitudes of the cotangents' terms
        if gth is not None:
            Edg = Edg + GTH * ((2 * TG * U + a2 * TU) * Eg + a2 * TG * Eu + a2 * U * Etg + a1 * Etu + act * (2 * TG * U + TU))
            Edu = Edu + GTH * (a2 * TG * Eg + a1 * Etg + act * TG)
            mdg, mdu = mdg + GTH * (a2 * TG * U + a1 * TU), mdu + GTH * a1 * TG
            mdtg, mdtu = GTH * a1 * U, GTH * a
            Edtg, Edtu = (GTH * (a2 * U * Eg + a1 * Eu + act * U) + (e + 2.0**-22) * mdtg + tiny,
                          GTH * (a1 * Eg + act) + (e + 2.0**-22) * mdtu + tiny)
        Edg, Edu = Edg + (e + 2.0**-21) * mdg + tiny, Edu + (e + 2.0**-21) * mdu + tiny
        f, m = _sum_error(2 * g.shape[1], dtype), _sum_error(x.shape[0] * (2 if gth is not None else 1), dtype)
        WG, WU, X = wg.abs(), wu.abs(), x.abs()
        bounds["dx"] = (Edg + f * mdg) @ WG + (Edu + f * mdu) @ WU
        bounds["dwg"], bounds["dwu"] = (Edg + m * mdg).T @ X, (Edu + m * mdu).T @ X
        if gth is not None:
            bounds["dtx"] = (Edtg + f * mdtg) @ WG + (Edtu + f * mdtu) @ WU
            bounds["dwg"], bounds["dwu"] = bounds["dwg"] + (Edtg + m * mdtg).T @ tx.abs(), bounds["dwu"] + (Edtu + m * mdtu).T @ tx.abs()
    small = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    for name, y in got.items():
        assert y.dtype == dtype and y.isfinite().all(), name
        y, w = flat(y), want[name]
        off, bound = (y - w).abs(), (1 + e) * bounds[name] + e * w.abs() + small
        assert (off <= bound).all(), (name, (off / bound).max().item())
        most = 1e-5 if dtype == torch.float32 else e * (1 if name in ("h", "th") else 4)
        if w.norm() > 0 and dtype != torch.float16 or w.norm() > 1e-3 * w.numel() ** 0.5:  # (not where fp16 has no normal numbers left)
            assert (y - w).norm() <= most * w.norm(), (name, ((y - w).norm() / w.norm()).item())


def _inputs(M, K, F, dt, seed, rows=None):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s, std=1.0: (torch.randn(*s, generator=g, device=DEV) * std).to(DT[dt])  # noqa: E731
    rows = rows or (M,)
    return r(*rows, K), r(*rows, K, std=0.3), r(F, K, std=K**-0.5), r(F, K, std=K**-0.5), r(*rows, F), r(*rows, F)


def _run(x, tx, wg, wu, gh, gth, name, step):
    leaves = [t if t is None else t.detach().requires_grad_() for t in (x, tx, wg, wu)]
    if not step.startswith("jvp"):
        h = gated_linear(leaves[0], leaves[2], leaves[3], name)
        got = {"h": h.detach()}
        if step == "fwd_bwd":
            got.update(zip(("dx", "dwg", "dwu"), torch.autograd.grad(h, [leaves[0], *leaves[2:]], gh)))
        return got
    h, th = torch.func.jvp(lambda v: gated_linear(v, leaves[2], leaves[3], name), (leaves[0],), (leaves[1],))
    got = {"h": h.detach(), "th": th.detach()}
    if step == "jvp_bwd":
        got.update(zip(("dx", "dtx", "dwg", "dwu"), torch.autograd.grad((h, th), leaves, (gh, gth))))
    elif step == "jvp_bwd_t":
        got.update(zip(("dx", "dtx", "dwg", "dwu"), torch.autograd.grad(th, leaves, gth)))
    return got


def _case(M, K, F, dt, name, step, seed=0, **kw):
    x, tx, wg, wu, gh, gth = _inputs(M, K, F, dt, seed + M + K + F, **kw)
    got = _run(x, tx, wg, wu, gh, gth, name, step)
    dual = step.startswith("jvp")
    _check(got, x, tx if dual else None, wg, wu, gh if step in ("fwd_bwd", "jvp_bwd") else None, gth if step in ("jvp_bwd", "jvp_bwd_t") else None,
           ACTIVATIONS[name])
    assert _lib.device_status() == 0


SIZES = [(1, 64, 64), (1, 8, 8), (3, 40, 24), (2, 1, 1), (5, 7, 9), (130, 72, 200), (257, 129, 131), (300, 512, 264), (64, 1000, 130), (1000, 64, 520),
         (513, 264, 1030), (127, 96, 128), (128, 256, 127), (256, 128, 256)]


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("M,K,F", SIZES)
@pytest.mark.parametrize("step", ["fwd_bwd", "jvp_bwd"])
def test_values_and_gradients(M, K, F, dt, step):
    _case(M, K, F, dt, list(ACTIVATIONS)[(M + K + F) % 4], step)


@pytest.mark.parametrize("name", list(ACTIVATIONS))
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("step", ["fwd", "jvp", "jvp_bwd_t"])
def test_activations(name, dt, step):
    _case(70, 136, 150, dt, name, step)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("step", ["fwd_bwd", "jvp_bwd"])
def test_several_tiles_of_a_cluster(dt, step):
    """More tiles than clusters, and a depth of several passes through the stages."""
    _case(2100, 704, 2312, dt, "silu", step)
    _case(400, 2500, 900, dt, "gelu_tanh", step)


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("M", [1, 2, 17, 64, 65, 128, 129])
@pytest.mark.parametrize("step", ["fwd_bwd", "jvp_bwd"])
def test_few_rows(M, dt, step):
    """Around the number of rows up to which the weights set the pace (128, value and tangent together), with clusters of one to eight CTAs."""
    for K, F in ((1032, 264), (4100, 72), (200, 3300), (264, 20000)):
        _case(M, K, F, dt, "silu" if K > 1000 else "gelu", step)


@pytest.mark.parametrize("rows", [(0,), (0, 3), (3, 0)])
def test_no_rows(rows):
    x, tx, wg, wu, gh, gth = _inputs(0, 16, 8, "bf16", 1, rows=rows)
    got = _run(x, tx, wg, wu, gh, gth, "silu", "jvp_bwd")
    assert got["h"].shape == got["th"].shape == (*rows, 8) and got["dx"].shape == (*rows, 16)
    assert not got["dwg"].any() and not got["dwu"].any()


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_layouts(dt):
    M, K, F = 60, 48, 56
    x, tx, wg, wu, gh, gth = _inputs(M, K, F, dt, 3, rows=(5, 12))
    both = torch.cat((wg, wu))
    wide = torch.zeros(5, 12, K + 3, device=DEV, dtype=DT[dt])
    wide[..., 1:K + 1] = x
    forms = {
        "halves": (x, both[:F], both[F:]), "between": (x, torch.stack((wg, wu), 1)[:, 0], torch.stack((wg, wu), 1)[:, 1]),
        "slice": (wide[..., 1:K + 1], wg, wu), "columns": (x.transpose(0, 2).contiguous().transpose(0, 2), wg.t().contiguous().t(), wu),
    }
    for name, (v, a, b) in forms.items():
        got = _run(v, tx.transpose(0, 1).contiguous().transpose(0, 1), a, b, gh, gth.transpose(0, 1).contiguous().transpose(0, 1), "silu", "jvp_bwd")
        _check(got, v, tx, a, b, gh, gth, 0)
    v = x[:1, :1].expand(5, 12, K)  # one row for all (which torch lets no tangent be written to)
    _check(_run(v, None, wg, wu, gh, None, "silu", "fwd_bwd"), v, None, wg, wu, gh, None, 0)
    h = gated_linear(x[0, 0], wg, wu)
    assert h.shape == (F,)
    _check({"h": h}, x[0, :1], None, wg, wu, None, None, 0)


def test_a_broadcast_cotangent():
    x, tx, wg, wu, _, _ = _inputs(40, 64, 48, "bf16", 4)
    x.requires_grad_()
    (dx,) = torch.autograd.grad(gated_linear(x, wg, wu).sum(), x)
    _check({"dx": dx}, x, None, wg, wu, torch.ones(40, 48, device=DEV), None, 0)


@pytest.mark.parametrize("name", list(ACTIVATIONS))
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_far_arguments(name, dt):
    """Gates of up to +-200: no overflow on the way, and tails that are zero where they should be."""
    K, F = 8, 64
    x = torch.zeros(50, K, device=DEV, dtype=DT[dt])
    x[:, 0] = torch.linspace(-200, 200, 50, device=DEV).to(DT[dt])
    x[:, 1] = 1
    wg, wu = torch.zeros(F, K, device=DEV, dtype=DT[dt]), torch.zeros(F, K, device=DEV, dtype=DT[dt])
    wg[:, 0], wu[:, 1] = 1, 1
    tx, g = torch.ones_like(x), torch.ones(50, F, device=DEV, dtype=DT[dt])
    got = _run(x, tx, wg, wu, g, g, name, "jvp_bwd")
    _check(got, x, tx, wg, wu, g, g, ACTIVATIONS[name])


@pytest.mark.parametrize("name", list(ACTIVATIONS))
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_arguments_at_the_end_of_the_range(name, dt):
    """Gates of +-1e12 and (but for the tanh form, whose cube is not finite there) +-1e30: a and a' have their limits, 0 and g, 0 and 1; for the sigmoid 0
    and 1, 0 and 0."""
    x = torch.zeros(4, 8, device=DEV, dtype=DT[dt])
    far = 1e12 if name == "gelu_tanh" else 1e30
    x[:, 0] = torch.tensor([-1e12, 1e12, -far, far], device=DEV)
    x[:, 1] = 1
    w = torch.zeros(2, 64, 8, device=DEV, dtype=DT[dt])
    w[0, :, 0], w[1, :, 1] = 1, 1
    tx = torch.zeros_like(x)
    tx[:, 0] = 1
    h, th = torch.func.jvp(lambda v: gated_linear(v, w[0], w[1], name), (x,), (tx,))
    up = torch.tensor([0.0, 1.0, 0.0, 1.0], device=DEV)[:, None].expand(4, 64).to(DT[dt])
    assert torch.equal(h, up if name == "sigmoid" else up * x[:, :1].clamp_min(0))
    assert torch.equal(th, torch.zeros_like(up) if name == "sigmoid" else up)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_nan_and_infinite_entries_stay_in_their_rows(dt):
    x, tx, wg, wu, gh, _ = _inputs(300, 64, 200, dt, 5)
    want = gated_linear(x, wg, wu)
    x[7, 3], x[299, 0], x[128, 63] = float("nan"), float("inf"), -float("inf")
    h = gated_linear(x, wg, wu)
    rows = torch.ones(300, dtype=torch.bool, device=DEV)
    rows[[7, 299, 128]] = False
    assert torch.equal(h[rows], want[rows])
    assert h[7].isnan().all() and not h[299].isfinite().any() or dt == "bf16" and h[7].isnan().all()


def test_results_are_the_same_from_run_to_run():
    for dt in ("bf16", "fp32"):
        args = _inputs(700, 520, 1200, dt, 6)
        first, second = (_run(*args, "silu", "jvp_bwd") for _ in range(2))
        assert all(torch.equal(first[k], second[k]) for k in first)


def test_a_gradient_penalty():
    x, tx, wg, wu, gh, _ = _inputs(90, 72, 136, "fp32", 7)
    out = []
    for own in (True, False):
        leaves = [(t if own else t.double()).detach().requires_grad_() for t in (x, wg, wu, gh)]
        f = gated_linear if own else lambda v, a, b: torch.nn.functional.silu(v @ a.T) * (v @ b.T)
        (dx,) = torch.autograd.grad(f(*leaves[:3]), leaves[0], leaves[3], create_graph=True)
        out.append(torch.autograd.grad((dx * (tx if own else tx.double())).sum(), leaves))
    for a, b in zip(*out):
        assert (a.double() - b).norm() <= 1e-5 * b.norm()


def test_projections_beyond_the_types_range():
    """fp16 gates of 10^5.  h is formed from sums in 32 bits, and the projections are kept with fp32's range; their cotangents are rounded to
    fp16, as documented, so a row in which one passes 65504 has a gradient that is not finite, and others are as exact as ever."""
    K, F = 64, 72
    x, _, wg, wu, gh, _ = _inputs(40, K, F, "fp16", 13)
    x = (x * 50).half()
    wg = (wg * 3000).half()  # |g| of 10^5 and more
    wu = (wu * 1e-4).half()
    want = [t.double().detach().requires_grad_() for t in (x, wg, wu)]
    g = want[0] @ want[1].T
    hw = torch.nn.functional.silu(g) * (want[0] @ want[2].T)
    assert (g.abs() > 65504).any() and (hw.abs() < 65504).all()
    for scale in (1.0, 2.0**-8):
        leaves = [t.detach().requires_grad_() for t in (x, wg, wu)]
        h = gated_linear(*leaves)
        assert (h.double() - hw).abs().max() <= 2.0**-10 * hw.abs().max()
        c = (gh * scale).half()
        du = (c.double() * torch.nn.functional.silu(g.detach())).abs()
        grads, ref = torch.autograd.grad(h, leaves, c), torch.autograd.grad(hw, want, c.double(), retain_graph=True)
        beyond = (du > 65520).any(1)  # (up to there a number rounds to 65504)
        assert beyond.any() if scale == 1.0 else not (du > 65504).any()
        assert torch.equal(~grads[0].isfinite().all(1), beyond)
        dx, rx = grads[0][~beyond].double(), ref[0][~beyond]
        assert (dx - rx).norm() <= 4 * 2.0**-11 * rx.norm()
        if scale < 1:
            for d, r in zip(grads[1:], ref[1:]):
                inside = r.abs() < 65504  # (the gradients themselves are fp16)
                assert (d.double() - r)[inside].norm() <= 4 * 2.0**-11 * r[inside].norm()


def test_graphs_of_a_call():
    x, tx, wg, wu, gh, gth = _inputs(20, 64, 48, "bf16", 14)
    x.requires_grad_(), wg.requires_grad_()
    h = gated_linear(x, wg, wg)  # one weight for both: its gradient is the sum
    (dw,) = torch.autograd.grad(h, wg, gh, retain_graph=True)
    w = wg.detach().double().requires_grad_()
    p = x.detach().double() @ w.T
    (ref,) = torch.autograd.grad(torch.nn.functional.silu(p) * p, w, gh.double())
    assert (dw.double() - ref).norm() <= 2 * 4 * 2.0**-8 * ref.norm()
    first, second = (torch.autograd.grad(h, x, gh, retain_graph=True)[0] for _ in range(2))
    assert torch.equal(first, second)
    torch.autograd.grad(h, x, gh)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(h, x, gh)
    h = gated_linear(x, wg, wu)
    with torch.no_grad():
        wg.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(h, x, gh)


def test_a_tangent_that_is_zero():
    """torch hands some zero tangents over as a shape without memory."""
    x, _, wg, wu, _, _ = _inputs(20, 64, 48, "bf16", 15)
    with torch.autograd.forward_ad.dual_level():
        zero = torch._efficientzerotensor(x.shape, dtype=x.dtype, device=x.device)
        h, th = torch.autograd.forward_ad.unpack_dual(gated_linear(torch.autograd.forward_ad.make_dual(x, zero), wg, wu))
    assert torch.equal(h, gated_linear(x, wg, wu)) and not th.any()


@pytest.mark.parametrize("M", [90, 400])
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_tangents_and_second_derivatives_of_the_weights(M, dt):
    """Against torch in float64.  Operands side by side are twice as wide, else these are the launches of the other tests: fp32 within 1e-5 of the
    norm (second derivatives: two gradients in a row, 2e-5), bf16 within e for values and 4 e for each gradient on the way."""
    x, tx, wg, wu, gh, gth = _inputs(M, 72, 136, dt, 18)
    tg, tu = (torch.randn_like(w) * 0.3 * 72**-0.5 for w in (wg, wu))
    e = 1e-5 if dt == "fp32" else 2.0**-8
    out = []
    for own in (True, False):
        cast = (lambda t: t) if own else (lambda t: t.double())
        f = gated_linear if own else lambda v, a, b: torch.nn.functional.silu(v @ a.T) * (v @ b.T)
        leaves = [cast(t).detach().requires_grad_() for t in (x, wg, wu)]
        tangents = [cast(t).detach().requires_grad_() for t in (tx, tg, tu)]
        h, th = torch.func.jvp(f, tuple(leaves), tuple(tangents))
        first = torch.autograd.grad((h, th), leaves + tangents, (cast(gh), cast(gth)))
        grads = torch.autograd.grad(f(*leaves), leaves, cast(gh), create_graph=True)
        second = torch.autograd.grad(grads, leaves, tangents)
        out.append([h, th, *first, *second])
    for i, (a, b) in enumerate(zip(*out)):
        most = e * (1 if i < 2 else (1 if dt == "fp32" else 4) * (1 if i < 8 else 2))
        assert (a.double() - b).norm() <= most * b.norm(), (i, ((a.double() - b).norm() / b.norm()).item())


def test_another_stream_and_captured_graphs():
    x, tx, wg, wu, gh, gth = _inputs(260, 100, 204, "bf16", 8)  # K = 100: copies in the workspace
    want = _run(x, tx, wg, wu, gh, gth, "silu", "jvp_bwd")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = _run(x, tx, wg, wu, gh, gth, "silu", "jvp_bwd")
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(got[k], want[k]) for k in want)
    with torch.no_grad():
        graphs, outs = [], []
        for _ in range(2):  # two graphs of one memory pool, replayed in turn
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
                outs.append(gated_linear(x, wg, wu))
            graphs.append(graph)
        x.copy_(tx)
        for graph, out in zip(graphs, outs):
            graph.replay()
        torch.cuda.synchronize()
        h = gated_linear(x, wg, wu)
    assert all(torch.equal(out, h) for out in outs)


def test_two_streams_at_once():
    """Calls that overlap on the GPU: each has its own workspace, and clusters wait for nothing of the other's."""
    args = [_inputs(1000, 260, 700, "fp32", s) for s in (9, 10)]
    want = [_run(*a, "gelu", "jvp_bwd") for a in args]
    streams = [torch.cuda.Stream() for _ in args]
    torch.cuda.synchronize()
    got = []
    for s, a in zip(streams, args):
        with torch.cuda.stream(s):
            got.append([_run(*a, "gelu", "jvp_bwd") for _ in range(3)])
    torch.cuda.synchronize()
    for runs, w in zip(got, want):
        assert all(torch.equal(r[k], w[k]) for r in runs for k in w)


def test_a_device_status_is_reported_and_cleared():
    x, tx, wg, wu, _, _ = _inputs(4, 64, 64, "bf16", 11)
    _lib.device_status_inject(5)
    try:
        with pytest.raises(RuntimeError, match="jvpfa_gated_fwd failed"):
            gated_linear(x, wg, wu)
    finally:
        assert _lib.device_status(clear=True) == 5
    assert gated_linear(x, wg, wu).isfinite().all()


def test_a_transformer_block_under_one_jvp():
    """Rotary, attention and the gated projection as a model strings them together, in fp32 against torch in float64: value, tangent
    and the gradients of a loss on both with respect to the weights."""
    B, L, H, D, F = 2, 66, 2, 32, 176
    E = H * D
    g = torch.Generator(device=DEV).manual_seed(12)
    r = lambda *s, std=1.0: torch.randn(*s, generator=g, device=DEV) * std  # noqa: E731
    x, tx, y1, y2 = r(B, L, E), r(B, L, E, std=0.3), r(B, L, E), r(B, L, E)
    weights = [r(3 * E, E, std=E**-0.5), r(E, E, std=E**-0.5), r(F, E, std=E**-0.5), r(F, E, std=E**-0.5), r(E, F, std=F**-0.5)]
    w = rot.rotary_frequencies(D, device=DEV)
    linear = torch.nn.functional.linear

    def block(x, wqkv, wo, wg, wu, wd, own):
        q, k, v = linear(x, wqkv).view(B, L, 3, H, D).transpose(1, 3).unbind(2)
        if own:
            q, k = rot.rotary(q, k, w)
            o = JVPAttn.fwd_dual(q, k, v, causal=True)
        else:
            q, k = formulas.turn(q, w), formulas.turn(k, w)
            s = (q @ k.transpose(-1, -2)) * D**-0.5
            o = torch.softmax(s.masked_fill(torch.ones(L, L, dtype=torch.bool, device=DEV).triu(1), -torch.inf), -1) @ v
        x = x + linear(o.transpose(1, 2).reshape(B, L, E), wo)
        h = gated_linear(x, wg, wu) if own else torch.nn.functional.silu(linear(x, wg)) * linear(x, wu)
        return x + linear(h, wd)

    out = []
    for own in (True, False):
        cast = (lambda t: t) if own else (lambda t: t.double())
        leaves = [cast(t).detach().requires_grad_() for t in weights]
        y, ty = torch.func.jvp(lambda v: block(v, *leaves, own), (cast(x),), (cast(tx),))
        out.append((y, ty, *torch.autograd.grad((y, ty), leaves, (cast(y1), cast(y2)))))
    for a, b in zip(*out):
        # five operators and three library products in a row, each within 1e-5 of its largest entry, and their gradients
        assert (a.double() - b).norm() <= 1e-4 * b.norm()


def test_a_captured_training_step():
    """Rotary in front of the gated projection, value, tangent and gradients, captured once and replayed on other inputs."""
    side = torch.cuda.Stream()  # (the legacy stream's graph nodes cannot be captured)
    g = torch.Generator(device=DEV).manual_seed(16)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).to(torch.bfloat16)  # noqa: E731
    q, tq, c, ct = r(2, 3, 50, 64), r(2, 3, 50, 64), r(2, 3, 50, 136), r(2, 3, 50, 136)
    wg, wu = (r(136, 64) / 8).requires_grad_(), (r(136, 64) / 8).requires_grad_()
    w = rot.rotary_frequencies(64, device=DEV)
    leaves = [q.requires_grad_(), tq.requires_grad_(), wg, wu]

    def step():
        h, th = torch.func.jvp(lambda x: gated_linear(rot.rotary(x, None, w), wg, wu), (q,), (tq,))
        return [h.detach(), th.detach(), *torch.autograd.grad((h, th), leaves, (c, ct))]

    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = step()
        with torch.no_grad():
            q.copy_(r(*q.shape)), c.copy_(r(*c.shape))
        graph.replay()
        first = [t.clone() for t in got]
        want = step()
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) and torch.equal(a, x) for a, b, x in zip(got, want, first))


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("M", [5, 700])
@pytest.mark.parametrize("step", ["fwd_bwd", "jvp_bwd"])
def test_a_replay_behind_a_launch_that_gave_up(M, dt, step):
    """With the status word set (from the host, as a thread that gives up a wait would) replayed kernels write NaN and end; cleared, they are
    themselves again.  K = 264, F = 2600: of 700 rows dw's tiles are cut, and joined."""
    args = _inputs(M, 264, 2600, dt, 17)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = _run(*args, "silu", step)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = _run(*args, "silu", step)
        for code in (9, 0):
            _lib.device_status_inject(code)
            try:
                graph.replay()
                side.synchronize()
            finally:
                assert _lib.device_status(clear=True) == code
            for name, y in got.items():
                assert y.isnan().all() if code else torch.equal(y, want[name]), (code, name)
