"""GPU tests of norm, residual and residual_norm against their formulas in float64.

Bound of an entry: half a step of its type, and for the arithmetic in 32 bits 2^-16 of the sum of the magnitudes that it is made of
(``_norm_formulas.sizes``).  A result is behind at most four sums over a row (two norms of two), each of at most 32 entries a thread, 5 steps
in a warp and 5 over warps (42 roundings), and behind about 40 other roundings: 4 * 42 + 40 < 256 = 2^8 roundings of 2^-24.  A vector's gradient is
besides a sum over rows, of at most 160 successive ones, 32 slices for each of 16 lanes and 16 of these, in these tests: 2^-15."""
import pytest
import torch

import jvp_flash_attention_b200.norms as norms
from tests import _norm_formulas as formulas

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
NAMES = ("x", "y", "weight", "bias", "scale", "shift", "gate", "post_weight")
ALL = set(NAMES)


def _near(got, want, size, bits, what):
    step = torch.finfo(got.dtype).eps / 2
    smallest = torch.finfo(got.dtype).smallest_normal * step * 2
    bound = step * want.abs() + (1 + step) * 2.0**-bits * size + smallest
    off = (got.double() - want).abs()
    assert got.shape == want.shape and (off <= bound).all(), (what, (off / bound).max().item())


def _operands(present, shape, group, dtype, vec, seed=0, mean=0.5, grad=False):
    g = torch.Generator(device=DEV).manual_seed(seed)
    out = []
    for name in NAMES:
        if name not in present:
            out.append(None)
            continue
        s = shape if name in "xy" else (shape[-1],) if name in ("weight", "bias", "post_weight") or group is None else (*group, shape[-1])
        t = torch.randn(s, generator=g, device=DEV) + (mean if name in "xy" else 1.0 if "weight" in name else 0.1)
        out.append(t.to(dtype if name in "xy" else vec).requires_grad_(grad))
    return out


def _call(x, kind, post, alpha=0.75, eps=1e-5):
    x, y, w, b, sc, sh, gate, pw = x
    if y is None:
        return (norms.norm(x, w, b, scale=sc, shift=sh, kind=kind, eps=eps),)
    if kind is None:
        return (norms.residual(x, y, gate=gate, post=post, post_weight=pw, alpha=alpha, eps=eps),)
    return norms.residual_norm(x, y, w, b, scale=sc, shift=sh, gate=gate, post=post, post_weight=pw, alpha=alpha, kind=kind, eps=eps)


def _options(kind, post, has_y, alpha=0.75, eps=1e-5):
    return norms.NORMS[kind], norms.NORMS[post], alpha if has_y else 1.0, eps, "norm"


NORM = {"x", "weight", "bias", "scale", "shift"}
CASES = [
    # present, shape, group, kind, post
    ({"x"}, (1, 1, 1), None, "rms", None),
    ({"x", "weight"}, (1, 8), None, "rms", None),
    (NORM, (3, 5, 64), (3, 1), "layer", None),
    ({"x", "scale"}, (2, 7, 33), (2, 1), "layer", None),
    ({"x", "shift", "bias"}, (2, 3, 5, 256), (2, 3, 1), "rms", None),
    ({"x", "weight", "scale", "shift"}, (4, 6, 257), (4, 6), "layer", None),
    ({"x", "weight", "scale"}, (70, 3, 40), (70, 1), "rms", None),
    ({"x", "weight"}, (37, 1366), None, "rms", None),
    ({"x", "weight", "bias"}, (9, 4096), None, "layer", None),
    ({"x", "weight", "bias"}, (3, 8191), None, "layer", None),
    ({"x", "y", "gate"}, (3, 17, 96), (3, 1), None, None),
    ({"x", "y"}, (5, 100), None, None, None),
    ({"x", "y", "post_weight", "gate"}, (2, 9, 1000), (2, 1), None, "layer"),
    (ALL, (4, 33, 264), (4, 1), "layer", "rms"),
    (ALL, (2, 300, 1024), (2, 1), "rms", "layer"),
    (ALL, (2, 2, 2731), None, "layer", "layer"),
    ({"x", "y", "weight", "post_weight"}, (600, 512), None, "rms", "rms"),
    ({"x", "y", "gate", "scale", "shift"}, (2, 3, 4104), (2, 1), "layer", None),
    (ALL, (2, 1, 16384), (2, 1), "layer", "rms"),
    ({"x", "y", "weight", "gate"}, (1, 3, 16383), None, "rms", None),
    (ALL, (300, 5, 48), (300, 1), "layer", "rms"),  # more groups than SMs
    ({"x", "y", "gate", "scale", "bias"}, (400, 72), (400,), "layer", "layer"),  # every row vectors of its own
    ({"x", "weight", "shift"}, (150, 2, 1032), (150, 1), "rms", None),
    ({"x", "y", "post_weight"}, (600, 5710), None, None, "layer"),  # too wide for shared memory, several rows of a CTA at once
    (ALL, (2, 300, 4104), (2, 1), "rms", "layer"),
]


@pytest.mark.parametrize("dt,vec", [("bf16", "bf16"), ("bf16", "fp32"), ("fp16", "fp16"), ("fp32", "fp32")])
@pytest.mark.parametrize("dual", [False, True])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_values_tangents_and_gradients(case, dual, dt, vec):
    present, shape, group, kind, post = CASES[case]
    x = _operands(present, shape, group, DT[dt], DT[vec], case, grad=True)
    tx = _operands(present, shape, group, DT[dt], DT[vec], 100 + case, mean=0.0, grad=True) if dual else [None] * 8
    at = [i for i in range(8) if x[i] is not None]
    options = _options(kind, post, x[1] is not None)

    def f(*xs):
        full = [None] * 8
        for i, t in zip(at, xs):
            full[i] = t
        return _call(full, kind, post)

    g = torch.Generator(device=DEV).manual_seed(7)
    cots = lambda n: [torch.randn(shape, generator=g, device=DEV).to(DT[dt]) for _ in range(n)]  # noqa: E731
    if dual:
        ys, tys = torch.func.jvp(f, tuple(x[i] for i in at), tuple(tx[i] for i in at))
    else:
        ys, tys = f(*(x[i] for i in at)), ()
    gs, gts = cots(len(ys)), cots(len(tys))
    leaves = [x[i] for i in at] + ([tx[i] for i in at] if dual else [])
    grads = torch.autograd.grad((*ys, *tys), leaves, (*gs, *gts), materialize_grads=True)
    where = lambda ts: ([ts[0], ts[1]] if len(ts) == 2 else [None, ts[0]] if x[1] is None else [ts[0], None]) if ts else [None, None]  # noqa: E731
    want, twant, _ = formulas.launch_fwd(x, tx, (), options, False)
    size, dsize, dtsize = formulas.sizes(x, tx, where(gs), where(gts), options)
    for name, got, ref, s in [("r", where(ys)[0], want[0], size["r"]), ("n", where(ys)[1], want[1], size.get("n"))]:
        if got is not None:
            _near(got.detach(), ref, s, 16, name)
    if dual:
        for name, got, ref, s in [("tr", where(tys)[0], twant[0], size["tr"]), ("tn", where(tys)[1], twant[1], size.get("tn"))]:
            if got is not None:
                _near(got.detach(), ref, s, 16, name)
    wanted = formulas.launch_bwd(x, tx, (), None, where(gs), where(gts), options, [True] * 16)
    for k, d in enumerate(grads):
        i = at[k % len(at)]
        s = (dsize if k < len(at) else dtsize)[i]
        _near(d, wanted[i if k < len(at) else 8 + i], s.expand(d.shape), 16 if i < 2 else 15, ("d" if k < len(at) else "dt") + NAMES[i])


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_layouts(dt):
    """Views with any strides, vectors expanded over the batch, broadcast cotangents, rows that begin anywhere."""
    base = torch.randn(4, 10, 6, 131, device=DEV).to(DT[dt])
    sc = torch.randn(1, 1, 128, device=DEV).to(DT[dt]).expand(10, 1, 128)
    for x in (base[0, :, :, :128], base[0, :, :, 3:], base[:, :, 2, 1:129], base.transpose(0, 1)[:, :, 1, :128], base[0].transpose(0, 1)[..., ::2],
              base[0, :, :1, :128].expand(10, 6, 128)):
        x = x[:, :, :66] if x.shape[-1] < 128 else x
        s = sc[..., :x.shape[-1]] if x.shape[0] == 10 else None
        y = norms.norm(x, scale=s, kind="layer", eps=1e-5)
        ops, none = [x, None, None, None, s, None, None, None], [None] * 8
        options = _options("layer", None, False)  # (aligned rows and others are added up in different orders: equal to rounding alone)
        _near(y, formulas.launch_fwd(ops, none, (), options, False)[0][1], formulas.sizes(ops, none, none[:2], none[:2], options)[0]["n"], 16, "n")
        assert y.is_contiguous()
    x = torch.randn(3, 40, 72, device=DEV).to(DT[dt]).requires_grad_()
    (a,) = torch.autograd.grad(norms.norm(x, kind="layer").sum(), x)
    (b,) = torch.autograd.grad(norms.norm(x, kind="layer"), x, torch.ones_like(x))
    assert torch.equal(a, b)


def test_large_means_and_tiny_rows():
    """The variance is about the mean; rows of zeros have the deviation sqrt(eps)."""
    x = 1e4 + torch.randn(64, 1000, device=DEV)
    want = torch.nn.functional.layer_norm(x.double(), (1000,), eps=1e-6)
    # the mean is off by 42 roundings of 2^-24 of 1e4 at most, as is each entry less the mean by one
    assert (norms.norm(x, kind="layer").double() - want).abs().max() < 43 * 2.0**-24 * 1.0001e4 * 1.1
    z = torch.zeros(2, 64, device=DEV, requires_grad=True)
    y = norms.norm(z, eps=1e-4)
    (d,) = torch.autograd.grad(y, z, torch.ones_like(y))
    assert not y.any() and torch.allclose(d, torch.full_like(d, 100.0))


def test_nonfinite_rows_stay_alone():
    x, y = torch.randn(6, 500, device=DEV), torch.randn(6, 500, device=DEV)
    x[1, 3], x[4, 499], y[2, 0] = float("nan"), float("inf"), float("-inf")
    r, n = norms.residual_norm(x, y, kind="layer")
    assert [bool(t.isfinite().all()) for t in n] == [True, False, False, True, False, True]
    assert (~r.isfinite()).sum() == 3


@pytest.mark.parametrize("shape", [(0, 16), (3, 0, 16)])
def test_empty(shape):
    x = torch.randn(shape, device=DEV, requires_grad=True)
    w = torch.randn(16, device=DEV, requires_grad=True)
    r, n = norms.residual_norm(x, x.detach(), w)
    dx, dw = torch.autograd.grad((r.sum() + n.sum()), (x, w))
    assert r.shape == n.shape == dx.shape == x.shape and not dw.any()


def test_many_rows_of_one_group():
    """As many rows as a training step has, against float64."""
    x = torch.randn(8192, 64, device=DEV).requires_grad_()
    w = torch.ones(64, device=DEV, requires_grad=True)
    gy = torch.randn(8192, 64, device=DEV)
    dx, dw = torch.autograd.grad(norms.norm(x, w), (x, w), gy)
    x64 = x.detach().double().requires_grad_()
    n = x64 * (x64.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    (rx,) = torch.autograd.grad(n, x64, gy.double())
    terms = (n * gy).abs().sum(0).detach()
    assert (dx.double() - rx).abs().max() < 2.0**-16 * 10
    assert ((dw.double() - (n * gy).sum(0)).abs() <= 2.0**-15 * terms).all()


def test_streams_graphs_and_determinism():
    x, y = (torch.randn(5, 70, 520, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    sc, w = torch.randn(5, 1, 520, device=DEV, dtype=torch.bfloat16, requires_grad=True), torch.randn(520, device=DEV, dtype=torch.bfloat16, requires_grad=True)

    def step():
        r, n = norms.residual_norm(x, y, w, scale=sc, gate=sc, post="rms", kind="layer")
        return (r.detach(), n.detach(), *torch.autograd.grad((r, n), (sc, w), (x, y)))

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
    x += 1
    want = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_second_derivatives():
    """Hessian-vector products and nested transforms against float64, by either route."""
    g = torch.Generator(device=DEV).manual_seed(3)
    x, y, vx = (torch.randn(4, 6, 40, generator=g, device=DEV) for _ in range(3))
    w, sc, gate = (1 + 0.1 * torch.randn(s, generator=g, device=DEV) for s in ((40,), (4, 1, 40), (4, 1, 40)))
    c1, c2 = (torch.randn(4, 6, 40, generator=g, device=DEV) for _ in range(2))
    options = (2, 1, 0.5, 1e-6, "x")

    def own(x, y, w, sc, gate):
        return norms.residual_norm(x, y, w, scale=sc, gate=gate, post="rms", alpha=0.5, kind="layer")

    def exact(x, y, w, sc, gate):
        return formulas._value((x, y, w, None, sc, None, gate, None), *options[:4])

    def loss(f, a):
        r, n = f(*a)
        return (r * c1.to(r.dtype)).sum() + (n * c2.to(n.dtype)).sum() + (n**3).sum()

    results = []
    for f, kind in ((own, torch.float32), (exact, torch.float64)):
        a = [t.to(kind).requires_grad_() for t in (x, y, w, sc, gate)]
        grads = torch.autograd.grad(loss(f, a), a, create_graph=True)
        v = vx.to(kind)
        hv = torch.autograd.grad((grads[0] * v).sum() + (grads[2] * v[0, 0]).sum() + (grads[4] * v[:, :1]).sum(), a)
        plain = [t.detach() for t in a]
        fr = torch.func.jvp(torch.func.grad(lambda *p: loss(f, p), argnums=(0, 1, 2)), tuple(plain), tuple(t.roll(1, -1) for t in plain))
        rr = torch.func.grad(lambda p: (torch.func.grad(lambda q: loss(f, (q, *plain[1:])))(p) * v).sum())(plain[0])
        results.append((*grads, *hv, *fr[0], *fr[1], rr))
    for got, want in zip(*results):
        # sums of some hundred terms of either sign in 32 bits, several times over: 2^-24 * 256, of the largest entry
        assert (got.double() - want).abs().max() <= 2.0**-14 * want.abs().max()


def test_refusals():
    x = torch.randn(4, 8, device=DEV, requires_grad=True)
    w = torch.randn(8, device=DEV)
    cases = [
        (TypeError, dict(x=x.double())), (TypeError, dict(weight=w.half())), (ValueError, dict(weight=w[:7])), (ValueError, dict(scale=torch.randn(3, 8, device=DEV))),
        (TypeError, dict(weight=w, bias=w.double())), (ValueError, dict(kind="mean")), (ValueError, dict(kind=None)), (ValueError, dict(weight=w.cpu())),
        (ValueError, dict(x=torch.randn(2, 16385, device=DEV))), (ValueError, dict(x=torch.randn(2, 0, device=DEV))),
    ]
    for error, kw in cases:
        with pytest.raises(error):
            norms.norm(**{"x": x, **kw})
    for error, kw in [(ValueError, dict(y=x[:3])), (TypeError, dict(y=x.half())), (ValueError, dict(y=x.cpu())), (ValueError, dict(post="x"))]:
        with pytest.raises(error):
            norms.residual(**{"x": x, "y": x, **kw})
    with pytest.raises(NotImplementedError, match="no rule for"):
        torch.func.vmap(lambda v: norms.norm(v))(x.detach())
    n = norms.norm(x)
    with pytest.raises(NotImplementedError, match="no rule for"):
        torch.autograd.grad(n, x, torch.randn(3, 4, 8, device=DEV), is_grads_batched=True, retain_graph=True)
    (d,) = torch.autograd.grad(n.square().sum(), x, create_graph=True)
    (d2,) = torch.autograd.grad(d.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="no third derivative"):
        torch.autograd.grad(d2.sum(), x)
    with pytest.raises(RuntimeError, match="further forward"):
        torch.func.jvp(lambda a: torch.func.jvp(norms.norm, (a,), (a,))[1], (x.detach(),), (x.detach(),))
