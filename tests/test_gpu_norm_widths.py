"""GPU tests of the norms' gradients at widths where another kernel takes over, several rows of each of a launch's CTAs.

Bounds as in test_gpu_norms.py: half a step of the type and 2^-16 of the magnitudes that an entry is made of; of a vector's gradient 2^-15, here a
sum of at most 400 / 148 rows of a CTA, 148 / 32 slices and 32 lanes, with tangents twice as many terms."""
import pytest
import torch

from tests import _norm_formulas as formulas
from tests.test_gpu_norms import ALL, DEV, DT, NAMES, _call, _near, _operands, _options

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("dual", [False, True])
@pytest.mark.parametrize("present", [{"x", "weight", "bias"}, {"x", "y", "gate"}, ALL])
@pytest.mark.parametrize("C", [4097, 4104, 6144, 8191, 8192, 8193, 8200])
def test_gradients(C, present, dual, dt):
    kind, post = (None, "rms") if present == {"x", "y", "gate"} else ("layer", "rms" if "y" in present else None)
    shape, group = (2, 200, C), (2, 1)
    x = _operands(present, shape, group, DT[dt], DT[dt], C, grad=True)
    tx = _operands(present, shape, group, DT[dt], DT[dt], C + 1, mean=0.0, grad=True) if dual else [None] * 8
    at = [i for i in range(8) if x[i] is not None]
    options = _options(kind, post, x[1] is not None)

    def f(*xs):
        full = [None] * 8
        for i, t in zip(at, xs):
            full[i] = t
        return _call(full, kind, post)

    ys, tys = torch.func.jvp(f, tuple(x[i] for i in at), tuple(tx[i] for i in at)) if dual else (f(*(x[i] for i in at)), ())
    g = torch.Generator(device=DEV).manual_seed(7)
    gs, gts = ([torch.randn(shape, generator=g, device=DEV).to(DT[dt]) for _ in ts] for ts in (ys, tys))
    leaves = [x[i] for i in at] + ([tx[i] for i in at] if dual else [])
    grads = torch.autograd.grad((*ys, *tys), leaves, (*gs, *gts), materialize_grads=True)
    where = lambda ts: ([ts[0], ts[1]] if len(ts) == 2 else [None, ts[0]] if x[1] is None else [ts[0], None]) if ts else [None, None]  # noqa: E731
    _, dsize, dtsize = formulas.sizes(x, tx, where(gs), where(gts), options)
    wanted = formulas.launch_bwd(x, tx, (), None, where(gs), where(gts), options, [True] * 16)
    for k, d in enumerate(grads):
        i = at[k % len(at)]
        s = (dsize if k < len(at) else dtsize)[i]
        _near(d, wanted[i if k < len(at) else 8 + i], s.expand(d.shape), 16 if i < 2 else 15, ("d" if k < len(at) else "dt") + NAMES[i])


@pytest.mark.parametrize("dual", [False, True])
def test_many_groups(dual):
    """Several thousand groups with vectors of their own, and others of all rows.  The sum over rows goes by 3 rows, the groups of one of
    64 parts (at most 4000 / 64 one after the other, by the lanes that take turns with them fewer), and these: with the magnitudes of a row (2^-16) and at
    most 130 roundings of 2^-24, 2^-15."""
    present, shape, group = {"x", "y", "weight", "bias", "scale", "gate", "post_weight"}, (4000, 3, 72), (4000, 1)
    x = _operands(present, shape, group, torch.float32, torch.float32, 1, grad=True)
    tx = _operands(present, shape, group, torch.float32, torch.float32, 2, mean=0.0, grad=True) if dual else [None] * 8
    at = [i for i in range(8) if x[i] is not None]

    def f(*xs):
        full = [None] * 8
        for i, t in zip(at, xs):
            full[i] = t
        return _call(full, "layer", "rms")

    ys, tys = torch.func.jvp(f, tuple(x[i] for i in at), tuple(tx[i] for i in at)) if dual else (f(*(x[i] for i in at)), ())
    g = torch.Generator(device=DEV).manual_seed(3)
    gs, gts = ([torch.randn(shape, generator=g, device=DEV) for _ in ts] for ts in (ys, tys))
    leaves = [x[i] for i in at] + ([tx[i] for i in at] if dual else [])
    grads = torch.autograd.grad((*ys, *tys), leaves, (*gs, *gts), materialize_grads=True)
    options, gts = _options("layer", "rms", True), list(gts) or [None, None]
    _, dsize, dtsize = formulas.sizes(x, tx, list(gs), gts, options)
    wanted = formulas.launch_bwd(x, tx, (), None, list(gs), gts, options, [True] * 16)
    for k, d in enumerate(grads):
        i = at[k % len(at)]
        s = (dsize if k < len(at) else dtsize)[i]
        _near(d, wanted[i if k < len(at) else 8 + i], s.expand(d.shape), 16 if i < 2 else 15, ("d" if k < len(at) else "dt") + NAMES[i])


@pytest.mark.parametrize("dual", [False, True])
@pytest.mark.parametrize("groups,rows,C", [(3, 1, 40), (33, 2, 72), (65, 9, 33), (148, 1, 520), (149, 4, 40), (2049, 1, 72)])
def test_groups_beside_vectors_of_all_rows(groups, rows, C, dual):
    """As many slices of a group and groups at once as there are.  At most 148 rows and slices of a group, and 2049 / 64 groups and 64 parts of them: 2^-15."""
    present, shape, group = {"x", "weight", "scale", "shift"}, (groups, rows, C), (groups, 1)
    x = _operands(present, shape, group, torch.float32, torch.float32, 1, grad=True)
    tx = _operands(present, shape, group, torch.float32, torch.float32, 2, mean=0.0, grad=True) if dual else [None] * 8
    at = [i for i in range(8) if x[i] is not None]

    def f(*xs):
        full = [None] * 8
        for i, t in zip(at, xs):
            full[i] = t
        return _call(full, "layer", None)

    ys, tys = torch.func.jvp(f, tuple(x[i] for i in at), tuple(tx[i] for i in at)) if dual else (f(*(x[i] for i in at)), ())
    g = torch.Generator(device=DEV).manual_seed(3)
    gs, gts = ([torch.randn(shape, generator=g, device=DEV) for _ in ts] for ts in (ys, tys))
    leaves = [x[i] for i in at] + ([tx[i] for i in at] if dual else [])
    grads = torch.autograd.grad((*ys, *tys), leaves, (*gs, *gts), materialize_grads=True)
    options, pair = _options("layer", None, False), ([None, *gs], [None, *gts] if dual else [None, None])
    _, dsize, dtsize = formulas.sizes(x, tx, *pair, options)
    wanted = formulas.launch_bwd(x, tx, (), None, *pair, options, [True] * 16)
    for k, d in enumerate(grads):
        i = at[k % len(at)]
        s = (dsize if k < len(at) else dtsize)[i]
        _near(d, wanted[i if k < len(at) else 8 + i], s.expand(d.shape), 16 if i < 2 else 15, ("d" if k < len(at) else "dt") + NAMES[i])
