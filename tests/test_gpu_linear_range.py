"""GPU tests of linear attention where decays are fast and operands of very different size, against its definition in float64.

Bounds as in test_gpu_linear_attention.py: half a step of the result's type, and of the sum of the magnitudes that an entry is made of 2^-11 for
16-bit types and (3 (L / 8 + D / 8 + 8) + 8) 2^-22 for sums in 32 bits.  They hold entry by entry, so nothing may depend on what stands in
other rows, columns or heads.  A decay's exponent w n is off by 2^-24 |w n| and its function by 2^-22, up to three times over (a chunk's, a segment's and a row's):
with |w n| <= 88, as far as 32 bits hold it, 3 (88 + 4) 2^-24 = 2^-15.8 of the sum besides."""
import pytest
import torch

import jvp_flash_attention_b200.linear_attention as la
from tests import _linear_formulas as formulas
from tests.test_gpu_linear_attention import DEV, DT, _bits, _near

pytestmark = pytest.mark.gpu
DECAYS = 3 * (88 + 4) * 2.0**-24


def _hold(x, tx, w, n, cots, tcots, scale=1.0):
    """Values, tangents and gradients of the operands (lists of q, k, v and perhaps a state) against the definition."""
    dual = bool(tx)
    leaf = lambda ts: [t.detach().requires_grad_() for t in ts]  # noqa: E731
    x, tx = leaf(x), leaf(tx)

    def f(q, k, v, s=None):
        return la.linear_attention(q, k, v, w, sm_scale=scale, state=s, lengths=n, return_state=True)

    y, ty = torch.func.jvp(f, tuple(x), tuple(tx)) if dual else (f(*x), ())
    grads = torch.autograd.grad((*y, *ty), (*x, *tx), [*cots, *(tcots if dual else ())], materialize_grads=True)
    full = lambda ts: list(ts) + [None] * (4 - len(ts))  # noqa: E731
    tcots = tcots if dual else [None, None]
    opts, extras = (scale, True, ""), (w, n)
    mag = lambda ts: [None if t is None else t.detach().abs() for t in ts]  # noqa: E731
    want, twant, _ = formulas.launch_fwd(full(x), full(tx), extras, opts, False)
    dwant = formulas.launch_bwd(full(x), full(tx), extras, None, cots, tcots, opts, [True] * 8)
    opts = (abs(scale), True, "")
    size, tsize, _ = formulas.launch_fwd(full(mag(x)), full(mag(tx)), extras, opts, False)
    dsize = formulas.launch_bwd(full(mag(x)), full(mag(tx)), extras, None, mag(cots), mag(tcots), opts, [True] * 8)
    L, D, E = x[0].shape[2], x[0].shape[3], x[2].shape[3]
    exact = _bits(L, max(D, E)) + DECAYS
    outs = exact if x[0].dtype == torch.float32 else exact + 2.0**-11
    _near(y[0].detach(), want[0], size[0], outs, "o")
    _near(y[1].detach(), want[1], size[1], exact, "state")
    if dual:
        _near(ty[0].detach(), twant[0], tsize[0], outs, "to")
        _near(ty[1].detach(), twant[1], tsize[1], exact, "tstate")
    m = len(x)
    for i, d in enumerate(grads):
        at = i if i < m else 4 + i - m
        _near(d, dwant[at], dsize[at], exact if at % 4 == 3 else outs, f"gradient {at}")


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("dual", [False, True])
@pytest.mark.parametrize("D,E,L", [(64, 64, 130), (32, 16, 64), (128, 128, 100), (33, 64, 190)])
def test_few_rows_and_fast_decays(D, E, L, dual, dt):
    """Keys in the first row of each chunk alone, cotangents in the last ones alone: all that is left has been decayed 64 rows long."""
    g = torch.Generator(device=DEV).manual_seed(D)
    w = torch.tensor([-0.25, -0.3, -0.5, -1.0, -1.2], device=DEV)
    B, H = 1, len(w)
    first, last = (torch.arange(L, device=DEV) % 64 == 0).float()[:, None], ((torch.arange(L, device=DEV) % 64 == 63) | (torch.arange(L, device=DEV) == L - 1)).float()[:, None]
    make = lambda: [_randn(g, B, H, L, D).to(DT[dt]), (_randn(g, B, H, L, D) * first).to(DT[dt]), _randn(g, B, H, L, E).to(DT[dt]), _randn(g, B, H, D, E)]  # noqa: E731
    cots = lambda: [(_randn(g, B, H, L, E) * last).to(DT[dt]), _randn(g, B, H, D, E)]  # noqa: E731
    _hold(make(), make() if dual else [], w, None, cots(), cots(), 0.3)


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("dual", [False, True])
@pytest.mark.parametrize("D,E", [(64, 64), (128, 40)])
def test_rows_and_columns_of_any_size(D, E, dual, dt):
    """Each row of q and each column of v, and of the cotangents likewise, of a size of its own."""
    g = torch.Generator(device=DEV).manual_seed(D + 1)
    B, H, L = 1, 2, 150
    most = 5 if dt == "fp16" else 25
    w = torch.tensor([0.0, -0.02], device=DEV)

    def sizes(*shape):
        return torch.exp2(torch.randint(-most, most + 1, shape, generator=g, device=DEV).float())

    rows, columns, channels = sizes(B, H, L, 1), sizes(B, H, 1, E), sizes(B, H, 1, D)
    make = lambda: [(_randn(g, B, H, L, D) * rows / channels).to(DT[dt]), (_randn(g, B, H, L, D) * channels).to(DT[dt]), (_randn(g, B, H, L, E) * columns).to(DT[dt])]  # noqa: E731
    cots = lambda: [(_randn(g, B, H, L, E) / rows / columns).to(DT[dt]), _randn(g, B, H, D, E)]  # noqa: E731
    _hold(make(), make() if dual else [], w, None, cots(), cots(), 2.0**-8 if dt == "fp16" else 1.0)  # (2^17 is beyond fp16)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_small_operands(dt):
    """Products of two operands near the lower end of 32 bits, brought back by the third."""
    g = torch.Generator(device=DEV).manual_seed(3)
    B, H, L, D = 1, 2, 130, 64
    w = torch.tensor([0.0, -0.05], device=DEV)
    for a, b, c in ((-55, -55, 60), (60, -55, -55), (-55, 60, -55)):
        x = [(_randn(g, B, H, L, D) * 2.0**k).to(DT[dt]) for k in (a, b, c)]
        o, s = la.linear_attention(*x, w, sm_scale=1.0, return_state=True)
        args = ((w, None), (1.0, True, ""), False)
        want, _, _ = formulas.launch_fwd([*x, None], [None] * 4, *args)
        size, _, _ = formulas.launch_fwd([*(t.abs() for t in x), None], [None] * 4, *args)
        exact = _bits(L, D) + DECAYS
        # (split numbers keep 2^-133 of their last digits at the lower end: of 2^-110, what a product has, 2^-23)
        _near(o, want[0], size[0], exact + (2.0**-11 if dt == "bf16" else 0), "o")
        _near(s, want[1], size[1], exact, "state")
