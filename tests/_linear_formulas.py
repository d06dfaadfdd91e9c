"""Test helper: linear attention from its definition in float64, every pair of rows by its weight, for the oracle side of the GPU tests and as
stand-ins for the launches in the CPU suite.  Only tests may use this.

Operands in the order q, k, v, state (None: absent); extras log_decay, lengths; options sm_scale, return_state, name."""
import torch


class Weights:
    """(B, H, L, L) weights of pairs, (B, H, L, 1) of the given state at each row and of each row in the last state, (B, H, 1, 1) of the given
    state in the last one; rows behind a sequence's end have none."""

    def __init__(self, q, extras):
        B, H, L, _ = q.shape
        w, n = extras
        w = torch.zeros(H, dtype=torch.float64, device=q.device) if w is None else w.double().clamp(min=-1e4)
        n = torch.full((B,), L, device=q.device) if n is None else n.long().clamp(0, L)
        t = torch.arange(L, device=q.device)
        self.live = live = (t < n[:, None])[:, None, :, None]
        w = w[None, :, None, None]
        apart = (t[:, None] - t).double()
        self.pairs = torch.where((apart >= 0) & live & live.transpose(-1, -2), torch.exp(w * apart.clamp(min=0)), 0.0)
        self.old = torch.where(live, torch.exp(w * (t + 1)[:, None]), 0.0)
        left = (n[:, None] - 1 - t)[:, None, :, None]
        self.last = torch.where(live, torch.exp(w * left.clamp(min=0)), 0.0)
        self.kept = torch.exp(w * n[:, None, None, None])


def value(q, k, v, state, W, scale):
    """(o, last state)."""
    o = scale * (((q @ k.transpose(-1, -2)) * W.pairs) @ v)
    last = (k * W.last).transpose(-1, -2) @ v
    if state is not None:
        o = o + scale * W.old * (q @ state)
        last = last + W.kept * state
    return o, last


def clean(x, W):
    """Without what stands behind the sequences' ends."""
    return [None if t is None else torch.where(W.live, t.double(), 0.0) if i < 3 else t.double() for i, t in enumerate(x)]


def _tangents(x, tx):
    return [None if v is None else torch.zeros_like(v) if t is None else t for v, t in zip(x, tx or [None] * 4)]


def launch_fwd(x, tx, extras, options, keep):
    """(y, ty, kept) as ``linear_attention._launch_fwd`` answers."""
    x = [None if t is None else t.detach() for t in x]
    W, scale = Weights(x[0], extras), options[0]
    f = lambda *a: value(*a, W, scale)  # noqa: E731
    dual = any(t is not None for t in tx)
    x, tx = clean(x, W), clean(_tangents(x, tx), W)
    q, k, v, s = x
    y = f(*x)
    ty = None
    if dual:
        tq, tk, tv, ts = tx
        zero = None if s is None else torch.zeros_like(s)
        parts = (f(tq, k, v, s), f(q, tk, v, zero), f(q, k, tv, zero), f(q, k * 0, v, ts))
        ty = [sum(p[0] for p in parts), sum(p[1] for p in parts[1:])]
    only = lambda t: [t[0], t[1] if options[1] else None]  # noqa: E731
    return only(y), (only(ty) if dual else None), torch.zeros(1)


def _grads(q, k, v, s, g, gs, W, scale):
    """Gradients of <g, o> + <gs, last>."""
    A, dA = scale * (q @ k.transpose(-1, -2)) * W.pairs, scale * (g @ v.transpose(-1, -2)) * W.pairs
    dq, dk, dv, ds = dA @ k, dA.transpose(-1, -2) @ q, A.transpose(-1, -2) @ g, None
    dk = dk + W.last * (v @ gs.transpose(-1, -2))
    dv = dv + W.last * (k @ gs)
    if s is not None:
        dq = dq + scale * W.old * (g @ s.transpose(-1, -2))
        ds = scale * (W.old * q).transpose(-1, -2) @ g + W.kept * gs
    return [dq, dk, dv, ds]


def launch_bwd(x, tx, extras, kept, g, gt, options, want):
    """Gradients as ``linear_attention._launch_bwd`` answers: the derivative is linear in each operand, so the gradients through the tangent are
    sums of the value's with one operand replaced by its tangent."""
    x = [None if t is None else t.detach() for t in x]
    W, scale = Weights(x[0], extras), options[0]
    tx = clean(_tangents(x, tx), W)
    x = clean(x, W)
    q, k, v, s = x

    def cotangents(c):
        o, last = value(q, k, v, s, W, scale)
        return [torch.zeros_like(z) if t is None else t.detach().double() for t, z in zip(c, (o, last))]

    (g, gs), (h, hs) = cotangents(g), cotangents(gt)
    h, g = (torch.where(W.live, c, 0.0) for c in (h, g))
    zero = [None if t is None else torch.zeros_like(t) for t in x]
    d, dt = _grads(*x, g, gs, W, scale), _grads(*x, h, hs, W, scale)
    for i in range(4):  # <h, ty> has the terms with one operand's tangent; of each, the gradients with respect to the other operands
        if x[i] is None:
            continue
        y = list(x)
        y[i] = tx[i]
        if i == 3:  # the state's term goes without the pairs
            part = _grads(q, k, v, tx[3], h, hs, W, scale)
            base = _grads(q, k, v, zero[3], h, hs, W, scale)
            d[0] = d[0] + part[0] - base[0]
            continue
        part = _grads(*y, h, hs, W, scale)
        if i == 0:
            d[1], d[2] = d[1] + part[1] - _last(y, hs, W)[0], d[2] + part[2] - _last(y, hs, W)[1]
            if s is not None:
                d[3] = d[3] + part[3] - W.kept * hs
        else:
            other = 2 if i == 1 else 1
            base = _grads(*[*y[:3], zero[3]], h, hs, W, scale)
            d[0], d[other] = d[0] + base[0], d[other] + base[other]
    out = [t if w else None for t, w in zip((*d, *dt), want)]
    return [None if t is None else t.clone() for t in out]


def _last(y, hs, W):
    """What of dk and dv goes through the last state, which q has no part in."""
    return W.last * (y[2] @ hs.transpose(-1, -2)), W.last * (y[1] @ hs)
