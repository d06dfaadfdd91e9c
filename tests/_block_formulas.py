"""Test helper: rotary positions and the gated projection from their formulas in float64, for the oracle side of the GPU tests and
as stand-ins for the launches in the CPU suite.  Only tests may use this."""
import torch


def turn(x, inv_freq, positions=None, offset=0, interleaved=False, amplitude=1.0, transposed=False):
    """Pairs as complex numbers, times amplitude * exp(i position frequency)."""
    B, _, L, _ = x.shape
    p = torch.arange(L, device=x.device) + offset if positions is None else positions
    angle = p.double()[..., None] * inv_freq
    by = torch.polar(torch.full_like(angle, amplitude), -angle if transposed else angle)
    by = by[:, None] if by.dim() == 3 else by
    n = inv_freq.shape[0]
    z = x.double()
    a, b = (z[..., 0:2 * n:2], z[..., 1:2 * n:2]) if interleaved else (z[..., :n], z[..., n:2 * n])
    c = torch.complex(a, b) * by
    pair = torch.stack((c.real, c.imag), -1).flatten(-2) if interleaved else torch.cat((c.real, c.imag), -1)
    return torch.cat((pair, z[..., 2 * n:]), -1)


def pair_norm(x, n, interleaved):
    """The length of the pair that each entry belongs to (0 for those that are not turned)."""
    z = x.double()
    a, b = (z[..., 0:2 * n:2], z[..., 1:2 * n:2]) if interleaved else (z[..., :n], z[..., n:2 * n])
    r = torch.hypot(a, b)
    r = torch.stack((r, r), -1).flatten(-2) if interleaved else torch.cat((r, r), -1)
    return torch.cat((r, torch.zeros_like(z[..., 2 * n:])), -1)


def activation(kind, g):
    """a, a', a'' of jvpfa_activation ``kind`` at g."""
    if kind in (0, 1):
        s, r = torch.sigmoid(g), torch.sigmoid(-g)
        d = s * r
        return (s, d, d * (r - s)) if kind == 1 else (g * s, s + g * d, d * (2 + g * (r - s)))
    if kind == 2:
        p, d = torch.special.ndtr(g), torch.exp(-0.5 * g * g) * (2 * torch.pi) ** -0.5
        return g * p, p + g * d, d * (2 - g * g)
    c, c3 = (2 / torch.pi) ** 0.5, 0.044715
    s, r = torch.sigmoid(2 * c * (g + c3 * g**3)), torch.sigmoid(-2 * c * (g + c3 * g**3))
    z1, z2, d = 2 * c * (1 + 3 * c3 * g * g), 12 * c * c3 * g, s * r
    return g * s, s + g * d * z1, d * (2 * z1 + g * (z2 + (r - s) * z1 * z1))


def gated_fwd(x, tx, w_gate, w_up, kind, keep=True):
    """(h, th, g, u, tg, tu) as ``gated._launch_fwd`` returns them."""
    x, tx, w_gate, w_up = (None if t is None else t.double() for t in (x, tx, w_gate, w_up))
    g, u = x @ w_gate.T, x @ w_up.T
    a, a1, _ = activation(kind, g)
    if tx is None:
        return (a * u, None, *((g, u) if keep else (None, None)), None, None)
    tg, tu = tx @ w_gate.T, tx @ w_up.T
    return (a * u, a1 * tg * u + a * tu, *((g, u, tg, tu) if keep else (None,) * 4))


def gated_bwd(x, tx, w_gate, w_up, g, u, tg, tu, gh, gth, kind, need_x=True, need_tx=True, need_w=True):
    """(dx, dtx, dwg, dwu) as ``gated._launch_bwd`` returns them."""
    x, tx, w_gate, w_up, g, u, tg, tu, gh, gth = (None if t is None else t.double() for t in (x, tx, w_gate, w_up, g, u, tg, tu, gh, gth))
    a, a1, a2 = activation(kind, g)
    dg, du = (torch.zeros_like(g), torch.zeros_like(g)) if gh is None else (gh * a1 * u, gh * a)
    dtg = dtu = None
    if gth is not None:
        dg, du = dg + gth * (a2 * tg * u + a1 * tu), du + gth * a1 * tg
        dtg, dtu = gth * a1 * u, gth * a
    flat = lambda t: t.reshape(-1, t.shape[-1])  # noqa: E731
    dx = dg @ w_gate + du @ w_up if need_x else None
    dtx = dtg @ w_gate + dtu @ w_up if need_tx and gth is not None else None
    dwg, dwu = (flat(d).T @ flat(x) for d in (dg, du)) if need_w else (None, None)
    if need_w and gth is not None:
        dwg, dwu = dwg + flat(dtg).T @ flat(tx), dwu + flat(dtu).T @ flat(tx)
    return dx, dtx, dwg, dwu


def launch_gated_fwd(x, tx, w_gate, w_up, kind, keep):
    """Stand-in for ``gated._launch_fwd``."""
    h, th, *projections = gated_fwd(x, tx, w_gate, w_up, kind)
    return h, th, torch.stack([t for t in projections if t is not None]) if keep else None


def launch_gated_bwd(x, tx, w_gate, w_up, kept, *args):
    """Stand-in for ``gated._launch_bwd``."""
    assert kept.shape[0] == (2 if tx is None else 4)
    return gated_bwd(x, tx, w_gate, w_up, *(*kept, None, None)[:4], *args)
