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
