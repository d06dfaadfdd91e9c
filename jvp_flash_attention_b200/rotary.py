"""Rotary positions for the queries and keys of ``JVPAttn``, with their tangents (csrc/rotary.cu).

``rotary`` turns q and k in one launch; where they carry tangents (``torch.func.jvp``, forward-AD dual tensors) the tangents are turned
in the same launch, as the map is linear.  Its gradient is the transposed turn, for values and tangents alike, and can be
differentiated any number of times.  ``rotary_frequencies`` makes the frequencies.  No upstream counterpart: upstream leaves
positions to the model.
"""
from __future__ import annotations

import ctypes as C
import math

import torch
from torch import Tensor
from torch.autograd import Function

from . import _lib
from .jvp_attention import _JVP, _is_tracing, _peek_functorch, _require_cuda, _unwrap

_POSITION_DTYPES = (torch.int32, torch.int64)


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: str | None = None, factor: float = 1.0,
                       original_length: int = 4096, quick: float = 32.0, slow: float = 1.0, device=None) -> Tensor:
    """Radians per position of the ``rotary_dim / 2`` pairs, ``base ** (-2 i / rotary_dim)``, in 64 bits.

    ``scaling`` stretches a context that the model was trained on, ``original_length`` positions, by ``factor``:

    * ``None``: none
    * ``"linear"``: every frequency divided by ``factor``
    * ``"base"``: a larger base, with which the slowest pair turns ``factor`` times slower and the quickest as before
    * ``"ramp"``: pairs of at least ``quick`` turns in ``original_length`` positions as they are, those of at most ``slow`` divided by
      ``factor``, and between the two a mixture that is linear in the pair's index (YaRN)
    * ``"bands"``: the same two ends, and between them a mixture that is linear in the number of turns
    """
    if rotary_dim < 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim has to be even and not negative, got {rotary_dim}")
    if not base > 0 or not factor > 0 or original_length < 1:
        raise ValueError("base, factor and original_length have to be positive")
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device)
    if scaling == "base" and rotary_dim > 2:
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    w = base ** (-i / max(rotary_dim, 1))
    if scaling in (None, "base"):
        return w
    if scaling == "linear":
        return w / factor
    if scaling not in ("ramp", "bands"):
        raise ValueError("scaling is None, 'linear', 'base', 'ramp' or 'bands'")
    if not quick > slow > 0 or not base > 1:
        raise ValueError("quick has to be above slow, slow positive and base above 1")
    if scaling == "bands":
        keep = (original_length * w / (2 * math.pi) - slow) / (quick - slow)
    else:
        # the pair index at which a pair makes so many turns in the original context, widened to whole indices
        at = lambda turns: rotary_dim * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        low, high = max(math.floor(at(quick)), 0), min(math.ceil(at(slow)), rotary_dim - 1)
        keep = 1 - (i / 2 - low) / max(high - low, 1e-3)
    keep = keep.clamp(0, 1)
    return w * keep + w / factor * (1 - keep)


def rotary(q: Tensor, k: Tensor | None, inv_freq: Tensor, positions: Tensor | None = None, *, offset: int = 0,
           interleaved: bool = False, amplitude: float = 1.0):
    """``(q, k)`` with every pair of the first ``2 * len(inv_freq)`` entries of a head turned by its position; ``q`` alone for ``k=None``.

    q: (B, H, L, D), k: (B, H', L, D), bfloat16, float16 or float32, of any strides; plain or dual.  What is not turned is copied.
    The results have the layout of q and k: the (B, H, L, D) view of a (B, L, H, D) tensor stays one, which ``attention`` reads in
    place.
    ``inv_freq``: radians per position, a float64 tensor (``rotary_frequencies``).  ``positions``: int32 or int64, (L), (1, L) or (B, L), of any
    sign and below 2**53; by default ``offset + [0 .. L)``.
    ``interleaved``: pair i is entries (2 i, 2 i + 1) instead of (i, len(inv_freq) + i).  ``amplitude`` multiplies what is turned.
    Angles are formed in 64 bits, so far positions lose nothing.
    """
    interp = _peek_functorch()
    if (interp is None or (interp.level() == 1 and interp.key() == _JVP)) and not _is_tracing():
        if not q.is_cuda:  # (the native layer checks CUDA tensors itself)
            _check(q, k, inv_freq, positions)
        out = _lib.native().rotary(q, k, inv_freq, positions, offset, interleaved, amplitude)
        if out is not None:
            return out
    _check(q, k, inv_freq, positions)
    return _general(q, k, inv_freq, positions, offset, interleaved, amplitude)


def _check(q, k, inv_freq, positions) -> None:
    for name, x in (("q", q), ("k", k)):
        if x is None:
            continue
        if x.dim() != 4:
            raise ValueError(f"{name} must have 4 dimensions (B, H, L, D), got {tuple(x.shape)}")
        if max(x.shape) >= 2**31:
            raise ValueError(f"{name} must have less than 2**31 entries along each dimension, got {tuple(x.shape)}")
        if x.dtype not in _lib.DTYPE_ENUM and x.is_cuda:
            raise TypeError(f"unsupported dtype {x.dtype} of {name}; expected bfloat16, float16 or float32")
        if x.dtype != q.dtype:
            raise TypeError(f"q and k must have one dtype, got {q.dtype} and {x.dtype}")
        if x.device != q.device:
            raise ValueError(f"q and k must be on one device, got {q.device} and {x.device}")
        if (x.shape[0], *x.shape[2:]) != (q.shape[0], *q.shape[2:]):
            raise ValueError(f"q and k must agree in all dimensions but the heads, got {tuple(q.shape)} and {tuple(x.shape)}")
    B, _, L, D = q.shape
    if inv_freq.dim() != 1 or inv_freq.dtype != torch.float64:
        raise TypeError(f"inv_freq must be a float64 vector (angles are formed in 64 bits), got {inv_freq.dtype} {tuple(inv_freq.shape)}")
    if not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be contiguous")
    if 2 * inv_freq.shape[0] > D:
        raise ValueError(f"{inv_freq.shape[0]} pairs do not fit a head of {D}")
    if inv_freq.requires_grad:
        raise NotImplementedError("rotary has no gradient with respect to inv_freq; pass inv_freq.detach()")
    if positions is not None:
        if positions.dtype not in _POSITION_DTYPES:
            raise TypeError(f"positions must be int32 or int64, got {positions.dtype}")
        if tuple(positions.shape) not in ((L,), (1, L), (B, L)):
            raise ValueError(f"positions must have the shape (L,), (1, L) or (B, L) with B={B} and L={L}, got {tuple(positions.shape)}")
    for name, x in (("inv_freq", inv_freq), ("positions", positions)):
        if x is not None and x.device != q.device:
            raise ValueError(f"{name} must be on {q.device} like q, got {x.device}")
    _require_cuda(q)


def _in_memory(t):
    """The plain tensor in memory: torch keeps some zeros as a shape alone."""
    return torch.zeros(t.shape, dtype=t.dtype, device=t.device) if t._is_zerotensor() else t


def _launch(x, inv_freq, positions, offset, interleaved, amplitude, transposed):
    """Runs jvpfa_rotary on one plain tensor and returns the result."""
    x = _in_memory(x)
    if x.stride(-1) != 1:
        x = x.contiguous()
    y = torch.empty_like(x)
    if y.numel() == 0:
        return y
    if y.stride(-1) != 1:
        y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    a = _lib.RotaryArgs()
    a.struct_size = C.sizeof(_lib.RotaryArgs)
    a.dtype = _lib.DTYPE_ENUM[x.dtype]
    a.B, _, a.L, a.D = x.shape
    a.n_freq = inv_freq.shape[0]
    a.n_tensors = 1
    a.interleaved, a.transposed = int(interleaved), int(transposed)
    a.amplitude = amplitude
    a.freq = inv_freq.data_ptr()
    a.offset = offset
    if positions is not None:
        a.positions = positions.data_ptr()
        a.position_bits = 64 if positions.dtype == torch.int64 else 32
        a.position_stride[0] = positions.stride(0) if positions.dim() == 2 and positions.shape[0] > 1 else 0
        a.position_stride[1] = positions.stride(-1)
    a.t[0].x, a.t[0].y, a.t[0].H = x.data_ptr(), y.data_ptr(), x.shape[1]
    for d in range(3):
        a.t[0].x_stride[d], a.t[0].y_stride[d] = x.stride(d), y.stride(d)
    _lib.check(_lib._launch(x, _lib.load().jvpfa_rotary, a), "jvpfa_rotary")
    return y


class _Rotary(Function):
    """One tensor's turn on the general route (functorch transforms other than a lone ``torch.func.jvp``).  Linear: its jvp and its
    backward are turns again."""

    @staticmethod
    def forward(x, inv_freq, positions, offset, interleaved, amplitude, transposed):
        return _launch(_unwrap(x), _unwrap(inv_freq), _unwrap(positions), offset, interleaved, amplitude, transposed)

    @staticmethod
    def setup_context(ctx, inputs, output):
        _, inv_freq, positions, *ctx.turn = inputs
        ctx.save_for_backward(inv_freq, positions)
        ctx.save_for_forward(inv_freq, positions)

    @staticmethod
    def jvp(ctx, tx, *_):
        return _Rotary.apply(tx, *ctx.saved_tensors, *ctx.turn)

    @staticmethod
    def backward(ctx, g):
        *turn, transposed = ctx.turn
        return (_Rotary.apply(g, *ctx.saved_tensors, *turn, not transposed), *(None,) * 6)


_turn = _Rotary.apply  # (the native layer's route to it)


def _general(q, k, inv_freq, positions, offset, interleaved, amplitude):
    out = tuple(None if x is None else _Rotary.apply(x, inv_freq, positions, offset, interleaved, amplitude, False) for x in (q, k))
    return out if k is not None else out[0]
