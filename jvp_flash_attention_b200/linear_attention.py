"""Causal linear attention with a decay for each head, and its tangent (csrc/linear.cu): attention whose cost grows with the length of a sequence
and not with its square, and whose past is one matrix of each head,

    S_t = exp(log_decay) S_{t-1} + k_t v_t^T        o_t = sm_scale * S_t^T q_t

``linear_attention`` takes whole sequences, in chunks on the tensor cores, and may begin with a state and answer the last one;
``linear_attention_step`` takes one more token of each sequence and updates the states in place.  Where operands carry tangents
(``torch.func.jvp``, forward-AD dual tensors) value and tangent come from one pass, and the gradient goes through both, as with ``JVPAttn.fwd_dual``;
positions are ``rotary``'s.  No upstream counterpart: upstream has softmax attention alone.
"""
from __future__ import annotations

import math
import sys

import torch
import torch.autograd.forward_ad as fwAD
from torch import Tensor

from . import _dual, _lib
from .jvp_attention import _JVP, _is_tracing, _peek_functorch, _require_cuda

MAX_WIDTH = 128
_MIN_SCALE, _MAX_SCALE = 2.0**-64, 2.0**64  # (a last state's cotangent is divided by it, in 32 bits)


def linear_attention(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor | None = None, *, sm_scale: float | None = None, state: Tensor | None = None,
                     lengths: Tensor | None = None, return_state: bool = False):
    """``o`` with ``o_t = sm_scale * sum over s <= t of exp(log_decay (t - s)) (q_t . k_s) v_s``, and with ``return_state`` ``(o, S)``, S the
    state behind the last row.

    q, k: (B, H, L, D), v: (B, H, L, E), bfloat16, float16 or float32, of any strides with contiguous entries, plain or dual; D and E from 1 to 128,
    fastest at 32, 64 and 128.  o has v's layout.  ``log_decay``: (H) float32, the logarithm of each head's decay, at most 0 (None: no decay; -inf:
    a row sees itself alone); no gradient, so one that requires it is taken under ``torch.no_grad()`` alone.  ``sm_scale``: 1 / sqrt(D) by default,
    2**-64 to 2**64 in size.  ``state``: (B, H, D, E) float32, S before the first row, plain or dual.  ``lengths``: (B) int32, rows of each
    sequence; those behind are not read and their results are zero, and S is that behind the last one.

    Sums and states are in 32 bits.  Entries are multiplied as they are; what is formed of them in 32 bits and multiplied again (decayed entries,
    states, the products of q and k within a chunk of rows) in 16 bits for bfloat16, which has 8, 19 for float16, which has 11, and 22 for float32 and
    the state that is answered, each with an exponent of its own: fast decays and rows or columns of very different size take no digits from one
    another.  A NaN or an infinite entry reaches its own row, all later ones and those before it of its chunk.  Results are the same from run to run;
    last bits depend on how a sequence is cut, so on B, H and L, on whether there are tangents, and in the 16-bit types on whether the last
    state is answered, which is then carried in more bits.

    The gradient goes to q, k, v and state, through values and tangents.  That of the values can be differentiated once more; that through the
    tangents cannot.  Gradients that are taken inside a forward-AD level carry their tangents, but for those through the tangent, which are
    third derivatives and NaN.  Under ``torch.func`` ``jvp``, ``vjp`` and ``grad`` nest as far as that goes; ``jvp`` of ``jvp`` and ``vmap`` are refused,
    and batched cotangents of ``torch.autograd.grad``.
    """
    scale = 1.0 / math.sqrt(max((1, *q.shape[-1:]))) if sm_scale is None else sm_scale
    options = (scale, return_state, "linear_attention")
    interp = _peek_functorch()
    out = None
    if (interp is None or (interp.level() == 1 and interp.key() == _JVP)) and not _is_tracing():
        if not q.is_cuda or not _MIN_SCALE <= abs(scale) <= _MAX_SCALE:  # (the native layer checks CUDA tensors itself)
            _check(q, k, v, log_decay, scale, state, lengths)
        out = _lib.native().linear((q, k, v, state), log_decay, lengths, options)
    if out is None:
        _check(q, k, v, log_decay, scale, state, lengths)
        out = _dual.apply(sys.modules[__name__], (q, k, v, state), (log_decay, lengths), options, 2)
    return out if return_state else out[0]


def linear_attention_step(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor | None, state: Tensor, *, sm_scale: float | None = None) -> Tensor:
    """o of one more token of each sequence, (B, H, E); ``state`` becomes ``exp(log_decay) state + k v^T``, in place.

    q, k: (B, H, D), v: (B, H, E), of any strides; ``state``: (B, H, D, E) float32, as ``linear_attention`` answers it, or any (B, H) view of such
    matrices that has none twice (a slice of a larger store).  Else as ``linear_attention``.  No gradient and no tangents.
    """
    scale = 1.0 / math.sqrt(max((1, *q.shape[-1:]))) if sm_scale is None else sm_scale
    out = None
    if q.is_cuda and _MIN_SCALE <= abs(scale) <= _MAX_SCALE:
        out = _lib.native().linear_step(q, k, v, log_decay, state, scale)
    if out is None:
        _check_step(q, k, v, log_decay, scale, state)
        raise ValueError(f"state must hold row-major (D, E) matrices in memory of their own; got strides {state.stride()} for {tuple(state.shape)}")
    return out


def _check_scale(scale) -> None:
    if not _MIN_SCALE <= abs(scale) <= _MAX_SCALE:
        raise ValueError(f"sm_scale must be from 2**-64 to 2**64 in size, got {scale}")


def _check_operands(q, k, v, state, log_decay, B, H, D, E) -> None:
    if not 1 <= D <= MAX_WIDTH or not 1 <= E <= MAX_WIDTH:
        raise ValueError(f"D and E must be from 1 to {MAX_WIDTH}, got {D} and {E}")
    if B * H > 2**24:
        raise ValueError(f"at most 2**24 heads of all sequences, got {B} x {H}")
    for name, x in (("q", q), ("k", k), ("v", v)):
        if x.is_cuda and x.dtype not in _lib.DTYPE_ENUM:
            raise TypeError(f"unsupported dtype {x.dtype} of {name}; expected bfloat16, float16 or float32")
        if x.dtype != q.dtype:
            raise TypeError(f"q, k and v must have one dtype, got {q.dtype} and {x.dtype}")
    if state is not None:
        if tuple(state.shape) != (B, H, D, E):
            raise ValueError(f"state must have the shape {(B, H, D, E)}, got {tuple(state.shape)}")
        if state.dtype != torch.float32 and state.is_cuda:
            raise TypeError(f"state must be float32, got {state.dtype}")
    if log_decay is not None:
        if log_decay.dtype != torch.float32 or tuple(log_decay.shape) != (H,):
            raise TypeError(f"log_decay must be a float32 vector of {H} values, got {log_decay.dtype} {tuple(log_decay.shape)}")
        if not log_decay.is_contiguous():
            raise ValueError("log_decay must be contiguous")
        if (log_decay.requires_grad and torch.is_grad_enabled()) or fwAD.unpack_dual(log_decay).tangent is not None:
            raise NotImplementedError("linear attention has no derivative with respect to log_decay; pass log_decay.detach()")
    for name, x in (("k", k), ("v", v), ("state", state), ("log_decay", log_decay)):
        if x is not None and x.device != q.device:
            raise ValueError(f"{name} must be on {q.device} like q, got {x.device}")


def _check(q, k, v, log_decay, scale, state, lengths) -> None:
    if q.dim() != 4 or k.shape != q.shape or v.dim() != 4 or v.shape[:3] != q.shape[:3]:
        raise ValueError(f"q, k and v must have the shapes (B, H, L, D), (B, H, L, D) and (B, H, L, E); got {tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)}")
    _check_scale(scale)
    B, H, L, D = q.shape
    if L > 2**30:
        raise ValueError("sequences must have at most 2**30 rows")
    _check_operands(q, k, v, state, log_decay, B, H, D, v.shape[3])
    if lengths is not None:
        if lengths.dtype != torch.int32 or tuple(lengths.shape) != (B,) or not lengths.is_contiguous():
            raise TypeError(f"lengths must be a contiguous int32 vector of {B} values, got {lengths.dtype} {tuple(lengths.shape)}")
        if lengths.device != q.device:
            raise ValueError(f"lengths must be on {q.device} like q, got {lengths.device}")
    _require_cuda(q)


def _check_step(q, k, v, log_decay, scale, state) -> None:
    if q.dim() != 3 or k.shape != q.shape or v.dim() != 3 or v.shape[:2] != q.shape[:2]:
        raise ValueError(f"q, k and v must have the shapes (B, H, D), (B, H, D) and (B, H, E); got {tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)}")
    _check_scale(scale)
    _check_operands(q, k, v, state, log_decay, *q.shape, v.shape[2])
    if _peek_functorch() is not None or any(fwAD.unpack_dual(x).tangent is not None for x in (q, k, v, state)) or (
            torch.is_grad_enabled() and any(x.requires_grad for x in (q, k, v, state))):
        raise NotImplementedError("linear_attention_step updates the state in place and has no derivatives; use linear_attention with a state, "
                                  "or torch.no_grad()")
    _require_cuda(q)


def _launch_fwd(x, tx, extras, options, keep):
    y, ty, kept = _lib.native().linear_launch_fwd(x, tx, extras, options, keep)
    return y, ty, x[0].new_empty(0) if kept is None else kept  # (without rows nothing is kept)


def _launch_bwd(x, tx, extras, kept, g, gt, options, want):
    return _lib.native().linear_launch_bwd(x, tx, extras, kept, g, gt, options, want)


def _backward_under_functorch(x, tx, extras, kept, g, gt, options):
    return _dual.backward_under_functorch(sys.modules[__name__], x, tx, extras, kept, g, gt, options)
