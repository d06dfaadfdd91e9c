"""The norm in front of a block and the residual sum behind one, with their tangents (csrc/norm.cu): one pass over the rows for

    r = x + alpha * gate * post(y)        and        n = norm(r) * weight * (1 + scale) + bias * (1 + scale) + shift

``norm``, ``residual`` and ``residual_norm`` are to the rest of a transformer block what ``JVPAttn.fwd_dual`` is to attention: where operands carry
tangents (``torch.func.jvp``, forward-AD dual tensors), those of the modulation included, values and tangents come from one launch, and the
gradient goes through both.  Gradients of the values can be differentiated once more.  No upstream counterpart: upstream leaves this to the
model.
"""
from __future__ import annotations

import sys

import torch
from torch import Tensor

from . import _dual, _lib
from .jvp_attention import _JVP, _is_tracing, _peek_functorch, _require_cuda

NORMS = {None: 0, "rms": 1, "layer": 2}
MAX_WIDTH = 16384
_VECTORS = ("weight", "bias", "scale", "shift", "gate", "post_weight")


def norm(x: Tensor, weight: Tensor | None = None, bias: Tensor | None = None, *, scale: Tensor | None = None, shift: Tensor | None = None,
         kind: str = "rms", eps: float = 1e-6) -> Tensor:
    """``n * weight * (1 + scale) + bias * (1 + scale) + shift``, ``n`` each row of x by its root mean square (``kind="rms"``) or less its mean and
    by its deviation (``"layer"``), ``eps`` added to the square.

    x: (..., C), bfloat16, float16 or float32, plain or dual, C up to 16384; rows that are 16-byte aligned are read 16 bytes at a time.
    weight, bias: (C,).  scale, shift: of a conditioned norm, (C,) or with x's leading dimensions up to some and ones behind, as (B, 1, C) for x
    (B, L, C).  The vectors have one type, x's or float32.  (A backward holds their sums in 32 bits, once for each group of rows that has vectors
    of its own, or 148 times: where every row has, that is four bytes an entry of x for each of weight or scale, bias or shift, and gate.)  All arithmetic is in 32 bits, and the result is rounded once.

    The gradient goes to all operands, through the value and through the tangent.  That of the value can be differentiated once more; that through
    the tangent cannot.  Gradients that are taken inside a forward-AD level carry their tangents, but for those through the tangent, which are
    third derivatives and NaN.  Under ``torch.func`` ``jvp``, ``vjp`` and ``grad`` nest as far as that goes; ``jvp`` of ``jvp`` and ``vmap`` are
    refused, and batched cotangents of ``torch.autograd.grad``.  Results are the same from run to run.
    """
    if kind is None:
        raise ValueError("kind is 'rms' or 'layer'")
    return _apply(x, None, (weight, bias, scale, shift, None, None), kind, None, 1.0, eps, "norm")[1]


def residual(x: Tensor, y: Tensor, *, gate: Tensor | None = None, post: str | None = None, post_weight: Tensor | None = None, alpha: float = 1.0,
             eps: float = 1e-6) -> Tensor:
    """``x + alpha * gate * y``, or with ``post="rms"`` or ``"layer"`` ``x + alpha * gate * norm(y) * post_weight``: a block's output y, of x's
    shape and type, added to what went into it.  gate: (C,) or of a sequence as ``norm``'s scale, post_weight: (C,).  Otherwise as ``norm``."""
    return _apply(x, y, (None, None, None, None, gate, post_weight), None, post, alpha, eps, "residual")[0]


def residual_norm(x: Tensor, y: Tensor, weight: Tensor | None = None, bias: Tensor | None = None, *, scale: Tensor | None = None,
                  shift: Tensor | None = None, gate: Tensor | None = None, post: str | None = None, post_weight: Tensor | None = None,
                  alpha: float = 1.0, kind: str = "rms", eps: float = 1e-6) -> tuple[Tensor, Tensor]:
    """``(r, n)``: ``r = residual(x, y, ...)`` and ``n = norm(r, ...)``, which the next block reads, in one pass.  n is the norm of the sum in 32 bits,
    before r is rounded.  Operands and derivatives as those of ``norm`` and ``residual``."""
    if kind is None:
        raise ValueError("kind is 'rms' or 'layer'; residual is the sum without a norm")
    r, n = _apply(x, y, (weight, bias, scale, shift, gate, post_weight), kind, post, alpha, eps, "residual_norm")
    return r, n


def _apply(x, y, vectors, kind, post, alpha, eps, name):
    for what, k in (("kind", kind), ("post", post)):
        if k not in NORMS:
            raise ValueError(f"{what} is 'rms' or 'layer'; got {k!r}")
    options = (NORMS[kind], NORMS[post], alpha, eps, name)
    interp = _peek_functorch()
    if (interp is None or (interp.level() == 1 and interp.key() == _JVP)) and not _is_tracing():
        if not x.is_cuda:  # (the native layer checks CUDA tensors itself)
            _check(x, y, vectors, post)
        out = _lib.native().norm((x, y, *vectors), *options)
        if out is not None:
            return out
    _check(x, y, vectors, post)
    return _dual.apply(sys.modules[__name__], (x, y, *vectors), (), options, 2)


def _check(x, y, vectors, post) -> None:
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_WIDTH:
        raise ValueError(f"x must have the shape (..., C) with C from 1 to {MAX_WIDTH}, got {tuple(x.shape)}")
    if x.numel() // x.shape[-1] > 2**30:
        raise ValueError("x must have at most 2**30 rows")
    if y is not None and y.shape != x.shape:
        raise ValueError(f"x and y must have one shape, got {tuple(x.shape)} and {tuple(y.shape)}")
    if x.is_cuda and x.dtype not in _lib.DTYPE_ENUM:
        raise TypeError(f"unsupported dtype {x.dtype} of x; expected bfloat16, float16 or float32")
    if y is not None and y.dtype != x.dtype:
        raise TypeError(f"x and y must have one dtype, got {x.dtype} and {y.dtype}")
    groups, first = None, None
    for name, v in zip(_VECTORS, vectors):
        if v is None:
            continue
        if v.dim() < 1 or v.dim() > x.dim() or v.shape[-1] != x.shape[-1]:
            raise ValueError(f"{name} must have the shape (C,) or x's leading dimensions up to some and ones behind; got {tuple(v.shape)} for x {tuple(x.shape)}")
        if first is not None and v.dtype != first.dtype:
            raise TypeError(f"the vectors must have one dtype, got {first.dtype} and {v.dtype} of {name}")
        first = v
        if v.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"{name} must be float32 or of x's dtype, got {v.dtype}")
        if v.numel() == v.shape[-1]:
            continue
        k = max((d + 1 for d in range(v.dim() - 1) if v.shape[d] != 1), default=0)
        if v.dim() != x.dim() or v.shape[:k] != x.shape[:k]:
            raise ValueError(f"{name} must have the shape (C,) or x's leading dimensions up to some and ones behind; got {tuple(v.shape)} for x {tuple(x.shape)}")
        if groups not in (None, v.numel()):
            raise ValueError("vectors of parts of x must have one shape")
        groups = v.numel()
    for name, t in (("y", y), *zip(_VECTORS, vectors)):
        if t is not None and t.device != x.device:
            raise ValueError(f"{name} must be on {x.device} like x, got {t.device}")
    _require_cuda(x)


def _launch_fwd(x, tx, extras, options, keep):
    return _lib.native().norm_launch_fwd(x, tx, options, keep)


def _launch_bwd(x, tx, extras, kept, g, gt, options, want):
    return _lib.native().norm_launch_bwd(x, tx, kept, g, gt, options, want)


def _backward_under_functorch(x, tx, extras, kept, g, gt, options):
    return _dual.backward_under_functorch(sys.modules[__name__], x, tx, extras, kept, g, gt, options)
