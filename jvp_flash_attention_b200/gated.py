"""The widening half of a gated feed-forward block with its tangent (csrc/gated.cu): ``h = a(x Wg^T) * (x Wu^T)`` in one kernel, both
products, the activation and the gate.

``gated_linear`` is to such a block what ``JVPAttn.fwd_dual`` is to attention: where x carries a tangent (``torch.func.jvp``, forward-AD
dual tensors) value and tangent come from one launch, and the gradient goes through both, to x, its tangent and the weights.  The
gradient of the value can be differentiated once more (Hessian-vector products, gradient penalties).  What follows in a block,
the product with the narrowing weights, is ``torch.nn.functional.linear``.  No upstream counterpart: upstream leaves it to the model.
"""
from __future__ import annotations

import ctypes as C

import torch
import torch.autograd.forward_ad as fwAD
from torch import Tensor
from torch.autograd import Function

from . import _lib
from .jvp_attention import _JVP, _is_tracing, _peek_functorch, _require_cuda, _unwrap
from .rotary import _in_memory

ACTIVATIONS = {"silu": 0, "sigmoid": 1, "gelu": 2, "gelu_tanh": 3}  # jvpfa_activation
_THIRD = "gated_linear cannot be differentiated a third time"
_ALONG_TANGENT = "the tangent output of gated_linear cannot be differentiated by a further forward transform"
_THROUGH_TANGENT = "the gradient through the tangent output of gated_linear cannot be differentiated a second time"


def gated_linear(x: Tensor, w_gate: Tensor, w_up: Tensor, activation: str = "silu") -> Tensor:
    """``activation(x @ w_gate.T) * (x @ w_up.T)``.

    x: (..., K), plain or dual; w_gate, w_up: (F, K), as ``torch.nn.Linear`` keeps them (two halves of one (2 F, K) tensor will do); all
    bfloat16, float16 or float32, of one type and device.  ``activation``: ``"silu"``, ``"sigmoid"``, ``"gelu"`` (exact) or ``"gelu_tanh"``.
    Rows of whole 16-byte pieces (K a multiple of 8) are read in place, others, and float32, through a copy.

    Sums are in 32 bits (16-bit types': the tensor cores' accumulators, which round towards zero every 16 terms), activations of 16-bit types within
    ``2**-17 (1 + |g|)``, and the result is rounded once.  For a backward the projections are kept in 24 bits an entry (float32: 32); their
    cotangents are rounded to x's type, so where one passes float16's 65504 the gradients of its row are not finite.  float32 is multiplied as
    three bfloat16 parts, about 1e-6 relative, whatever ``set_fp32_precision`` says of attention; an infinite entry gives NaN in its row.  Results
    are the same from run to run.

    Tangents of the weights, and a second differentiation of their gradients, run on operands side by side, ``[tx | x]`` and ``[w | tw]``,
    at twice the depth (where a weight's tangent is not finite, neither is the value there); the gradient through the tangent output cannot
    be differentiated again.  Gradients that are taken inside a forward-AD level carry their tangents (Hessian-vector products; attention's
    do not), which is a further backward: take them behind the level where only they are wanted.  The tangent of one through the tangent
    output would be a third derivative; it is NaN.  Under ``torch.func`` ``jvp``, ``vjp`` and ``grad`` nest as far as that goes; ``jvp`` of
    ``jvp`` and ``vmap`` (so ``jacfwd``, ``jacrev`` and ``hessian``) are refused, and batched cotangents of ``torch.autograd.grad``.
    """
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation is one of {', '.join(ACTIVATIONS)}; got {activation!r}")
    act = ACTIVATIONS[activation]
    interp = _peek_functorch()
    if (interp is None or (interp.level() == 1 and interp.key() == _JVP)) and not _is_tracing():
        if not x.is_cuda:  # (the native layer checks CUDA tensors itself)
            _check(x, w_gate, w_up)
        out = _lib.native().gated(x, w_gate, w_up, act)
        if out is not None:
            return out
        if any(fwAD.unpack_dual(w).tangent is not None for w in (w_gate, w_up)):
            _check(x, w_gate, w_up)
            xs, txs, *ws = _side_by_side(*(t for operand in (x, w_gate, w_up) for t in fwAD.unpack_dual(operand)))
            out = _lib.native().gated(fwAD.make_dual(xs, txs), *ws, act, side_by_side=True)
            if out is not None:
                return out
    _check(x, w_gate, w_up)
    return _Gated.apply(x, w_gate, w_up, act)[0]


def _check(x, w_gate, w_up) -> None:
    if x.dim() < 1 or w_gate.dim() != 2 or w_up.shape != w_gate.shape or x.shape[-1] != w_gate.shape[1]:
        raise ValueError("x, w_gate and w_up must have the shapes (..., K), (F, K) and (F, K); got "
                         f"{tuple(x.shape)}, {tuple(w_gate.shape)} and {tuple(w_up.shape)}")
    if w_gate.numel() == 0:
        raise ValueError(f"the weights must not be empty, got {tuple(w_gate.shape)}")
    if x.numel() // x.shape[-1] >= 2**31:
        raise ValueError("x must have less than 2**31 rows")
    for name, t in (("x", x), ("w_gate", w_gate), ("w_up", w_up)):
        if t.is_cuda and t.dtype not in _lib.DTYPE_ENUM:
            raise TypeError(f"unsupported dtype {t.dtype} of {name}; expected bfloat16, float16 or float32")
        if t.dtype != x.dtype:
            raise TypeError(f"x, w_gate and w_up must have one dtype, got {x.dtype} and {t.dtype}")
        if t.device != x.device:
            raise ValueError(f"x, w_gate and w_up must be on one device, got {x.device} and {t.device}")
    _require_cuda(x, w_gate, w_up)


def _side_by_side(x, tx, w_gate, t_gate, w_up, t_up):
    """Operands of twice the width with the same value and, in the tangent, the weights' part as well:
    ``[x | 0] [w | tw]^T = x w^T`` and ``[tx | x] [w | tw]^T = tx w^T + x tw^T``."""
    or_zero = lambda t, like: torch.zeros_like(like) if t is None else t.to(like.dtype)  # noqa: E731
    cat = lambda a, b: torch.cat((a, b), -1)  # noqa: E731
    return (cat(x, torch.zeros_like(x)), cat(or_zero(tx, x), x), cat(w_gate, or_zero(t_gate, w_gate)), cat(w_up, or_zero(t_up, w_up)))


def _second(x, w_gate, w_up, gh, vx, v_gate, v_up, activation, tgh=None):
    """The gradients of <(dx, dwg, dwu), (vx, v_gate, v_up)> with respect to x, w_gate, w_up and gh, where (dx, dwg, dwu) are those of <gh, h>: of
    <gh, th> for the tangents v, and th itself.  The first three are also (dx, dwg, dwu)'s tangent along v, and with ``tgh``, which adds those of
    <tgh, h>, along v and gh's tangent."""
    K = x.shape[-1]
    if v_gate is None and v_up is None:
        _, th, kept = _launch_fwd(x, vx, w_gate, w_up, activation, True)
        dx, _, dwg, dwu = _launch_bwd(x, vx, w_gate, w_up, kept, tgh, gh, activation, True, False, True)
        return dx, dwg, dwu, th
    wide = _side_by_side(x, vx, w_gate, v_gate, w_up, v_up)
    _, th, kept = _launch_fwd(*wide, activation, True)
    dx, dtx, dwg, dwu = _launch_bwd(*wide, kept, tgh, gh, activation, True, True, True)
    return dx[..., :K] + dtx[..., K:], dwg[:, :K], dwu[:, :K], th


# ---- the general route (functorch transforms other than a lone torch.func.jvp) --------------------------------------------
def _launch_fwd(x, tx, w_gate, w_up, activation, keep):
    """Runs jvpfa_gated_fwd on plain tensors: (h, th, kept), what a backward reads with ``keep``."""
    F, K = w_gate.shape
    x2, tx2, wg, wu = (None if t is None else _rows(t) for t in (x, tx, w_gate, w_up))
    h, th = (torch.empty(*x.shape[:-1], F, device=x.device, dtype=x.dtype) if wanted else None for wanted in (True, tx is not None))
    n = _lib.load().jvpfa_gated_kept_bytes(_lib.DTYPE_ENUM[x.dtype], x2.shape[0], F, tx is not None)
    kept = torch.empty(n, device=x.device, dtype=torch.uint8) if keep else None
    if x.numel():
        a = _lib.GatedFwdArgs()
        _describe(a, x2, tx2, wg, wu, activation)
        a.h, a.th, a.kept = (_lib.ptr(t) for t in (h, th, kept))
        _run(a, x2, "jvpfa_gated_fwd")
    return h, th, kept


def _launch_bwd(x, tx, w_gate, w_up, kept, gh, gth, activation, need_x, need_tx, need_w):
    """Runs jvpfa_gated_bwd on plain tensors: (dx, dtx, dwg, dwu), None for those not asked for.  tx as in the forward
    that left ``kept``."""
    F, K = w_gate.shape
    x2, wg, wu = _rows(x), _rows(w_gate), _rows(w_up)
    tx2 = _rows(tx) if gth is not None else None
    gh, gth = (None if c is None else _dense(c, x.dtype) for c in (gh, gth))
    make = torch.empty if x.numel() else torch.zeros
    out = [make(shape, device=x.device, dtype=x.dtype) if wanted else None
           for wanted, shape in ((need_x, x.shape), (need_tx and gth is not None, x.shape), (need_w, (F, K)), (need_w, (F, K)))]
    if x.numel() and any(t is not None for t in out):
        a = _lib.GatedBwdArgs()
        _describe(a, x2, tx2, wg, wu, activation)
        a.kept, a.gh, a.gth = (_lib.ptr(t) for t in (kept, gh, gth))
        a.kept_tangent = tx is not None
        a.dx, a.dtx, a.dwg, a.dwu = (_lib.ptr(t) for t in out)
        _run(a, x2, "jvpfa_gated_bwd")
    return tuple(out)


def _rows(t):
    t = _in_memory(t)
    t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 else t.contiguous()


def _dense(t, dtype):
    """Row-major and on a 16-byte boundary, where the entry wants a cotangent (a slice of a longer one begins anywhere)."""
    t = _in_memory(t).to(dtype).contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def _describe(a, x, tx, wg, wu, activation):
    a.struct_size = C.sizeof(a)
    a.dtype = _lib.DTYPE_ENUM[x.dtype]
    (a.M, a.K), a.F, a.activation = x.shape, wg.shape[0], activation
    for name, t in (("x", x), ("tx", tx), ("wg", wg), ("wu", wu)):
        if t is not None:
            setattr(a, name, t.data_ptr())
            setattr(a, name + "_stride", t.stride(0))


def _run(a, x, entry):
    lib = _lib.load()
    with torch.cuda.device(x.device):
        n = getattr(lib, entry + "_workspace")(C.byref(a))
    workspace = torch.empty(n, device=x.device, dtype=torch.uint8) if n else None
    a.workspace, a.workspace_bytes = _lib.ptr(workspace), n
    _lib.check(_lib._launch(x, getattr(lib, entry), a), entry)


class _Operator(Function):
    """A launch as torch.autograd and torch.func's jvp, vjp and grad see it."""

    @staticmethod
    def vmap(info, in_dims, *args):
        raise NotImplementedError("gated_linear has no rule for torch.func.vmap (nor for jacfwd, jacrev and hessian, which are made of it): "
                                  "the rows of x are a batch already")


def _unknown(like, message):
    """Tangents that take a third derivative: refused where a transform asks for them, NaN inside a forward-AD level (as the native layer's)."""
    if _peek_functorch() is not None:
        raise RuntimeError(message)
    return tuple(torch.full_like(t, torch.nan) for t in like)


class _Gated(_Operator):
    """h, and what its backward reads."""

    @staticmethod
    def forward(x, w_gate, w_up, activation):
        h, _, kept = _launch_fwd(_unwrap(x), None, _unwrap(w_gate), _unwrap(w_up), activation, True)
        return h, kept

    @staticmethod
    def setup_context(ctx, inputs, outputs):
        x, w_gate, w_up, ctx.activation = inputs
        ctx.mark_non_differentiable(outputs[1])
        ctx.save_for_backward(x, w_gate, w_up, outputs[1])
        ctx.save_for_forward(x, w_gate, w_up)
        ctx.set_materialize_grads(False)

    @staticmethod
    def jvp(ctx, tx, t_gate, t_up, *_):
        x, w_gate, w_up = ctx.saved_tensors
        if t_gate is not None or t_up is not None:
            x, tx, w_gate, w_up = _side_by_side(x, tx, w_gate, t_gate, w_up, t_up)
        return (None if tx is None else _GatedTangent.apply(x, tx.to(x.dtype), w_gate, w_up, ctx.activation)[0]), None

    @staticmethod
    def backward(ctx, gh, *_):
        if gh is None:
            return None, None, None, None
        x, w_gate, w_up, kept = ctx.saved_tensors
        return (*_GatedGrad.apply(x, None, w_gate, w_up, kept, gh, ctx.activation), None)


class _GatedTangent(_Operator):
    """th, differentiable once with respect to x, its tangent and the weights."""

    @staticmethod
    def forward(x, tx, w_gate, w_up, activation):
        _, th, kept = _launch_fwd(*(_unwrap(t) for t in (x, tx, w_gate, w_up)), activation, True)
        return th, kept

    @staticmethod
    def setup_context(ctx, inputs, outputs):
        *tensors, ctx.activation = inputs
        ctx.mark_non_differentiable(outputs[1])
        ctx.save_for_backward(*tensors, outputs[1])
        ctx.set_materialize_grads(False)

    @staticmethod
    def jvp(ctx, *tangents):
        raise RuntimeError(_ALONG_TANGENT)

    @staticmethod
    def backward(ctx, gth, *_):
        if gth is None:
            return (None,) * 5
        dx, dtx, dwg, dwu = _GatedDualGrad.apply(*ctx.saved_tensors, gth, ctx.activation)
        return dx, dtx, dwg, dwu, None


class _GatedGrad(_Operator):
    """(dx, dwg, dwu) of <gh, h>, differentiable once more, in either direction.  ``tx``: of the forward that left ``kept``, or
    None."""

    @staticmethod
    def forward(x, tx, w_gate, w_up, kept, gh, activation):
        x, tx, w_gate, w_up, kept, gh = (None if t is None else _unwrap(t) for t in (x, tx, w_gate, w_up, kept, gh))
        dx, _, dwg, dwu = _launch_bwd(x, tx, w_gate, w_up, kept, gh, None, activation, True, False, True)
        return dx, dwg, dwu

    @staticmethod
    def setup_context(ctx, inputs, outputs):
        x, tx, w_gate, w_up, kept, gh, ctx.activation = inputs
        ctx.save_for_backward(x, w_gate, w_up, gh)
        ctx.save_for_forward(x, tx, w_gate, w_up, kept, gh)
        ctx.set_materialize_grads(False)

    @staticmethod
    def jvp(ctx, vx, _, v_gate, v_up, __, tgh, ___):
        x, tx, w_gate, w_up, kept, gh = ctx.saved_tensors
        if vx is None and v_gate is None and v_up is None:  # linear in gh
            return _GatedGrad.apply(x, tx, w_gate, w_up, kept, tgh, ctx.activation)
        return _GatedGradTangent.apply(x, w_gate, w_up, gh, vx, v_gate, v_up, tgh, ctx.activation)

    @staticmethod
    def backward(ctx, vx, v_gate, v_up):
        if vx is None and v_gate is None and v_up is None:
            return (None,) * 7
        dx, dwg, dwu, th = _GatedSecond.apply(*ctx.saved_tensors, vx, v_gate, v_up, ctx.activation)
        return dx, None, dwg, dwu, None, th, None


class _GatedSecond(_Operator):
    """``_second``: differentiable in the tangents v, which it is linear in, and forward only."""

    @staticmethod
    def forward(x, w_gate, w_up, gh, vx, v_gate, v_up, activation):
        return _second(*(None if t is None else _unwrap(t) for t in (x, w_gate, w_up, gh, vx, v_gate, v_up)), activation)

    @staticmethod
    def setup_context(ctx, inputs, outputs):
        *tensors, ctx.activation = inputs
        ctx.save_for_forward(*tensors[:4])
        ctx.set_materialize_grads(False)

    @staticmethod
    def jvp(ctx, tx, t_gate, t_up, tgh, vx, v_gate, v_up, _):
        if tx is None and t_gate is None and t_up is None and tgh is None:
            return _GatedSecond.apply(*ctx.saved_tensors, vx, v_gate, v_up, ctx.activation)
        return _unknown(ctx.saved_tensors, _THIRD)

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(_THIRD)


class _GatedGradTangent(_Operator):
    """The tangents of (dx, dwg, dwu) of <gh, h>."""

    @staticmethod
    def forward(x, w_gate, w_up, gh, vx, v_gate, v_up, tgh, activation):
        x, w_gate, w_up, gh, vx, v_gate, v_up, tgh = (None if t is None else _unwrap(t) for t in (x, w_gate, w_up, gh, vx, v_gate, v_up, tgh))
        return _second(x, w_gate, w_up, gh, vx, v_gate, v_up, activation, tgh)[:3]

    @staticmethod
    def setup_context(ctx, inputs, outputs):
        pass

    @staticmethod
    def jvp(ctx, *tangents):
        raise RuntimeError(_THIRD)

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(_THIRD)


class _GatedDualGrad(_Operator):
    """(dx, dtx, dwg, dwu) of <gth, th>."""

    @staticmethod
    def forward(x, tx, w_gate, w_up, kept, gth, activation):
        x, tx, w_gate, w_up, kept, gth = (_unwrap(t) for t in (x, tx, w_gate, w_up, kept, gth))
        return _launch_bwd(x, tx, w_gate, w_up, kept, None, gth, activation, True, True, True)

    @staticmethod
    def setup_context(ctx, inputs, outputs):
        *tensors, ctx.activation = inputs
        ctx.save_for_forward(*tensors[:-1])
        ctx.set_materialize_grads(False)

    @staticmethod
    def jvp(ctx, vx, vtx, v_gate, v_up, _, tgth, __):
        if vx is None and vtx is None and v_gate is None and v_up is None:  # linear in gth
            return _GatedDualGrad.apply(*ctx.saved_tensors, tgth, ctx.activation)
        return _unknown(ctx.saved_tensors[:4], _THROUGH_TANGENT)

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(_THROUGH_TANGENT)


def _backward_under_functorch(x, tx, w_gate, w_up, kept, gh, gth, activation):
    """The native layer's backward where a cotangent is a tensor of a functorch transform: Functions take part in it, the part through h in one
    that can be differentiated again."""
    dx = dtx = dwg = dwu = None
    if gth is not None:
        dx, dtx, dwg, dwu = _GatedDualGrad.apply(x, tx, w_gate, w_up, kept, gth, activation)
    if gh is not None:
        part = _GatedGrad.apply(x, tx, w_gate, w_up, kept, gh, activation)
        dx, dwg, dwu = part if dx is None else (a + b for a, b in zip((dx, dwg, dwu), part))
    return dx, dtx, dwg, dwu
