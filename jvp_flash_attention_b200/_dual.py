"""Operators of several inputs and outputs under functorch transforms (the general route: the native layer, csrc/native_dual.h, serves plain
tensors, dual tensors and a lone ``torch.func.jvp``).

An operator is a module with two launches,

    _launch_fwd(x, tx, extras, options, keep) -> (y, ty or None, kept)
    _launch_bwd(x, tx, extras, kept, g, gt, options, want) -> gradients of <g, y> + <gt, ty> with respect to x and tx

``x``, ``tx`` lists of tensors (None: absent, a tangent of zero), ``extras`` tensors without gradients, ``options`` a tuple whose last entry is the
operator's name.  Everything else follows from what holds for all of them: the gradient of <grads(g), v> with respect to x is that of <g, ty> along
the tangents v, and with respect to g it is ty; the tangents of the gradients along (v, tg) are the gradients of <tg, y> + <g, ty>.
"""
from __future__ import annotations

import torch
from torch.autograd import Function

from .jvp_attention import _peek_functorch, _unwrap


def _plain(ts):
    return [None if t is None else _unwrap(t) for t in ts]


def _any(ts):
    return any(t is not None for t in ts)


class _Call:
    """An operator's launches with what they take besides tensors that have gradients."""

    def __init__(self, module, extras, options, n, m):
        self.module, self.extras, self.options, self.n, self.m = module, extras, options, n, m
        self.name = options[-1]

    def forward(self, x, tx, keep):
        return self.module._launch_fwd(_plain(x), _plain(tx), _plain(self.extras), self.options, keep)

    def backward(self, x, tx, kept, g, gt, want_tx=True):
        want = [t is not None for t in x] + [want_tx and t is not None for t in tx]
        return self.module._launch_bwd(_plain(x), _plain(tx), _plain(self.extras), _unwrap(kept), _plain(g), _plain(gt), self.options, want)

    def none(self, k=1):
        return [None] * k


def _through_tangent(call):
    return f"there is no second derivative through the tangent outputs of {call.name}"


def _third(call):
    return f"there is no third derivative of {call.name}"


def _unknown(like, message):
    """Tangents that take a derivative there is none of: refused where a transform asks for them, NaN inside a forward-AD level (as the native
    layer's)."""
    if _peek_functorch() is not None:
        raise RuntimeError(message)
    return tuple(None if t is None else torch.full_like(t, torch.nan) for t in like)


class _Operator(Function):
    @staticmethod
    def vmap(info, in_dims, call, *args):
        raise NotImplementedError(f"{call.name} has no rule for torch.func.vmap (nor for jacfwd, jacrev and hessian, which are made of it): "
                                  "its operands have batch dimensions already")


class _Value(_Operator):
    """(y..., kept) of (call, x...)."""

    @staticmethod
    def forward(call, *x):
        y, _, kept = call.forward(x, call.none(call.n), True)
        return (*y, kept)

    @staticmethod
    def setup_context(ctx, inputs, outputs):
        ctx.call, *x = inputs
        ctx.mark_non_differentiable(outputs[-1])
        ctx.save_for_backward(*x, outputs[-1])
        ctx.save_for_forward(*x)
        ctx.set_materialize_grads(False)

    @staticmethod
    def jvp(ctx, _, *tx):
        x = ctx.saved_tensors
        if not _any(tx):
            return (None,) * (ctx.call.m + 1)
        tx = [None if t is None else t.to(v.dtype) for t, v in zip(tx, x)]
        return (*_Tangent.apply(ctx.call, *x, *tx)[:-1], None)

    @staticmethod
    def backward(ctx, *g):
        call, (*x, kept) = ctx.call, ctx.saved_tensors
        if not _any(g[:-1]):
            return (None,) * (1 + call.n)
        return None, *_Grad.apply(call, kept, *x, *call.none(call.n), *g[:-1])


class _Tangent(_Operator):
    """(ty..., kept) of (call, x..., tx...), differentiable once."""

    @staticmethod
    def forward(call, *xs):
        _, ty, kept = call.forward(xs[:call.n], xs[call.n:], True)
        return (*ty, kept)

    @staticmethod
    def setup_context(ctx, inputs, outputs):
        ctx.call, *xs = inputs
        ctx.mark_non_differentiable(outputs[-1])
        ctx.save_for_backward(*xs, outputs[-1])
        ctx.set_materialize_grads(False)

    @staticmethod
    def jvp(ctx, *tangents):
        raise RuntimeError(f"the tangent outputs of {ctx.call.name} cannot be differentiated by a further forward transform")

    @staticmethod
    def backward(ctx, *gt):
        call, (*xs, kept) = ctx.call, ctx.saved_tensors
        if not _any(gt[:-1]):
            return (None,) * (1 + 2 * call.n)
        return None, *_DualGrad.apply(call, kept, *xs, *gt[:-1])


class _Grad(_Operator):
    """Gradients of <g, y> with respect to x: of (call, kept, x..., tx..., g...), differentiable once more in either direction; tx: of the forward
    that left ``kept``."""

    @staticmethod
    def forward(call, kept, *xs):
        n, m = call.n, call.m
        return tuple(call.backward(xs[:n], xs[n:2 * n], kept, xs[2 * n:], call.none(m), False)[:n])

    @staticmethod
    def setup_context(ctx, inputs, outputs):
        ctx.call, kept, *xs = inputs
        ctx.save_for_backward(kept, *xs)
        ctx.save_for_forward(kept, *xs)
        ctx.set_materialize_grads(False)

    @staticmethod
    def jvp(ctx, _, __, *tangents):
        call, (kept, *xs) = ctx.call, ctx.saved_tensors
        n = call.n
        x, v, tg = xs[:n], tangents[:n], tangents[2 * n:]
        if not _any(v):  # linear in g
            return _Grad.apply(call, kept, *xs[:2 * n], *tg)
        return _GradTangent.apply(call, *x, *xs[2 * n:], *v, *tg)

    @staticmethod
    def backward(ctx, *v):
        call, (_, *xs) = ctx.call, ctx.saved_tensors
        n, m = call.n, call.m
        if not _any(v):
            return (None,) * (2 + 2 * n + m)
        out = _Second.apply(call, *xs[:n], *xs[2 * n:], *v)
        return None, None, *out[:n], *call.none(n), *out[n:]


class _Second(_Operator):
    """Gradients of <grads(g), v> with respect to x and g: of (call, x..., g..., v...).  Linear in v, which a forward transform may move."""

    @staticmethod
    def forward(call, *xs):
        n, m = call.n, call.m
        x, g, v = xs[:n], xs[n:n + m], xs[n + m:]
        _, ty, kept = call.forward(x, v, True)
        d = call.backward(x, v, kept, call.none(m), g, False)[:n]
        return *d, *(t if c is not None else None for t, c in zip(ty, g))

    @staticmethod
    def setup_context(ctx, inputs, outputs):
        ctx.call, *xs = inputs
        ctx.save_for_forward(*xs)
        ctx.set_materialize_grads(False)

    @staticmethod
    def jvp(ctx, _, *tangents):
        call, xs = ctx.call, ctx.saved_tensors
        k = call.n + call.m
        if not _any(tangents[:k]):
            return _Second.apply(call, *xs[:k], *tangents[k:])
        return _unknown(xs[:k], _third(call))

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(_third(ctx.call))


class _GradTangent(_Operator):
    """The tangents of the gradients of <g, y>: of (call, x..., g..., v..., tg...)."""

    @staticmethod
    def forward(call, *xs):
        n, m = call.n, call.m
        x, g, v, tg = xs[:n], xs[n:n + m], xs[n + m:2 * n + m], xs[2 * n + m:]
        _, _, kept = call.forward(x, v, True)
        return tuple(call.backward(x, v, kept, tg, g, False)[:n])

    @staticmethod
    def setup_context(ctx, inputs, outputs):
        ctx.call = inputs[0]

    @staticmethod
    def jvp(ctx, *tangents):
        raise RuntimeError(_third(ctx.call))

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(_third(ctx.call))


class _DualGrad(_Operator):
    """Gradients of <gt, ty> with respect to x and tx: of (call, kept, x..., tx..., gt...)."""

    @staticmethod
    def forward(call, kept, *xs):
        n, m = call.n, call.m
        return tuple(call.backward(xs[:n], xs[n:2 * n], kept, call.none(m), xs[2 * n:]))

    @staticmethod
    def setup_context(ctx, inputs, outputs):
        ctx.call, kept, *xs = inputs
        ctx.save_for_forward(kept, *xs)
        ctx.set_materialize_grads(False)

    @staticmethod
    def jvp(ctx, _, __, *tangents):
        call, (kept, *xs) = ctx.call, ctx.saved_tensors
        n = call.n
        if not _any(tangents[:2 * n]):  # linear in gt
            return _DualGrad.apply(call, kept, *xs[:2 * n], *tangents[2 * n:])
        return _unknown(xs[:2 * n], _through_tangent(call))

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(_through_tangent(ctx.call))


def apply(module, x, extras, options, m):
    """The operator's outputs, by Functions."""
    return _Value.apply(_Call(module, extras, options, len(x), m), *x)[:m]


def backward_under_functorch(module, x, tx, extras, kept, g, gt, options):
    """The native layer's backward where a cotangent is a tensor of a functorch transform: Functions take part in it, the part through y in one
    that can be differentiated again."""
    call = _Call(module, extras, options, len(x), len(g))
    tx = list(tx) or call.none(call.n)
    d = call.none(2 * call.n)
    if _any(gt):
        d = list(_DualGrad.apply(call, kept, *x, *tx, *gt))
    if _any(g):
        part = _Grad.apply(call, kept, *x, *tx, *g)
        for i, t in enumerate(part):
            if t is not None:
                d[i] = t if d[i] is None else d[i] + t
    return d
