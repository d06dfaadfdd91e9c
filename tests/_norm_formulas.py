"""Test helper: norms and residual sums from their formulas in float64, for the oracle side of the GPU tests (``launch_*``, by torch's
differentiation) and as stand-ins for the launches in the CPU suite (``stub_*``); and the size of what the sums behind each result are made of, for bounds of their rounding.  Only tests may use this.

Operands in the order x, y, weight, bias, scale, shift, gate, post_weight (None: absent)."""
import torch


def _mean(x):
    return x.mean(-1, keepdim=True)


def _normed(x, kind, eps):
    x = x - _mean(x) if kind == 2 else x
    s = (_mean(x * x) + eps).rsqrt()
    return x * s, s


def _value(x, kind, post, alpha, eps):
    """(r, n) by elementary operations, which torch differentiates."""
    x, y, w, b, sc, sh, gate, pw = x
    r = x
    if y is not None:
        m = _normed(y, post, eps)[0] if post else y
        for f in (gate, pw):
            m = m if f is None else m * f
        r = x + alpha * m
    n = None
    if kind:
        n = _normed(r, kind, eps)[0]
        n = n if w is None else n * w
        n = n if b is None else n + b
        n = n if sc is None else n * (1 + sc)
        n = n if sh is None else n + sh
    return (r if y is not None else None), n


def launch_fwd(x, tx, extras, options, keep):
    """(y, ty, kept) as ``norms._launch_fwd`` answers."""
    kind, post, alpha, eps, _ = options
    x = [None if t is None else t.detach().double() for t in x]
    at = [i for i, t in enumerate(x) if t is not None]
    tx = [torch.zeros_like(x[i]) if tx[i] is None else tx[i].detach().double() for i in at] if any(t is not None for t in tx) else None

    def f(*xs):
        full = [None] * 8
        for i, t in zip(at, xs):
            full[i] = t
        return tuple(t for t in _value(full, kind, post, alpha, eps) if t is not None)

    def both(ts):
        ts = list(ts)
        return [ts.pop(0) if x[1] is not None else None, ts.pop(0) if kind else None]

    xs = [x[i] for i in at]
    if tx is None:
        return both(f(*xs)), None, torch.zeros(1)
    # the tangent by differentiating the gradient's product with a dummy cotangent: no forward transform is needed inside one
    with torch.enable_grad():
        xs = [t.requires_grad_() for t in xs]
        ys = f(*xs)
        us = [torch.zeros_like(t, requires_grad=True) for t in ys]
        gs = torch.autograd.grad(ys, xs, us, create_graph=True, materialize_grads=True)
        ts = torch.autograd.grad(sum((g * t).sum() for g, t in zip(gs, tx)), us, materialize_grads=True)
    return both(t.detach() for t in ys), both(t.detach() for t in ts), torch.zeros(1)


def launch_bwd(x, tx, extras, kept, g, gt, options, want):
    """Gradients as ``norms._launch_bwd`` answers."""
    kind, post, alpha, eps, _ = options
    n = len(x)
    x = [None if t is None else t.detach().double().requires_grad_() for t in x]
    tx = [None] * n if not tx else tx
    tx = [None if t is None else t.detach().double().requires_grad_() for t in tx]
    at = [i for i in range(n) if x[i] is not None]
    with torch.enable_grad():
        ys = [t for t in _value(x, kind, post, alpha, eps)]
        loss = sum((c.double() * y).sum() for c, y in zip(g, ys) if c is not None) + 0.0 * sum(x[i].sum() for i in at)
        pairs = [(c.double(), y) for c, y in zip(gt, ys) if c is not None]
        if pairs:
            along = torch.autograd.grad([y for _, y in pairs], [x[i] for i in at], [c for c, _ in pairs], create_graph=True, materialize_grads=True)
            loss = loss + sum((d * tx[i]).sum() for d, i in zip(along, at) if tx[i] is not None)
        loss = loss + 0.0 * sum(t.sum() for t in tx if t is not None)
        leaves = [t for t in (*x, *tx) if t is not None]
        grads = list(torch.autograd.grad(loss, leaves, materialize_grads=True))
    out = [None if t is None else grads.pop(0) for t in (*x, *tx)]
    return [t if w else None for t, w in zip(out, want)]


# ---- stand-ins for the launches: without torch's differentiation, which cannot be used inside a transform --------------------------------
def _along(v, n, s, kind):
    v = v - _mean(v) if kind == 2 else v
    return s * (v - n * _mean(n * v))


def _norm_grads(g, h, n, s, t, kind):
    """Gradients of <g, n> + <h, tn> with respect to x and its tangent t."""
    if not kind:
        return g, h
    tn, b = _along(t, n, s, kind), _mean(n * t)
    return _along(g - s * b * h, n, s, kind) - s * (_mean(n * h) * tn + _mean(h * tn) * n), _along(h, n, s, kind)


class _Parts:
    """All that lies between operands and results; absent operands as what they stand for, absent tangents zero."""

    def __init__(self, x, tx, options):
        kind, self.post, self.alpha, eps, _ = options
        x = [None if t is None else t.detach() for t in x]
        one, zero = torch.ones((), dtype=x[0].dtype), torch.zeros((), dtype=x[0].dtype)
        self.w, self.b, sc, self.sh, self.gate, self.pw = (o if t is None else t for t, o in zip(x[2:], (one, zero, zero, zero, one, one)))
        tx = [zero if t is None else t.detach() for t in (tx or [None] * 8)]
        self.tw, self.tb, self.tsc, self.tsh, self.tgate, self.tpw = tx[2:]
        self.sc = 1 + sc
        self.G, self.tG = self.w * self.sc, self.tw * self.sc + self.w * self.tsc
        self.E, self.tE = self.alpha * self.gate * self.pw, self.alpha * (self.tgate * self.pw + self.gate * self.tpw)
        self.r, self.tr = x[0], tx[0].expand(x[0].shape)
        self.m = self.tm = self.ms = zero
        self.ty = zero
        if x[1] is not None:
            self.ty = tx[1].expand(x[1].shape)
            self.m, self.ms = _normed(x[1], self.post, eps) if self.post else (x[1], one)
            self.tm = _along(self.ty, self.m, self.ms, self.post) if self.post else self.ty
            self.r, self.tr = self.r + self.E * self.m, self.tr + self.tE * self.m + self.E * self.tm
        self.kind = kind
        if kind:
            self.n, self.s = _normed(self.r, kind, eps)
            self.tn = _along(self.tr, self.n, self.s, kind)


def stub_fwd(x, tx, extras, options, keep):
    p = _Parts(x, tx, options)
    y = [p.r if x[1] is not None else None, p.n * p.G + p.b * p.sc + p.sh if p.kind else None]
    ty = [p.tr if x[1] is not None else None, p.tn * p.G + p.n * p.tG + p.tb * p.sc + p.b * p.tsc + p.tsh if p.kind else None]
    return [None if t is None else t.clone() for t in y], ty if any(t is not None for t in tx) else None, torch.zeros(1)


def stub_bwd(x, tx, extras, kept, g, gt, options, want):
    p = _Parts(x, tx, options)
    zero = torch.zeros_like(x[0])
    gr, gn, gtr, gtn = (zero if c is None else c for c in (*g, *gt))
    dr, dtr = gr, gtr
    d, dt = [None] * 8, [None] * 8
    if p.kind:
        a, c = _norm_grads(gn * p.G + gtn * p.tG, gtn * p.G, p.n, p.s, p.tr, p.kind)
        dr, dtr = dr + a, dtr + c
        pg, ptg = gn * p.n + gtn * p.tn, gtn * p.n
        d[2:6] = p.sc * pg + p.tsc * ptg, p.sc * gn + p.tsc * gtn, p.w * pg + p.tw * ptg + p.b * gn + p.tb * gtn, gn
        dt[2:6] = p.sc * ptg, p.sc * gtn, p.w * ptg + p.b * gtn, gtn
    d[0], dt[0] = dr, dtr
    if x[1] is not None:
        pe, pte = dr * p.m + dtr * p.tm, dtr * p.m
        d[6:8] = p.alpha * (p.pw * pe + p.tpw * pte), p.alpha * (p.gate * pe + p.tgate * pte)
        dt[6:8] = p.alpha * p.pw * pte, p.alpha * p.gate * pte
        d[1], dt[1] = _norm_grads(p.E * dr + p.tE * dtr, p.E * dtr, p.m, p.ms, p.ty, p.post)
    out = [t if w else None for t, w in zip((*d, *dt), want)]
    return [None if t is None else t.clone() if i % 8 < 2 else t.sum_to_size(x[i % 8].shape).clone() for i, t in enumerate(out)]


def sizes(x, tx, g, gt, options):
    """For r, n, tr, tn and the gradients of x and tx the sum of the magnitudes of what each entry is added up from (float64): the formulas
    with every term's absolute value.  Absent operands are None; absent tangents and cotangents zero."""
    kind, post, alpha, eps, _ = options
    a = [None if t is None else t.detach().double() for t in x]
    X, Y, W, B, SC, SH, GATE, PW = a
    zero = torch.zeros_like(X)
    one = torch.ones((), dtype=torch.float64, device=X.device)
    t = [zero if v is None else v.detach().double().abs() for v in tx]
    tX, tY, tW, tB, tSC, tSH, tGATE, tPW = t
    mag = lambda v, otherwise: otherwise if v is None else v.abs()  # noqa: E731
    g = [zero if c is None else c.double().abs() for c in g]
    gt = [zero if c is None else c.double().abs() for c in gt]

    def around(v, k):  # a norm's entries and what its mean was made of
        n, s = _normed(v[0], k, eps)
        return (n.abs() + s * (v[1] + _mean(v[1])) if k else v[1]), s

    def along(v, n, s):
        return s * (v + _mean(v) + n * _mean(n * v))

    gate, pw = alpha * mag(GATE, one), mag(PW, one)
    E, tE = gate * pw, abs(alpha) * (tGATE * pw + mag(GATE, one) * tPW)
    rv, ra, tra = X, X.abs(), tX
    m = tm = None
    if Y is not None:
        m, ms = around((Y, Y.abs()), post) if post else (Y.abs(), one)
        tm = along(tY, m, ms) if post else tY
        ra, tra = ra + E * m, tra + tE * m + E * tm
        rv = _value(a, 0, post, alpha, eps)[0]
    out = {"r": ra, "tr": tra}
    d, dt = [None] * 8, [None] * 8
    dr, dtr = g[0], gt[0]
    if kind:
        n, s = around((rv, ra), kind)
        tn = along(tra, n, s)
        sc = 1 + mag(SC, 0 * one)
        G, tG = mag(W, one) * sc, tW * sc + mag(W, one) * tSC
        O, tO = mag(B, 0 * one) * sc + mag(SH, 0 * one), tB * sc + mag(B, 0 * one) * tSC + tSH  # noqa: E741
        out |= {"n": n * G + O, "tn": tn * G + n * tG + tO}
        h, gg = gt[1] * G, g[1] * G + gt[1] * tG
        b = _mean(n * tra)
        dr = dr + along(gg + s * b * h, n, s) + s * (_mean(n * h) * tn + _mean(h * tn) * n)
        dtr = dtr + along(h, n, s)
        pg, ptg, po, pto = g[1] * n + gt[1] * tn, gt[1] * n, g[1], gt[1]
        d[2], dt[2] = sc * pg + tSC * ptg, sc * ptg
        d[3], dt[3] = sc * po + tSC * pto, sc * pto
        d[4], dt[4] = mag(W, one) * pg + tW * ptg + mag(B, 0 * one) * po + tB * pto, mag(W, one) * ptg + mag(B, 0 * one) * pto
        d[5], dt[5] = po, pto
    d[0], dt[0] = dr, dtr
    if Y is not None:
        pe, pte = dr * m + dtr * tm, dtr * m
        d[6], dt[6] = abs(alpha) * (pw * pe + tPW * pte), abs(alpha) * pw * pte
        d[7], dt[7] = abs(alpha) * (mag(GATE, one) * pe + tGATE * pte), abs(alpha) * mag(GATE, one) * pte
        hp, gp = E * dtr, E * dr + tE * dtr
        if post:
            b = _mean(m * tY)
            d[1] = along(gp + ms * b * hp, m, ms) + ms * (_mean(m * hp) * tm + _mean(hp * tm) * m)
            dt[1] = along(hp, m, ms)
        else:
            d[1], dt[1] = gp, hp
    for i in range(2, 8):
        if a[i] is None:
            d[i] = dt[i] = None
        else:
            d[i], dt[i] = ((v.expand_as(X) if v.dim() else v.expand(X.shape)).sum_to_size(a[i].shape) for v in (d[i], dt[i]))
    return out, d, dt
