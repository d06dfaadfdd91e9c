"""Performance cases of the operators around and instead of attention in a transformer block: norms with the residual sum, gate and
modulation that stand beside them, and linear attention with a decay for each head, over sequences and for single tokens.

A case names one pass through one of them:

* ``op``     ``norm``      a norm of the rows, with its weights and a sequence's modulation
             ``residual``  ``r = x + alpha gate * post(y)`` and the norm of r, which the next block reads
             ``linear``    causal linear attention over sequences
             ``token``     linear attention of one more token of each sequence, its states updated in place
* ``step``   ``fwd``, ``fwd_bwd``, ``jvp``, ``jvp_bwd`` as in attention: the value without gradients; the value and the gradients of all
             inputs; value and tangent; value and tangent, and the gradients through both
* ``api``    how the tangents travel: ``func`` = ``torch.func.jvp``, ``fwad`` = ``torch.autograd.forward_ad`` dual tensors
* ``layout`` ``bhld`` contiguous queries, keys and values, ``blhd`` the (B, H, L, D) views of (B, L, H, D) projections, ``packed`` the
             views of one (B, L, 3 H, D) projection

The cotangents are inputs: in a model they arrive from the layers above.
"""
from __future__ import annotations

import math

import torch
import torch.autograd.forward_ad as fwAD

own = False
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
TANGENT_STD = 0.1
EPS = 1e-6
CHUNK = 128  # rows that the plain form of linear attention takes together


def _norm(name, step, dtype, B, L, C, kind, weights=True, modulated=False, api="func"):
    """weights: of the channels (with a bias for "layer"); modulated: scale and shift of each sequence."""
    return {"name": name, "op": "norm", "step": step, "dtype": dtype, "B": B, "L": L, "C": C, "kind": kind, "weights": weights,
            "modulated": modulated, "api": api}


def _residual(name, step, dtype, B, L, C, kind, post="", weights=False, modulated=True, gated=True, alpha=1.0, api="func"):
    """post: the norm of the block's output ("" for none), with weights; gated: a gate of each sequence."""
    return _norm(name, step, dtype, B, L, C, kind, weights, modulated, api) | {"op": "residual", "post": post, "gated": gated, "alpha": alpha}


def _linear(name, step, dtype, B, H, L, D, E, layout="blhd", api="func", decay=True, continued=False, ragged=False):
    """D, E: width of queries and keys, of values; continued: a state of earlier rows is given and the last one is answered;
    ragged: sequences of different lengths."""
    return {"name": name, "op": "linear", "step": step, "dtype": dtype, "B": B, "H": H, "L": L, "D": D, "E": E, "layout": layout,
            "api": api, "decay": decay, "continued": continued, "ragged": ragged}


def _token(name, dtype, B, H, D, E, decay=True):
    return {"name": name, "op": "token", "step": "fwd", "dtype": dtype, "B": B, "H": H, "D": D, "E": E, "decay": decay}


def listed():
    return [
        # one new token of each of eight sequences: the time of a call
        _norm("norm_token", "fwd", "bf16", 8, 1, 1024, "rms"),
        # the headline configuration's rows with a conditioned norm, a JVP-consistency training step
        _norm("norm_step", "jvp_bwd", "bf16", 4, 2048, 1024, "layer", weights=False, modulated=True),
        # ordinary training, tokens and a width that no vector divides
        _norm("norm_ragged", "fwd_bwd", "fp16", 3, 1330, 2731, "rms"),
        # fp32 with tangents, an odd length
        _residual("residual_fp32", "jvp", "fp32", 2, 1023, 768, "layer", api="fwad"),
        # the headline configuration's rows between two conditioned blocks, a JVP-consistency training step
        _residual("residual_step", "jvp_bwd", "bf16", 4, 2048, 1024, "layer"),
        # ordinary training between two blocks of generic width, norms behind and in front of each
        _residual("residual_wide", "fwd_bwd", "bf16", 4, 2048, 4096, "rms", post="rms", weights=True, modulated=False, gated=False, alpha=0.5),
        # prompts of different lengths in one batch, continued from earlier rows
        _linear("linear_prompt", "fwd", "bf16", 5, 12, 1330, 64, 64, layout="packed", continued=True, ragged=True),
        # fp32 with tangents, contiguous tensors, an odd length
        _linear("linear_fp32", "jvp", "fp32", 2, 8, 1023, 128, 128, layout="bhld", api="fwad"),
        # the headline configuration's projections, a JVP-consistency training step
        _linear("linear_step", "jvp_bwd", "bf16", 4, 16, 2048, 64, 64),
        # ordinary training on the long-sequence configuration's projections
        _linear("linear_long", "fwd_bwd", "bf16", 4, 16, 8192, 128, 128),
        # the next token of four sequences: the time of a call
        _token("tokens_few", "bf16", 4, 16, 64, 64),
        # the next token of a full batch: the states are read and written, and little else
        _token("tokens_many", "bf16", 256, 16, 128, 128),
    ]


def draw(rng):
    """One more case of the same ranges: from one row to long sequences, odd sizes among them, every type, norm, layout and form, at
    no more work than the largest listed."""
    dtype, op = rng.choice(["bf16", "bf16", "fp16", "fp32"]), rng.choice(["norm", "residual", "linear", "linear", "token"])
    step, api = rng.choice(["fwd", "fwd_bwd", "jvp", "jvp_bwd"]), rng.choice(["func", "fwad"])
    most = {c["name"]: work(c) for c in listed()}
    while True:
        B = rng.randint(1, 8)
        if op in ("norm", "residual"):
            C = round(2 ** rng.uniform(3, 13))
            if rng.random() < 0.6:  # widths are mostly multiples of eight
                C = C // 8 * 8
            case = _norm("", step, dtype, B, round(2 ** rng.uniform(0, 13)), C, rng.choice(["rms", "layer"]), rng.random() < 0.5,
                         rng.random() < 0.5, api)
            if op == "residual":
                case = _residual("", step, dtype, B, case["L"], C, case["kind"], rng.choice(["", "", "rms", "layer"]), case["weights"],
                                 case["modulated"], rng.random() < 0.6, rng.choice([1.0, 0.5]), api)
            fits = work(case)["bytes"] <= most["residual_wide"]["bytes"]
        elif op == "linear":
            D = rng.choice([32, 64, 64, 128, rng.randint(8, 128)])
            continued = step.startswith("fwd") and rng.random() < 0.5
            case = _linear("", step, dtype, B, rng.randint(1, 16), round(2 ** rng.uniform(0, 13)), D,
                           rng.choice([D, D, D, rng.choice([32, 64, 128])]), rng.choice(["bhld", "blhd", "packed"]), api,
                           rng.random() < 0.8, continued, step == "fwd" and rng.random() < 0.5)
            fits = work(case)["flops"] <= most["linear_long"]["flops"] / (4 if dtype == "fp32" else 1)
        else:
            D = rng.choice([32, 64, 64, 128, rng.randint(8, 128)])
            case = _token("", dtype, round(2 ** rng.uniform(0, 8)), rng.randint(1, 16), D, rng.choice([D, D, rng.choice([32, 64, 128])]),
                          rng.random() < 0.8)
            fits = work(case)["bytes"] <= most["tokens_many"]["bytes"]
        if fits:
            del case["name"]
            return case


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    dual, back = case["step"].startswith("jvp"), case["step"].endswith("bwd")
    sides = (2 if dual else 1) * (2 if back else 1)  # values, their tangents, and the gradients of both
    if case["op"] == "token":
        n, D, E = case["B"] * case["H"], case["D"], case["E"]
        return {"bytes": n * (2 * D + 2 * E) * size + 2 * n * D * E * 4, "flops": 5 * n * D * E}
    if case["op"] == "linear":
        n, D, E = case["B"] * case["H"], case["D"], case["E"]
        rows = n * (3 * case["L"] // 4 if case["ragged"] else case["L"])
        tensors = rows * (2 * D + E) * sides + rows * E * sides  # q, k, v and the result; their gradients and its cotangent
        states = 2 * n * D * E * (2 if back else 1) if case["continued"] else 0
        products = (2 + 5 if back else 2) * (3 if dual else 1)  # of 2 D E for each row: state, result; state, dq, its reverse, dk, dv
        return {"bytes": tensors * size + 4 * states, "flops": 2 * D * E * rows * products}
    n = case["B"] * case["L"] * case["C"]
    tensors = 2 if case["op"] == "norm" else 4
    vectors = (case["weights"] * (2 if case["kind"] == "layer" else 1) + (case.get("post", "") != "")) * case["C"]
    vectors += (2 * case["modulated"] + case.get("gated", False)) * case["B"] * case["C"] * (2 if dual else 1)
    return {"bytes": (tensors * n * sides + vectors * (2 if back else 1)) * size, "flops": 8 * tensors * n * sides}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def randn(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)

    state = dict(case)
    grad, B = case["step"].endswith("bwd"), case["B"]
    if case["op"] in ("norm", "residual"):
        L, C = case["L"], case["C"]
        rows, one = (B, L, C), (B, 1, C)
        shapes = {"x": rows}
        if case["op"] == "residual":
            shapes["y"] = rows
            if case["gated"]:
                shapes["gate"] = one
        if case["modulated"]:
            shapes |= {"scale": one, "shift": one}
        std = {"x": 2.0, "y": 1.0, "gate": 0.5, "scale": 0.3, "shift": 0.3}
        state["names"] = tuple(shapes)
        state["primals"] = tuple(randn(*s, std=std[n]).requires_grad_(grad) for n, s in shapes.items())
        state["tangents"] = tuple(randn(*s, std=TANGENT_STD).requires_grad_(grad) for s in shapes.values())
        weights = {}
        if case["weights"]:
            weights["weight"] = 1 + randn(C, std=0.1)
            if case["kind"] == "layer":
                weights["bias"] = randn(C, std=0.1)
        if case.get("post"):
            weights["post_weight"] = 1 + randn(C, std=0.1)
        state["weights"] = {n: w.requires_grad_(grad) for n, w in weights.items()}
        state["cotangents"] = tuple(randn(*rows) for _ in range(4))
        return state
    H, D, E = case["H"], case["D"], case["E"]
    # a head's memory: from 32 rows to 4096
    state["log_decay"] = torch.log1p(-torch.exp2(-5 - 7 * torch.arange(H, device="cuda") / max(H - 1, 1))) if case["decay"] else None
    if case["op"] == "token":
        both = randn(B, H, 2 * D)
        state["qkv"] = (both[..., :D], both[..., D:], randn(B, H, E))
        state["state"] = torch.randn(B, H, D, E, generator=g, device="cuda") * 4
        return state
    L = case["L"]

    def projections(std):
        if case["layout"] == "packed" and D == E:
            x = randn(B, L, 3 * H, D, std=std).transpose(1, 2)
            return x[:, :H], x[:, H:2 * H], x[:, 2 * H:]
        if case["layout"] == "bhld":
            return randn(B, H, L, D, std=std), randn(B, H, L, D, std=std), randn(B, H, L, E, std=std)
        return tuple(randn(B, L, H, w, std=std).transpose(1, 2) for w in (D, D, E))

    state["primals"] = tuple(x.detach().requires_grad_(grad) for x in projections(1.0))
    state["tangents"] = tuple(x.detach().requires_grad_(grad) for x in projections(TANGENT_STD))
    state["cotangents"] = tuple(randn(B, H, L, E) for _ in range(2))
    state["lengths"] = torch.randint(L // 2, L + 1, (B,), generator=g, device="cuda", dtype=torch.int32) if case["ragged"] else None
    if case["continued"]:
        state["state"] = (torch.randn(B, H, D, E, generator=g, device="cuda") * 4).requires_grad_(grad)
        state["state_cotangent"] = torch.randn(B, H, D, E, generator=g, device="cuda")
    return state


# ---- plain forms: norms ----------------------------------------------------------------------------------------------------
def _normed(x, kind):
    """n of the rows, and 1 / their deviation."""
    x = x - x.mean(-1, keepdim=True) if kind == "layer" else x
    s = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return x * s, s


def _along(v, n, s, kind):
    """The derivative of n along v, which is a symmetric map of v."""
    v = v - v.mean(-1, keepdim=True) if kind == "layer" else v
    return s * (v - n * (n * v).mean(-1, keepdim=True))


def _norm_backward(gn, gtn, n, s, tx, kind):
    """The gradients of <gn, n> + <gtn, tn> with respect to x and tx."""
    if gtn is None:
        return _along(gn, n, s, kind), None
    tn = _along(tx, n, s, kind)
    a, b, e = ((n * gtn).mean(-1, keepdim=True), (n * tx).mean(-1, keepdim=True), (gtn * tn).mean(-1, keepdim=True))
    return _along(gn - s * b * gtn, n, s, kind) - s * (a * tn + e * n), _along(gtn, n, s, kind)


def _of_sequence(x):
    return x.sum(1, keepdim=True)


def _of_channel(x):
    return x.sum((0, 1))


def _plain_norms(state):
    """Norm, or the residual sum and its norm, with tangents and gradients as the step asks."""
    dtype, kind, post, alpha = state["primals"][0].dtype, state["kind"], state.get("post", ""), state.get("alpha", 1.0)
    dual, back, residual = state["step"].startswith("jvp"), state["step"].endswith("bwd"), state["op"] == "residual"
    p = {n: t.float() for n, t in zip(state["names"], state["primals"])}
    t = {n: v.float() for n, v in zip(state["names"], state["tangents"])} if dual else {}
    w = {n: v.float() for n, v in state["weights"].items()}
    weight, bias, post_weight = w.get("weight", 1.0), w.get("bias", 0.0), w.get("post_weight", 1.0)
    scale, shift, gate = 1 + p.get("scale", 0.0), p.get("shift", 0.0), alpha * p.get("gate", 1.0)
    tscale, tshift, tgate = t.get("scale", 0.0), t.get("shift", 0.0), alpha * t.get("gate", 0.0)
    # values and tangents
    r, tr, out = p["x"], t.get("x"), []
    if residual:
        m, ms = _normed(p["y"], post) if post else (p["y"], 1.0)
        r = r + gate * post_weight * m
        out.append(r)
        if dual:
            tm = _along(t["y"], m, ms, post) if post else t["y"]
            tr = tr + post_weight * (tgate * m + gate * tm)
    n, s = _normed(r, kind)
    gain, offset = weight * scale, bias * scale + shift
    out.append(n * gain + offset)
    if dual:
        tn, tgain = _along(tr, n, s, kind), weight * tscale
        out += [tr] * residual + [tn * gain + n * tgain + bias * tscale + tshift]
    if not back:
        return tuple(o.to(dtype) for o in out)
    # gradients: first of what the norm answered, then of the sum
    cots = [c.float() for c in state["cotangents"]]
    gr, gn = (cots[0], cots[1]) if residual else (0.0, cots[0])
    gtr, gtn = ((cots[2], cots[3]) if residual else (0.0, cots[1])) if dual else (None, None)
    dn = gn * gain + (gtn * tgain if dual else 0.0)
    dr, dtr = _norm_backward(dn, gtn * gain if dual else None, n, s, tr, kind)
    dr, dtr = dr + gr, dtr + gtr if dual else None
    d, dt, dw = {"x": dr}, {"x": dtr}, {}
    both = gn * n + (gtn * tn if dual else 0.0)
    if state["modulated"]:
        d |= {"scale": _of_sequence(both * weight + gn * bias), "shift": _of_sequence(gn)}
        if dual:
            dt |= {"scale": _of_sequence(gtn * (n * weight + bias)), "shift": _of_sequence(gtn)}
    if "weight" in w:
        dw["weight"] = _of_channel(both * scale + (gtn * n * tscale if dual else 0.0))
    if "bias" in w:
        dw["bias"] = _of_channel(gn * scale + (gtn * tscale if dual else 0.0))
    if residual:
        by_m = dr * m + (dtr * tm if dual else 0.0)
        if state["gated"]:
            d["gate"] = _of_sequence(alpha * post_weight * by_m)
            if dual:
                dt["gate"] = _of_sequence(alpha * post_weight * dtr * m)
        if post:
            dw["post_weight"] = _of_channel(gate * by_m + (tgate * dtr * m if dual else 0.0))
        dm, dtm = post_weight * (dr * gate + (dtr * tgate if dual else 0.0)), post_weight * gate * dtr if dual else None
        d["y"], dt["y"] = _norm_backward(dm, dtm, m, ms, t.get("y"), post) if post else (dm, dtm)
    grads = [d[n] for n in state["names"]] + ([dt[n] for n in state["names"]] if dual else []) + [dw[n] for n in w]
    return tuple(o.to(dtype) for o in out + grads)


# ---- plain forms: linear attention -------------------------------------------------------------------------------------------
def _chunks(x, lead):
    """(B, H, N, CHUNK, width) in 32 bits, `lead` rows of zeros in front."""
    L = x.shape[2]
    x = torch.nn.functional.pad(x.float(), (0, 0, lead, -(L + lead) % CHUNK))
    return x.unflatten(2, (-1, CHUNK))


def _scan(a, b, c, w, first=None, ahead=1, backwards=False, rows=None):
    """``out_t = sum_{s <= t} exp(w (t - s)) (a_t . b_s) c_s + exp(w (t + ahead)) a_t first`` and the state behind the last row,
    ``sum_s exp(w (L - 1 - s)) b_s c_s^T + exp(w (L - 1 + ahead)) first``; backwards: with the rows in reverse order.  rows: which row
    of its sequence stands at each place, (B, L), where sequences begin late."""
    L, H = a.shape[2], a.shape[1]
    rows = torch.arange(L, device=a.device)[None] if rows is None else rows
    if backwards:
        a, b, c = (x.flip(2) for x in (a, b, c))
    w = (torch.zeros(H, device=a.device) if w is None else w)[:, None, None]
    old = 0.0
    if first is not None:
        old = torch.exp(w * (rows + ahead).clamp(min=0)[:, None, :, None]) * (a.float() @ first.float())
    w = w[..., None]  # of (H, N, rows, ...)
    lead = -L % CHUNK  # places in front: the last chunk is full, so that its state is the last row's
    a, b, c = (_chunks(x, lead) for x in (a, b, c))
    i, j = torch.arange(CHUNK, device=a.device), torch.arange(a.shape[2], device=a.device)
    apart, chunks = i[:, None] - i, j[:, None] - j
    inside = torch.where(apart >= 0, torch.exp(w * apart.clamp(min=0)), 0.0)
    out = ((a @ b.transpose(-1, -2)) * inside) @ c
    added = (b * torch.exp(w * (CHUNK - 1 - i)[:, None])).transpose(-1, -2) @ c  # by each chunk, seen from its last row
    between = torch.where(chunks >= 0, torch.exp(w[:, 0] * (chunks.clamp(min=0) * CHUNK)), 0.0)  # (H, N, N)
    states = (between @ added.flatten(-2)).unflatten(-1, added.shape[-2:])  # behind each chunk's last row
    before = torch.nn.functional.pad(states[:, :, :-1], (0, 0, 0, 0, 1, 0))
    out = (out + torch.exp(w * (i + 1)[:, None]) * (a @ before)).flatten(2, 3)[:, :, lead:] + old
    last = states[:, :, -1]
    if first is not None:
        last = last + torch.exp(w[:, 0] * (rows[:, -1] + ahead)[:, None, None, None]) * first.float()
    return (out.flip(2) if backwards else out), last


def _plain_linear(state):
    dtype, w, first = state["primals"][0].dtype, state["log_decay"], state.get("state")
    q, k, v = (x.float() for x in state["primals"])
    q = q * q.shape[-1] ** -0.5
    out, lengths, row = [], state["lengths"], None
    if lengths is not None:  # the rows of a sequence end at its length: the others are moved in front of it, as zeros
        L = q.shape[2]
        row = torch.arange(L, device=q.device) - (L - lengths[:, None])  # of the place, in its sequence
        q, k, v = (x.gather(2, row.clamp(min=0)[:, None, :, None].expand_as(x)) * (row >= 0)[:, None, :, None] for x in (q, k, v))
    o, last = _scan(q, k, v, w, first, rows=row)
    if lengths is not None:
        place = torch.arange(L, device=q.device) + (L - lengths[:, None])
        o = o.gather(2, place.clamp(max=L - 1)[:, None, :, None].expand_as(o)) * (place < L)[:, None, :, None]
    out.append(o)
    if first is not None:
        out.append(last)
    dual, back = state["step"].startswith("jvp"), state["step"].endswith("bwd")
    if dual:
        tq, tk, tv = (x.float() for x in state["tangents"])
        tq = tq * q.shape[-1] ** -0.5
        out.append(_scan(tq, k, v, w)[0] + _scan(q, tk, v, w)[0] + _scan(q, k, tv, w)[0])
    if back:
        go, gto = (c.float() for c in state["cotangents"])
        glast = state["state_cotangent"] if first is not None else None
        flip = lambda x: None if x is None else x.transpose(-1, -2)  # noqa: E731
        dq = _scan(go, v, k, w, flip(first))[0]
        dk, dfirst = _scan(v, go, q, w, flip(glast), 0, True)
        dv = _scan(k, q, go, w, glast, 0, True)[0]
        if dual:
            dtq, dtk, dtv = _scan(gto, v, k, w)[0], _scan(v, gto, q, w, None, 0, True)[0], _scan(k, q, gto, w, None, 0, True)[0]
            dq = dq + _scan(gto, tv, k, w)[0] + _scan(gto, v, tk, w)[0]
            dk = dk + _scan(tv, gto, q, w, None, 0, True)[0] + _scan(v, gto, tq, w, None, 0, True)[0]
            dv = dv + _scan(tk, q, gto, w, None, 0, True)[0] + _scan(k, tq, gto, w, None, 0, True)[0]
        by = q.shape[-1] ** -0.5
        out += [dq * by, dk, dv]
        if dual:
            out += [dtq * by, dtk, dtv]
        if first is not None:
            out.append(flip(dfirst) * (1.0 if w is None else torch.exp(w)[:, None, None]))
    keep = 1 if first is not None else None  # the states stay in 32 bits
    last = len(out) - 1 if first is not None and back else None
    return tuple(x if i in (keep, last) else x.to(dtype) for i, x in enumerate(out))


def _plain_token(state):
    (q, k, v), s = (x.float() for x in state["qkv"]), state["state"]
    if state["log_decay"] is not None:
        s *= torch.exp(state["log_decay"])[:, None, None]
    s += k[..., :, None] * v[..., None, :]
    o = (q[..., None, :] * q.shape[-1] ** -0.5 @ s)[..., 0, :]
    return o.to(state["qkv"][0].dtype), s


# ---- the framework's -----------------------------------------------------------------------------------------------------
def _with_tangents(f, state):
    """Values and tangents of f along the state's tangents, flat: the values first."""
    if state["api"] == "func":
        out, tangents = torch.func.jvp(f, state["primals"], state["tangents"])
    else:
        with fwAD.dual_level():
            out = f(*map(fwAD.make_dual, state["primals"], state["tangents"]))
            if isinstance(out, torch.Tensor):
                return tuple(fwAD.unpack_dual(out))
            out, tangents = zip(*map(fwAD.unpack_dual, out))
    return (out, tangents) if isinstance(out, torch.Tensor) else (*out, *tangents)


def _own(state, f, weights=(), cotangents=None):
    """A pass through f, which takes the state's primals and answers with one tensor or several."""
    step = state["step"]
    if not step.endswith("bwd"):
        with torch.no_grad():
            out = f(*state["primals"]) if step == "fwd" else _with_tangents(f, state)
        return (out,) if isinstance(out, torch.Tensor) else tuple(out)
    out = f(*state["primals"]) if step == "fwd_bwd" else _with_tangents(f, state)
    out = (out,) if isinstance(out, torch.Tensor) else tuple(out)
    leaves = state["primals"] + (state["tangents"] if step == "jvp_bwd" else ()) + tuple(weights)
    cotangents = state["cotangents"][:len(out)] if cotangents is None else cotangents
    return (*(o.detach() for o in out), *torch.autograd.grad(out, leaves, cotangents))


def _own_norms(state):
    from jvp_flash_attention_b200.norms import norm, residual_norm

    names, weights, kind = state["names"], state["weights"], state["kind"]
    if state["op"] == "norm":
        return _own(state, lambda x, *more: norm(x, **dict(zip(names[1:], more)), **weights, kind=kind, eps=EPS), weights.values())
    return _own(state, lambda x, y, *more: residual_norm(x, y, **dict(zip(names[2:], more)), **weights, kind=kind, post=state["post"] or None,
                                                         alpha=state["alpha"], eps=EPS), weights.values())


def _own_linear(state):
    from jvp_flash_attention_b200.linear_attention import linear_attention

    w, lengths, first = state["log_decay"], state["lengths"], state.get("state")
    if first is None:
        return _own(state, lambda q, k, v: linear_attention(q, k, v, w, lengths=lengths))
    cotangents = (state["cotangents"][0], state["state_cotangent"])
    return _own(state, lambda q, k, v: linear_attention(q, k, v, w, state=first, lengths=lengths, return_state=True), (first,), cotangents)


def run(state):
    if not own:
        with torch.no_grad():
            if state["op"] == "token":
                return _plain_token(state)
            return _plain_linear(state) if state["op"] == "linear" else _plain_norms(state)
    if state["op"] == "token":
        from jvp_flash_attention_b200.linear_attention import linear_attention_step

        return linear_attention_step(*state["qkv"], state["log_decay"], state["state"]), state["state"]
    return _own_linear(state) if state["op"] == "linear" else _own_norms(state)


# ---- in 64 bits ----------------------------------------------------------------------------------------------------------
def _differentiated(f, state, weights, cotangents):
    """Values, tangents and gradients of f(primals, weights) by torch's own differentiation; a value that is a tuple has several."""
    step = state["step"]
    leaf = lambda t: t.detach().double().requires_grad_(step.endswith("bwd"))  # noqa: E731
    primals, tangents, weights = (tuple(map(leaf, ts)) for ts in (state["primals"], state["tangents"], weights))
    if step.startswith("jvp"):
        out = [t for part in torch.func.jvp(lambda *p: f(p, weights), primals, tangents) for t in part]
    else:
        out = list(f(primals, weights))
    if not step.endswith("bwd"):
        return tuple(out)
    leaves = (*primals, *(tangents if step == "jvp_bwd" else ()), *weights)
    grads = torch.autograd.grad(out, leaves, [c.double() for c in cotangents[:len(out)]])
    return (*(o.detach() for o in out), *grads)


def _exact_norms(state):
    names, which = state["names"], tuple(state["weights"])

    def rms(x):
        return x / (x.square().mean(-1, keepdim=True) + EPS).sqrt()

    def layer(x):
        x = x - x.mean(-1, keepdim=True)
        return x / (x.square().mean(-1, keepdim=True) + EPS).sqrt()

    kinds = {"rms": rms, "layer": layer, "": lambda x: x}

    def value(primals, weights):
        p, w = dict(zip(names, primals)), dict(zip(which, weights))
        x = p["x"]
        if state["op"] == "residual":
            x = x + state["alpha"] * p.get("gate", 1.0) * (kinds[state["post"]](p["y"]) * w.get("post_weight", 1.0))
        n = kinds[state["kind"]](x) * w.get("weight", 1.0) + w.get("bias", 0.0)
        if "scale" in p:
            n = n * (1 + p["scale"]) + p["shift"]
        return (x, n) if state["op"] == "residual" else (n,)

    return _differentiated(value, state, tuple(state["weights"].values()), state["cotangents"])


def _exact_linear(state):
    """Every head by its matrix of weights over all pairs of rows."""
    B, H, L, _ = state["primals"][0].shape
    first, lengths, keep_last = state.get("state"), state["lengths"], state["continued"]

    def head(b, h):
        n = L if lengths is None else int(lengths[b])
        w = 0.0 if state["log_decay"] is None else state["log_decay"][h].double()
        t = torch.arange(L, device="cuda", dtype=torch.float64)
        live = (t < n).double()[:, None]
        weight = torch.exp(w * (t[:, None] - t)).tril() if not torch.is_tensor(w) else torch.exp(w * (t[:, None] - t).clamp(min=0)).tril()

        def value(primals, rest):
            q, k, v = primals
            q = q * live / math.sqrt(q.shape[-1])
            o = (q @ k.T * weight) @ (v * live)
            if not keep_last:
                return (o,)
            o = o + torch.exp(w * (t + 1))[:, None] * (q @ rest[0])
            last = (k * live * torch.exp(w * (n - 1 - t).clamp(min=0))[:, None]).T @ (v * live)
            return o, last + torch.exp(torch.as_tensor(w * n, device="cuda", dtype=torch.float64)) * rest[0]

        one = {"step": state["step"], "primals": [x[b, h] for x in state["primals"]], "tangents": [x[b, h] for x in state["tangents"]]}
        cots = [c[b, h] for c in state["cotangents"]]
        if keep_last:
            cots = [cots[0], state["state_cotangent"][b, h]]
        return _differentiated(value, one, [first[b, h]] if keep_last else [], cots)

    heads = [head(b, h) for b in range(B) for h in range(H)]
    return tuple(torch.stack(xs).unflatten(0, (B, H)) for xs in zip(*heads))


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "token":
        (q, k, v), s = (x.double() for x in state["qkv"]), state["state"].double()
        by = 1.0 if state["log_decay"] is None else torch.exp(state["log_decay"].double())[None, :, None, None]
        s = by * s + torch.einsum("bhd,bhe->bhde", k, v)
        return torch.einsum("bhd,bhde->bhe", q, s) / math.sqrt(q.shape[-1]), s
    return _exact_linear(state) if case["op"] == "linear" else _exact_norms(state)
