"""Performance cases of the operators that stand beside attention in a transformer block: rotary positions and gated projections.

A case names one pass through one of them, in one of the forms that attention has:

* ``op``     ``rotary``  queries and keys (and their tangents) turned by their positions
             ``gated``   ``a(x Wg^T) * (x Wu^T)``, the widening half of a gated feed-forward block
* ``step``   ``fwd``      the value without gradients (inference)
             ``fwd_bwd``  the value and the gradients with respect to every floating-point input (ordinary training)
             ``jvp``      value and tangent (sampling, forward-mode probes)
             ``jvp_bwd``  value and tangent, and the gradients through both with respect to inputs, tangents and weights
* ``api``    how the tangents travel: ``func`` = ``torch.func.jvp``, ``fwad`` = ``torch.autograd.forward_ad`` dual tensors
* ``layout`` ``bhld`` contiguous queries and keys, ``blhd`` the (B, H, L, D) views of (B, L, H, D) projections, ``packed`` the views
             of one (B, L, H + 2 Hk, D) projection

The cotangents are inputs: in a model they arrive from the layers above.
"""
from __future__ import annotations

import math

import torch
import torch.autograd.forward_ad as fwAD

own = False
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
TANGENT_STD = 0.1


def _rotary(name, step, dtype, B, H, Hk, L, D, rot, pairs="half", layout="blhd", api="func", start=0, ragged=False, stretch=1.0):
    return {"name": name, "op": "rotary", "step": step, "dtype": dtype, "B": B, "H": H, "Hk": Hk, "L": L, "D": D, "rot": rot,
            "pairs": pairs, "layout": layout, "api": api, "start": start, "ragged": ragged, "stretch": stretch}


def _gated(name, step, dtype, M, K, F, activation="silu", api="func"):
    return {"name": name, "op": "gated", "step": step, "dtype": dtype, "M": M, "K": K, "F": F, "activation": activation, "api": api}


def listed():
    return [
        # one new token of each of eight sequences, far into their contexts: the time of a call
        _rotary("rotary_token", "fwd", "bf16", 8, 16, 16, 1, 64, 64, start=100_000, ragged=True),
        # the headline configuration's queries and keys, a JVP-consistency training step
        _rotary("rotary_step", "jvp_bwd", "bf16", 4, 16, 16, 2048, 64, 64),
        # ordinary training at a length that no tile divides, shared key heads, half of the head turned, neighbours as pairs
        _rotary("rotary_train_ragged", "fwd_bwd", "fp16", 3, 12, 4, 1330, 64, 32, pairs="neighbours", layout="packed"),
        # fp32 with tangents, contiguous tensors, an odd length and positions of each sequence's own
        _rotary("rotary_fp32", "jvp", "fp32", 2, 8, 8, 1023, 128, 128, pairs="neighbours", layout="bhld", api="fwad", ragged=True),
        # the long-sequence configuration's queries and keys on one GPU, stretched to a longer context
        _rotary("rotary_long", "jvp", "bf16", 4, 16, 16, 8192, 128, 128, stretch=8.0),
        # one token through a block of generic width: the weights are read, and little else
        _gated("gated_token", "fwd", "bf16", 1, 4096, 11008),
        # a few tokens with their tangents (a probe along one direction)
        _gated("gated_few", "jvp", "fp16", 24, 1024, 2736, activation="gelu", api="fwad"),
        # the key-padding configuration's block in fp32, ordinary training on one of its sequences
        _gated("gated_fp32", "fwd_bwd", "fp32", 1024, 768, 2048, activation="gelu_tanh"),
        # tokens and a width that no tile divides
        _gated("gated_ragged", "fwd_bwd", "fp16", 3990, 1024, 2731),
        # the headline configuration's block, a JVP-consistency training step
        _gated("gated_step", "jvp_bwd", "bf16", 8192, 1024, 2736),
        # the long-sequence configuration's block: value and tangent of one sequence
        _gated("gated_long", "jvp", "bf16", 8192, 2048, 5464, activation="gelu_tanh", api="fwad"),
        # ordinary training of a block of generic width
        _gated("gated_wide", "fwd_bwd", "bf16", 8192, 4096, 11008),
    ]


def draw(rng):
    """One more case of the same ranges: from one token to long sequences, odd sizes among them, every type, layout, form and
    activation, at no more work than the largest listed."""
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    step, api = rng.choice(["fwd", "fwd_bwd", "jvp", "jvp_bwd"]), rng.choice(["func", "fwad"])
    while True:
        if rng.random() < 0.45:
            D = rng.choice([32, 64, 64, 96, 128, 128])
            Hk = rng.randint(1, 16)
            case = _rotary("", step, dtype, rng.randint(1, 8), Hk * rng.choice([1, 1, 2, 4]), Hk, round(2 ** rng.uniform(0, 13)), D,
                           rng.choice([D, D, D // 2, 2 * rng.randint(1, D // 2)]), rng.choice(["half", "neighbours"]),
                           rng.choice(["bhld", "blhd", "packed"]), api, rng.choice([0, 0, rng.randint(1, 1_000_000)]),
                           rng.random() < 0.4, rng.choice([1.0, 1.0, 4.0]))
            most = work(listed()[4])["bytes"]
            fits = work(case)["bytes"] <= most
        else:
            M, K, F = round(2 ** rng.uniform(0, 13.3)), round(2 ** rng.uniform(6, 12.3)), round(2 ** rng.uniform(7, 13.5))
            if rng.random() < 0.6:  # widths are mostly multiples of eight
                K, F = max(8, K // 8 * 8), max(8, F // 8 * 8)
            case = _gated("", step, dtype, M, K, F, rng.choice(["silu", "silu", "gelu", "gelu_tanh", "sigmoid"]), api)
            fits = work(case)["flops"] <= work(listed()[-1])["flops"] / (4 if dtype == "fp32" else 1)
        if fits:
            del case["name"]
            return case


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    step = case["step"]
    dual = step.startswith("jvp")
    if case["op"] == "rotary":
        n = case["B"] * (case["H"] + case["Hk"]) * case["L"] * case["D"]
        tensors = (2 if dual else 1) * (2 if step.endswith("bwd") else 1)  # each read and written
        turned = n // case["D"] * case["rot"]
        return {"bytes": 2 * tensors * n * size, "flops": 3 * tensors * turned}
    M, K, F = case["M"], case["K"], case["F"]
    rows = 2 * M if dual else M
    values = rows * K + 2 * F * K + rows * F
    flops = 4 * rows * K * F
    if step.endswith("bwd"):  # the cotangents, and the gradients of all that was read
        values += rows * F + rows * K + 2 * F * K
        flops *= 3
    return {"bytes": values * size, "flops": flops}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def randn(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)

    state = {k: case[k] for k in ("op", "step", "api")}
    grad = case["step"].endswith("bwd")
    if case["op"] == "gated":
        M, K, F = case["M"], case["K"], case["F"]
        state["activation"] = case["activation"]
        state["weights"] = tuple(randn(F, K, std=K**-0.5).requires_grad_(grad) for _ in range(2))
        state["primals"] = (randn(M, K).requires_grad_(grad),)
        state["tangents"] = (randn(M, K, std=TANGENT_STD).requires_grad_(grad),)
        state["cotangents"] = tuple(randn(M, F) for _ in range(2))
        return state
    B, H, Hk, L, D = (case[k] for k in ("B", "H", "Hk", "L", "D"))

    def queries_and_keys(std):
        if case["layout"] == "bhld":
            return randn(B, H, L, D, std=std), randn(B, Hk, L, D, std=std)
        if case["layout"] == "blhd":
            return randn(B, L, H, D, std=std).transpose(1, 2), randn(B, L, Hk, D, std=std).transpose(1, 2)
        x = randn(B, L, H + 2 * Hk, D, std=std).transpose(1, 2)
        return x[:, :H], x[:, H:H + Hk]

    state["primals"] = tuple(x.detach().requires_grad_(grad) for x in queries_and_keys(1.0))
    state["tangents"] = tuple(x.detach().requires_grad_(grad) for x in queries_and_keys(TANGENT_STD))
    state["cotangents"] = (randn(B, H, L, D), randn(B, Hk, L, D), randn(B, H, L, D), randn(B, Hk, L, D))
    positions = torch.arange(L, device="cuda") + case["start"]
    if case["ragged"]:  # every sequence begins at a place of its own
        positions = positions[None, :] + torch.randint(0, 1000, (B, 1), generator=g, device="cuda")
    state["positions"] = positions
    state["frequencies"] = _frequencies(case["rot"], case["stretch"])
    state["amplitude"] = 1.0 + 0.1 * math.log(case["stretch"])
    state["neighbours"] = case["pairs"] == "neighbours"
    return state


def _frequencies(rot, stretch):
    """Radians per position of each pair.  A context that is stretched keeps its quick pairs and slows its slow ones down, by a ramp
    over the turns that a pair makes in the original 4096 positions."""
    w = 10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    turns = 4096 * w / (2 * math.pi)
    keep = ((turns - 1) / 31).clamp(0, 1)
    return w * keep + w / stretch * (1 - keep)


# ---- plain forms ---------------------------------------------------------------------------------------------------------
def _turn(x, cos, sin, neighbours):
    """x * cos + (x turned by a quarter) * sin on the first 2 * cos.shape[-1] entries of the last dimension, in 32 bits."""
    rot = 2 * cos.shape[-1]
    t = x[..., :rot].float()
    a, b = (t[..., 0::2], t[..., 1::2]) if neighbours else (t[..., :rot // 2], t[..., rot // 2:])
    a, b = a * cos - b * sin, a * sin + b * cos
    t = torch.stack((a, b), -1).flatten(-2) if neighbours else torch.cat((a, b), -1)
    return torch.cat((t, x[..., rot:].float()), -1).to(x.dtype)


def _plain_rotary(state):
    angles = state["positions"].double()[..., None] * state["frequencies"]  # 64 bits: far positions
    cos, sin = (f(angles).mul(state["amplitude"]).float() for f in (torch.cos, torch.sin))
    if cos.dim() == 3:
        cos, sin = cos[:, None], sin[:, None]
    tensors = state["primals"] + (state["tangents"] if state["step"].startswith("jvp") else ())
    out = [_turn(x, cos, sin, state["neighbours"]) for x in tensors]
    if state["step"].endswith("bwd"):  # the transposed turn
        out += [_turn(x, cos, -sin, state["neighbours"]) for x in state["cotangents"][:len(tensors)]]
    return tuple(out)


def _activation(kind, g):
    """a, a' and a'' at g."""
    if kind in ("silu", "sigmoid"):
        s = torch.sigmoid(g)
        d = s * (1 - s)
        if kind == "sigmoid":
            return s, d, d * (1 - 2 * s)
        return g * s, s + g * d, d * (2 + g * (1 - 2 * s))
    if kind == "gelu":
        p, d = 0.5 * (1 + torch.erf(g * 0.5**0.5)), torch.exp(-0.5 * g * g) * (2 * math.pi) ** -0.5
        return g * p, p + g * d, d * (2 - g * g)
    c, c3 = (2 / math.pi) ** 0.5, 0.044715
    t = torch.tanh(c * (g + c3 * g**3))
    i, d = c * (1 + 3 * c3 * g * g), 1 - t * t
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * d * i, d * i + 0.5 * g * (d * 6 * c * c3 * g - 2 * t * d * i * i)


def _plain_gated(state):
    (x,), (tx,), (wg, wu) = state["primals"], state["tangents"], state["weights"]
    dtype, step = x.dtype, state["step"]
    x, tx, wg, wu, gh, gth = (t.float() for t in (x, tx, wg, wu, *state["cotangents"]))
    g, u = x @ wg.T, x @ wu.T
    a, a1, a2 = _activation(state["activation"], g)
    out = [a * u]
    if step.startswith("jvp"):
        tg, tu = tx @ wg.T, tx @ wu.T
        out.append(a1 * tg * u + a * tu)
    if step == "fwd_bwd":
        dg, du = gh * a1 * u, gh * a
        out += [dg @ wg + du @ wu, dg.T @ x, du.T @ x]
    if step == "jvp_bwd":
        dg = gh * a1 * u + gth * (a2 * tg * u + a1 * tu)
        du = gh * a + gth * a1 * tg
        dtg, dtu = gth * a1 * u, gth * a
        out += [dg @ wg + du @ wu, dtg @ wg + dtu @ wu, dg.T @ x + dtg.T @ tx, du.T @ x + dtu.T @ tx]
    return tuple(t.to(dtype) for t in out)


# ---- the framework's -----------------------------------------------------------------------------------------------------
def _with_tangents(f, state):
    """Values and tangents of f along the state's tangents."""
    if state["api"] == "func":
        return torch.func.jvp(f, state["primals"], state["tangents"])
    with fwAD.dual_level():
        out = f(*(fwAD.make_dual(p, t) for p, t in zip(state["primals"], state["tangents"])))
        if isinstance(out, torch.Tensor):
            return tuple(fwAD.unpack_dual(out))
        return tuple(zip(*(tuple(fwAD.unpack_dual(o)) for o in out)))


def _own(state, f):
    """A pass through f, which takes the state's primals and answers with one tensor or several."""
    step = state["step"]
    if not step.endswith("bwd"):
        with torch.no_grad():
            out = f(*state["primals"]) if step == "fwd" else _with_tangents(f, state)
    else:
        out = f(*state["primals"]) if step == "fwd_bwd" else _with_tangents(f, state)
    flat = []
    for o in (out,) if isinstance(out, torch.Tensor) else out:
        flat += [o] if isinstance(o, torch.Tensor) else list(o)
    if not step.endswith("bwd"):
        return tuple(flat)
    leaves = state["primals"] + (state["tangents"] if step == "jvp_bwd" else ()) + state.get("weights", ())
    return (*(o.detach() for o in flat), *torch.autograd.grad(flat, leaves, state["cotangents"][:len(flat)]))


def run(state):
    if not own:
        with torch.no_grad():
            return _plain_rotary(state) if state["op"] == "rotary" else _plain_gated(state)
    if state["op"] == "rotary":
        from jvp_flash_attention_b200.rotary import rotary

        return _own(state, lambda q, k: rotary(q, k, state["frequencies"], state["positions"], interleaved=state["neighbours"],
                                               amplitude=state["amplitude"]))
    from jvp_flash_attention_b200.gated import gated_linear

    return _own(state, lambda x: gated_linear(x, *state["weights"], activation=state["activation"]))


# ---- in 64 bits ----------------------------------------------------------------------------------------------------------
def _exact_rotary(state):
    """Every pair as one complex number, multiplied by one of the unit circle's."""
    turn = torch.polar(torch.full((), state["amplitude"], device="cuda", dtype=torch.float64),
                       state["positions"].double()[..., None] * state["frequencies"])
    turn = turn[:, None] if turn.dim() == 3 else turn
    rot = 2 * turn.shape[-1]

    def apply(x, by):
        z = x.detach().double()
        head = z[..., :rot]
        if not state["neighbours"]:  # halves -> neighbours
            head = head.unflatten(-1, (2, rot // 2)).transpose(-1, -2).reshape(head.shape)
        head = torch.view_as_real(torch.view_as_complex(head.reshape(*head.shape[:-1], -1, 2)) * by)
        head = (head if state["neighbours"] else head.transpose(-1, -2)).reshape(*z.shape[:-1], rot)
        return torch.cat((head, z[..., rot:]), -1)

    tensors = state["primals"] + (state["tangents"] if state["step"].startswith("jvp") else ())
    out = [apply(x, turn) for x in tensors]
    if state["step"].endswith("bwd"):
        out += [apply(x, turn.conj()) for x in state["cotangents"][:len(tensors)]]
    return tuple(out)


def _exact_gated(state):
    """Differentiated by torch from the value alone, in either direction."""
    F = torch.nn.functional
    act = {"silu": F.silu, "sigmoid": torch.sigmoid, "gelu": F.gelu, "gelu_tanh": lambda g: F.gelu(g, approximate="tanh")}[state["activation"]]
    step = state["step"]
    (x,), (tx,), (wg, wu) = state["primals"], state["tangents"], state["weights"]
    x, tx, wg, wu = (t.detach().double().requires_grad_(step.endswith("bwd")) for t in (x, tx, wg, wu))
    value = lambda v: act(F.linear(v, wg)) * F.linear(v, wu)  # noqa: E731
    out = torch.func.jvp(value, (x,), (tx,)) if step.startswith("jvp") else (value(x),)
    if not step.endswith("bwd"):
        return tuple(out)
    leaves = (x, tx, wg, wu) if step == "jvp_bwd" else (x, wg, wu)
    grads = torch.autograd.grad(out, leaves, [c.double() for c in state["cotangents"][:len(out)]])
    return (*(o.detach() for o in out), *grads)


def exact(case, seed):
    state = prepare(case, seed)
    return _exact_rotary(state) if case["op"] == "rotary" else _exact_gated(state)
