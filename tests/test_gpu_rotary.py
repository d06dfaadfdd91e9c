"""GPU tests of rotary against its formula in float64.

Bound of an entry: half a step of its type, and for the arithmetic in 32 bits 2^-21 of its pair's length r: the fraction of a turn is
rounded to 32 bits (the angle is off by up to pi 2^-25 = 9.4e-8), sine and cosine are off by up to two units of their last place
(2^-23), the amplitude, the two products and the sum are rounded (4 times 2^-24, on values up to sqrt(2) r):
9.4e-8 + 1.7 * 1.2e-7 + ... < 4.77e-7 = 2^-21.  What is not turned is copied bit by bit."""
import pytest
import torch

import jvp_flash_attention_b200.rotary as rot
from jvp_flash_attention_b200.jvp_attention import JVPAttn
from oracle import jvp_attention_oracle as orc
from tests import _block_formulas as formulas

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _near(y, x, w, n, interleaved, amplitude=1.0, **kw):
    want = formulas.turn(x, w, interleaved=interleaved, amplitude=amplitude, **kw)
    step = torch.finfo(y.dtype).eps / 2
    smallest = torch.finfo(y.dtype).smallest_normal * step * 2  # half the spacing of the smallest numbers
    bound = step * want.abs() + (1 + step) * 2.0**-21 * abs(amplitude) * formulas.pair_norm(x, n, interleaved) + smallest
    off = (y.double() - want).abs()
    assert (off <= bound).all(), (off - bound).max().item()
    assert torch.equal(y[..., 2 * n:], x[..., 2 * n:])


def _make(shape, dtype, layout, g, std=1.0):
    B, H, L, D = shape
    if layout == "bhld":
        return (torch.randn(shape, generator=g, device=DEV) * std).to(dtype)
    if layout == "blhd":
        return (torch.randn(B, L, H, D, generator=g, device=DEV) * std).to(dtype).transpose(1, 2)
    if layout == "packed":
        return (torch.randn(B, L, H + 2, D, generator=g, device=DEV) * std).to(dtype).transpose(1, 2)[:, 1:H + 1]
    if layout == "odd":  # rows that begin anywhere
        return (torch.randn(B, H, L, D + 1, generator=g, device=DEV) * std).to(dtype)[..., 1:]
    return (torch.randn(B, H, D, L, generator=g, device=DEV) * std).to(dtype).transpose(2, 3)  # "columns": not contiguous in D


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,H,HK,L,D,rot_dim,layout", [
    (1, 1, 1, 1, 64, 64, "bhld"), (8, 16, 4, 1, 64, 64, "blhd"), (2, 3, 1, 7, 32, 32, "packed"), (2, 4, 2, 130, 128, 64, "blhd"),
    (1, 5, 5, 33, 96, 20, "bhld"), (3, 2, 1, 65, 40, 6, "odd"), (1, 2, 2, 9, 33, 32, "bhld"), (2, 2, 1, 17, 7, 2, "blhd"),
    (1, 3, 1, 31, 64, 0, "bhld"), (2, 2, 2, 12, 64, 64, "columns"), (4, 40, 8, 600, 64, 48, "blhd"),
])
def test_values(dt, interleaved, B, H, HK, L, D, rot_dim, layout):
    g = torch.Generator(device=DEV).manual_seed(B + L + D)
    q, k = _make((B, H, L, D), DT[dt], layout, g), _make((B, HK, L, D), DT[dt], layout, g)
    w = rot.rotary_frequencies(rot_dim, device=DEV)
    yq, yk = rot.rotary(q, k, w, interleaved=interleaved, offset=11)
    for y, x in ((yq, q), (yk, k)):
        assert y.shape == x.shape and y.dtype == x.dtype and y.stride(-1) == 1
        _near(y, x, w, rot_dim // 2, interleaved, offset=11)
    if layout == "blhd" and L > 1:
        assert yq.transpose(1, 2).is_contiguous()


@pytest.mark.parametrize("kind", ["far32", "far64", "negative", "rows", "one_row", "strided"])
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_positions(kind, dt):
    B, H, L, D = 3, 2, 21, 64
    g = torch.Generator(device=DEV).manual_seed(3)
    q = _make((B, H, L, D), DT[dt], "blhd", g)
    w = rot.rotary_frequencies(64, device=DEV)
    r = torch.randint(0, 1 << 20, (B, L), generator=g, device=DEV)
    pos = {"far32": (2**31 - 1 - r).to(torch.int32), "far64": (1 << 33) + r, "negative": -r, "rows": r, "one_row": r[:1],
           "strided": torch.stack((r, -r), -1)[..., 0]}[kind]
    y = rot.rotary(q, None, w, pos, amplitude=0.75)
    want = formulas.turn(q, w, pos, amplitude=0.75)
    # 64 bits: the product of position and frequency is off by 2^-52 of itself (two roundings here, one in the formula's)
    far = pos.abs().max().item() * 2.0**-51
    step = torch.finfo(y.dtype).eps / 2
    bound = step * want.abs() + (2.0**-21 + far) * formulas.pair_norm(q, 32, False)
    assert ((y.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dt,interleaved,layout", [("bf16", False, "blhd"), ("fp16", True, "packed"), ("fp32", True, "bhld"), ("fp32", False, "odd")])
def test_tangents_and_gradients(dt, interleaved, layout):
    B, H, HK, L, D, n = 2, 6, 2, 77, 64, 16
    g = torch.Generator(device=DEV).manual_seed(5)
    shapes = ((B, H, L, D), (B, HK, L, D))
    q, k, tq, tk = leaves = [_make(s, DT[dt], layout, g, std).detach().requires_grad_() for std in (1.0, 0.1) for s in shapes]
    cots = [_make(s, DT[dt], "bhld", g) for s in shapes * 2]
    w = rot.rotary_frequencies(2 * n, device=DEV)
    (yq, yk), (zq, zk) = torch.func.jvp(lambda a, b: rot.rotary(a, b, w, offset=5, interleaved=interleaved), (q, k), (tq, tk))
    grads = torch.autograd.grad((yq, yk, zq, zk), leaves, cots)
    for y, x in zip((yq, yk, zq, zk), leaves):
        _near(y.detach(), x.detach(), w, n, interleaved, offset=5)
    for d, c in zip(grads, cots):
        _near(d, c, w, n, interleaved, offset=5, transposed=True)
    # a cotangent that is broadcast (of a sum): rows of stride 0
    (d,) = torch.autograd.grad(rot.rotary(q, None, w, interleaved=interleaved).sum(), q)
    _near(d, torch.ones_like(q), w, n, interleaved, transposed=True)


def test_nan_and_infinite_entries_stay_in_their_pair():
    q = torch.randn(1, 2, 40, 64, device=DEV)
    q[0, 1, 3, 5], q[0, 0, 9, 40] = float("nan"), float("inf")
    w = rot.rotary_frequencies(64, device=DEV)
    y = rot.rotary(q, None, w)
    bad = ~y.isfinite()
    want = torch.zeros_like(bad)
    want[0, 1, 3, 5] = want[0, 1, 3, 37] = want[0, 0, 9, 40] = want[0, 0, 9, 8] = True
    assert torch.equal(bad, want)


@pytest.mark.parametrize("shape", [(0, 2, 4, 64), (2, 2, 0, 64), (2, 0, 4, 64)])
def test_empty(shape):
    q = torch.randn(shape, device=DEV, requires_grad=True)
    w = rot.rotary_frequencies(64, device=DEV)
    k = torch.randn(shape[0], 3, *shape[2:], device=DEV)
    yq, yk = rot.rotary(q, k, w)
    assert yq.shape == q.shape and yk.shape == k.shape
    (d,) = torch.autograd.grad(yq.sum(), q)
    assert d.shape == q.shape
    if k.numel():
        _near(yk, k, w, 32, False)


def test_another_stream_and_a_captured_graph():
    q, k = torch.randn(2, 4, 50, 64, device=DEV, dtype=torch.bfloat16), torch.randn(2, 1, 50, 64, device=DEV, dtype=torch.bfloat16)
    pos = torch.arange(50, device=DEV)
    w = rot.rotary_frequencies(64, device=DEV)
    want = rot.rotary(q, k, w, pos)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = rot.rotary(q, k, w, pos)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rot.rotary(q, k, w, pos)
    pos += 1000  # positions are read when the graph runs
    graph.replay()
    torch.cuda.synchronize()
    want = rot.rotary(q, k, w, pos)
    assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_positions_changed_before_the_backward_are_noticed():
    q = torch.randn(1, 1, 4, 64, device=DEV, requires_grad=True)
    pos = torch.arange(4, device=DEV)
    y = rot.rotary(q, None, rot.rotary_frequencies(64, device=DEV), pos)
    pos += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_attention_on_turned_queries_and_keys():
    """Rotary in front of the fused attention under one torch.func.jvp, against float64."""
    B, H, L, D = 2, 4, 130, 64
    g = torch.Generator(device=DEV).manual_seed(8)
    q, k, v, w1, w2 = (_make((B, H, L, D), torch.float32, "blhd", g) for _ in range(5))
    tq, tk, tv = (_make((B, H, L, D), torch.float32, "blhd", g, 0.1) for _ in range(3))
    w = rot.rotary_frequencies(D, device=DEV)
    a = [x.detach().requires_grad_() for x in (q, k, v)]

    def block(q, k, v):
        q, k = rot.rotary(q, k, w)
        return JVPAttn.fwd_dual(q, k, v, causal=True)

    o, to = torch.func.jvp(block, tuple(a), (tq, tk, tv))
    grads = torch.autograd.grad((o, to), a, (w1, w2))
    turned = [formulas.turn(x, w) for x in (q, k, tq, tk)]
    ro, rto, dq, dk, dv = orc.grads_through_both(*(x.cpu() for x in (turned[0], turned[1], v.double(), turned[2], turned[3], tv.double(),
                                                                     w1.double(), w2.double())), causal=True)
    want = (ro, rto, formulas.turn(dq.to(DEV), w, transposed=True), formulas.turn(dk.to(DEV), w, transposed=True), dv)
    for got, r in zip((o, to, *grads), want):
        r = r.to(DEV)
        # attention's own bound (1e-5 of the largest entry), twice: the turns before and behind it are off by 2^-21 of a pair
        assert (got.double() - r).abs().max() <= 2e-5 * r.abs().max()
