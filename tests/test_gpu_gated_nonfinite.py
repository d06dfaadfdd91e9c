"""GPU tests of gated_linear: NaN and infinite entries of x, in every row that has one and in no other.

An infinite entry makes every projection of its row infinite, or NaN (fp32, whose parts are infinity and infinity less infinity).  silu(g) u is then an
infinite number times one, or NaN (g s at minus infinity: infinity times zero, as is an infinite entry times a weight of zero); a'(g) tg u + a(g) tu
alike.  No entry can be finite."""
import pytest
import torch

from jvp_flash_attention_b200 import _lib
from tests.test_gpu_gated import _inputs, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("M", [1, 60, 128, 300])  # of few rows and of many, with a tangent 2 M
@pytest.mark.parametrize("step", ["fwd", "jvp"])
def test_nan_and_infinite_entries_stay_in_their_rows(dt, M, step):
    x, tx, wg, wu, _, _ = _inputs(M, 64, 200, dt, 41)
    want = _run(x, tx, wg, wu, None, None, "silu", step)
    bad = {M // 3: float("nan"), M - 1: float("inf"), M // 2: -float("inf")}
    for column, (row, value) in enumerate(bad.items()):
        x[row, 20 * column + 3] = value
    rows = torch.ones(M, dtype=torch.bool, device=x.device)
    rows[list(bad)] = False
    for name, y in _run(x, tx, wg, wu, None, None, "silu", step).items():
        assert torch.equal(y[rows], want[name][rows]), name
        for row, value in bad.items():
            assert (y[row].isnan().all() if value != value or dt == "fp32" else not y[row].isfinite().any()), (name, row)
    assert _lib.device_status() == 0
