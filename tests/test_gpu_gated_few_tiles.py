"""GPU tests of gated_linear for few rows, at numbers of tiles (64 features, or 128 columns of dx) where one to three rounds of two or three CTAs an SM
take them: 172, 313, 448 and 625, and dx's 320."""
import pytest

from tests.test_gpu_gated import _case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("K,F", [(136, 11008), (136, 20000), (136, 28672), (136, 40000), (40960, 72)])
@pytest.mark.parametrize("M,step", [(1, "fwd_bwd"), (100, "fwd_bwd"), (60, "jvp_bwd")])
def test_numbers_of_tiles(dt, K, F, M, step):
    _case(M, K, F, dt, "silu", step)
