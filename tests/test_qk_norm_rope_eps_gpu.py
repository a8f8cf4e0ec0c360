"""The gradients of qk_norm_rope where eps does not hold 1 / rms down: eps = 0, heads that leave slots of a warp empty."""
import pytest
import torch

from tests.test_qk_norm_rope_gpu import BF, HF, check, data

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from strata_b200 import ops
    return ops


# heads and tokens that fill no whole round of a warp, few-headed tokens, a token's heads over several blocks, head widths
# that leave lanes idle
@pytest.mark.parametrize("M,hq,hk,hd", [(5, 3, 1, 64), (7, 4, 2, 64), (33, 2, 1, 32), (301, 12, 3, 80), (9, 3, 40, 64),
                                        (1, 48, 1, 128), (44, 48, 12, 256), (1000, 1, 1, 16), (9001, 5, 3, 96)])
@pytest.mark.parametrize("table", [None, torch.float16, torch.float32])
@pytest.mark.parametrize("t", [BF, HF])
def test_eps_of_zero(ops, M, hq, hk, hd, table, t):
    rot = None if table is None else hd // 16 * 16
    d = data(M, hq, hk, hd, t, rot=rot, rows=M, f32=table == torch.float32, seed=M + hq)
    assert all(bool((d[x].float().abs().amax(-1) > 0).all()) for x in "qk")      # every head has a norm
    for adjacent in (True, False):
        at = None if rot is None else torch.arange(M, device="cuda").flip(0)
        check(ops, d, adjacent, at, eps=0.0, **({} if rot is None else dict(positions=at)))
