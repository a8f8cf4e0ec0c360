"""The gradients of qk_norm_rope where eps does not hold 1 / rms down: eps = 0, heads that leave slots of a warp empty,
values from one end of bf16 to the other."""
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


# (the squares of a head and their sum stay inside fp32)
@pytest.mark.parametrize("power", [-54, -44, 42, 54])
@pytest.mark.parametrize("hq,hk,hd,rot", [(3, 1, 64, 64), (12, 12, 64, None), (16, 4, 128, 64)])
def test_large_and_small_heads(ops, power, hq, hk, hd, rot):
    """dx has both of its terms, dw its sum, at any size of q and k."""
    M = 50
    d = data(M, hq, hk, hd, BF, rot=rot, rows=M, f32=True, seed=hq)
    d["q"], d["k"] = d["q"] * 2.0 ** power, d["k"] * 2.0 ** power
    for adjacent in (True, False):
        check(ops, d, adjacent, torch.arange(M, device="cuda"), eps=0.0)
    if power > 0:
        check(ops, d, True, torch.arange(M, device="cuda"))


def test_heads_of_zeros(ops):
    """r = eps^-1/2 and nothing else is left."""
    d = data(9, 4, 2, 64, BF)
    d["q"], d["k"] = d["q"].clone(), d["k"].clone()
    d["q"][3:5], d["k"][4] = 0, 0
    for eps in (1e-6, 1e-26, 1e-30):
        check(ops, d, True, eps=eps)
