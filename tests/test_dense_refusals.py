"""Calls of the dense layer and of the q/k norm that have no right answer: refused before anything is launched."""
import pytest
import torch
from torch._subclasses import FakeTensorMode

from strata_b200 import ops

BF = torch.bfloat16


@pytest.fixture
def cuda():
    """Makes fake CUDA tensors: shapes, strides, types and a device, no memory."""
    with FakeTensorMode(allow_non_fake_inputs=True):
        yield lambda *shape, dtype=BF: torch.empty(*shape, dtype=dtype, device="cuda:0")


@pytest.mark.parametrize("eps", [-1e-6, -0.5, float("nan"), float("inf")])
def test_eps_that_is_none(cuda, eps):
    q, k = cuda(0, 4, 64), cuda(0, 2, 64)
    with pytest.raises(ValueError, match="eps"):
        ops.qk_norm_rope(q, k, eps=eps)
    with pytest.raises(ValueError, match="eps"):
        ops.qk_norm_rope_backward(q, k, q, k, eps=eps)
