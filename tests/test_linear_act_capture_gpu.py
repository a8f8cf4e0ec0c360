"""A captured training step over leaves whose gradient accumulation something keeps, as data-parallel wrappers do."""
import pytest
import torch

from tests.test_linear_act_gpu import BF, data

pytestmark = pytest.mark.gpu


def test_capture_on_the_stream_of_the_warm_up():
    from strata_b200 import torch_ops  # noqa: F401  (registers the operators)
    d = data(256, 64, 48, BF)
    w, b = d["w"].clone().requires_grad_(), d["b"].clone().requires_grad_()
    forward = lambda: torch.ops.strata_b200.linear_act(d["x"], w, b, "gelu", None, True)[0]
    step = lambda: torch.autograd.grad(forward(), (w, b), d["dy"])
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        y = forward()
        kept = y.grad_fn.next_functions
        del y                                        # (the accumulations live on)
        want = step()
    torch.cuda.synchronize()
    assert any(hasattr(node, "variable") for node, _ in kept)
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="capture on their stream"):
        with torch.cuda.graph(g):
            forward()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        got = step()
    for seed in (1, 2):
        new = data(256, 64, 48, BF, seed=seed)
        for k in ("x", "dy"):
            d[k].copy_(new[k])
        g.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, v) for a, v in zip(got, want))
