"""Refusals of the dense layer and of the q/k norm with rotation, and the leaf check of their differentiable forms: all on
the host, before anything is launched (fake CUDA tensors stand for real ones)."""
import pytest
import torch
from torch._subclasses import FakeTensorMode

from strata_b200 import _lib, ops, torch_ops

BF, HF = torch.bfloat16, torch.float16


@pytest.fixture
def cuda():
    """Makes fake CUDA tensors: shapes, strides, types and a device, no memory."""
    with FakeTensorMode(allow_non_fake_inputs=True):
        yield lambda *shape, dtype=BF: torch.empty(*shape, dtype=dtype, device="cuda:0")


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(4, 16, dtype=BF), torch.zeros(8, 16, dtype=BF)
    h = torch.zeros(4, 2, 64, dtype=BF)
    for call in (lambda: ops.linear_act(x, w), lambda: ops.linear_act_backward(torch.zeros(4, 8, dtype=BF), x, w),
                 lambda: ops.qk_norm_rope(h, h), lambda: ops.qk_norm_rope_backward(h, h, h, h)):
        with pytest.raises(_lib.StrataLibraryError):
            call()


@pytest.mark.parametrize("change,error", [
    (dict(x=((4, 16), torch.float32)), TypeError), (dict(w=((8, 16), HF)), TypeError),
    (dict(w=((8, 17), BF)), ValueError), (dict(w=((8,), BF)), ValueError), (dict(x=((16,), BF)), ValueError),
    (dict(b=((8,), BF)), TypeError), (dict(b=((7,), torch.float32)), ValueError),
    (dict(r=((4, 8), HF)), TypeError), (dict(r=((1, 8), BF)), ValueError), (dict(r=((2, 2, 8), BF)), ValueError),
    (dict(out=((4, 9), BF)), ValueError), (dict(out=((4, 8), HF)), TypeError), (dict(act="tanh"), ValueError),
    (dict(act=None), ValueError)])
def test_linear_act_refuses(cuda, change, error):
    a = dict(x=((4, 16), BF), w=((8, 16), BF), b=((8,), torch.float32), r=((4, 8), BF), out=None, act="gelu")
    a.update(change)
    t = {k: v if k == "act" or v is None else cuda(*v[0], dtype=v[1]) for k, v in a.items()}
    with pytest.raises(error):
        ops.linear_act(t["x"], t["w"], t["b"], t["act"], t["r"], out=t["out"])


def test_linear_act_refuses_rows_that_overlap_as_output(cuda):
    x, w = cuda(4, 16), cuda(8, 16)
    for out in (cuda(8).expand(4, 8), cuda(8, 4).t(), cuda(64).as_strided((4, 8), (4, 1))):
        with pytest.raises(ValueError):
            ops.linear_act(x, w, out=out)


@pytest.mark.parametrize("change,error", [
    (dict(z=None), ValueError), (dict(z=((4, 7), BF)), ValueError), (dict(z=((4, 8), HF)), TypeError),
    (dict(g=((4, 9), BF)), ValueError), (dict(g=((4, 8), HF)), TypeError), (dict(x=((5, 16), BF)), ValueError),
    (dict(x=((4, 15), BF)), ValueError), (dict(w=((8, 16, 1), BF)), ValueError), (dict(act="swish"), ValueError)])
def test_linear_act_backward_refuses(cuda, change, error):
    a = dict(g=((4, 8), BF), x=((4, 16), BF), w=((8, 16), BF), z=((4, 8), BF), act="gelu")
    a.update(change)
    t = {k: v if k == "act" or v is None else cuda(*v[0], dtype=v[1]) for k, v in a.items()}
    with pytest.raises(error):
        ops.linear_act_backward(t["g"], t["x"], t["w"], t["act"], t["z"])


@pytest.mark.parametrize("change,error", [
    (dict(q=((5, 4, 64), torch.float32)), TypeError), (dict(k=((5, 2, 64), HF)), TypeError),
    (dict(k=((4, 2, 64), BF)), ValueError), (dict(k=((5, 2, 56), BF)), ValueError), (dict(q=((5, 64), BF)), ValueError),
    (dict(q=((5, 4, 60), BF), k=((5, 2, 60), BF)), ValueError), (dict(q=((5, 4, 264), BF), k=((5, 2, 264), BF)), ValueError),
    (dict(q=((5, 0, 64), BF)), ValueError), (dict(qw=((64,), BF)), TypeError), (dict(kw=((4, 64), torch.float32)), ValueError),
    (dict(cs=((5, 32, 2), torch.float64)), TypeError), (dict(cs=((5, 64), HF)), ValueError),
    (dict(cs=((5, 36, 2), HF)), ValueError), (dict(cs=((5, 2, 2), HF)), ValueError),
    (dict(cs=((5, 20, 2), HF), interleaved=False), ValueError), (dict(cs=((0, 32, 2), HF)), ValueError),
    (dict(cs=((4, 32, 2), HF)), ValueError), (dict(tokens_per_tile=2, hw=2), ValueError),
    (dict(tokens_per_tile=0), ValueError), (dict(hw=0), ValueError), (dict(pos=((4,), torch.int64)), ValueError),
    (dict(pos=((5,), torch.float32)), TypeError), (dict(pos=((5,), torch.int64), hw=5), ValueError),
    (dict(pos=((5,), torch.int64), cs=None), ValueError)])
def test_qk_norm_rope_refuses(cuda, change, error):
    a = dict(q=((5, 4, 64), BF), k=((5, 2, 64), BF), qw=None, kw=None, cs=((5, 32, 2), HF), pos=None)
    more = {k: v for k, v in change.items() if k not in a}
    a.update({k: v for k, v in change.items() if k in a})
    t = {k: None if v is None else cuda(*v[0], dtype=v[1]) for k, v in a.items()}
    table = dict(rope_cs=t["cs"], positions=t["pos"], **more)
    with pytest.raises(error):
        ops.qk_norm_rope(t["q"], t["k"], t["qw"], t["kw"], **table)
    with pytest.raises(error):
        ops.qk_norm_rope_backward(t["q"], t["k"], t["q"], t["k"], t["qw"], t["kw"], **table)


def test_sizes_that_32_bits_do_not_count_are_refused(cuda):
    big = 2 ** 32 + 8
    with pytest.raises(ValueError, match="supported"):
        ops.linear_act(cuda(1, 16).expand(big, 16), cuda(8, 16))
    with pytest.raises(ValueError, match="supported"):
        ops.linear_act_backward(cuda(4, 8), cuda(4, big), cuda(8, big))
    with pytest.raises(ValueError, match="supported"):
        ops.qk_norm_rope(cuda(big, 1, 8), cuda(big, 1, 8))


def test_empty_batches_come_back_empty(cuda):
    y, z = ops.linear_act(cuda(2, 0, 16), cuda(8, 16), activation="silu", save_preact=True)
    assert y.shape == z.shape == (2, 0, 8)
    q, k = ops.qk_norm_rope(cuda(0, 4, 64), cuda(0, 1, 64))
    assert q.shape == (0, 4, 64) and k.shape == (0, 1, 64)


def test_leaves_of_a_living_eager_graph_are_refused_under_capture():
    a = torch.randn(3, requires_grad=True)
    edges = lambda y: y.grad_fn.next_functions
    alive = a * 2
    torch_ops.claim_leaves(edges(alive), 1, False)
    torch_ops.claim_leaves(edges(a * alive), 1, True)            # the same stream; an operand that is no leaf
    torch_ops.claim_leaves(edges(a + 1), 2, False)               # eager on another stream: torch orders the two
    with pytest.raises(RuntimeError, match="alive on another stream"):
        torch_ops.claim_leaves(edges(a + 1), 2, True)
    del alive
    torch_ops.claim_leaves(edges(a + 1), 2, True)                # nothing holds the old accumulation any more
