"""Calls of the dense layer and of the q/k norm that have no right answer: refused before anything is launched."""
import itertools
import random

import pytest
import torch
from torch._subclasses import FakeTensorMode

from strata_b200 import _lib, ops

BF = torch.bfloat16


class Launched(Exception):
    pass


@pytest.fixture
def host(monkeypatch):
    """Lets host tensors through to where the library would be called."""
    monkeypatch.setattr(ops, "_require_16bit", lambda t, name: ops._DTYPES[t.dtype])

    def launch(*_):
        raise Launched
    monkeypatch.setattr(_lib, "load", launch)
    monkeypatch.setattr(_lib, "on_device", launch)


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


def test_memory_that_two_operands_share():
    """Against the sets of their bytes."""
    rng = random.Random(0)

    def operand():
        dims = [(rng.choice((0, 2, 4, 6, 16, 24, 30, 48, 120)), rng.randint(1, 4)) for _ in range(rng.randint(0, 2))]
        start, run = rng.randint(0, 200), 2 * rng.randint(1, 8)
        at = [start + sum(stride * i for (stride, _), i in zip(dims, index))
              for index in itertools.product(*(range(n) for _, n in dims))]
        return ops._span(start, run, *dims), {a + i for a in at for i in range(run)}

    found = set()
    for _ in range(20000):
        (a, bytes_a), (b, bytes_b) = operand(), operand()
        assert ops._meet(a, b) == ops._meet(b, a) == bool(bytes_a & bytes_b)
        found.add((bool(bytes_a & bytes_b), a[1] <= b[0] or b[1] <= a[0]))
    assert len(found) == 3
    rows = [(2 * 16 * 64, 10 ** 9), (2 * 64, 8)]            # packed heads, a great many tokens
    assert not ops._meet(ops._span(0, 128, *rows), ops._span(8 * 128, 128, *rows))
    assert ops._meet(ops._span(0, 128, *rows), ops._span(7 * 128 + 126, 128, *rows))


def test_out_that_shares_memory_with_an_operand(host):
    """Blocks of rows and columns that lie apart are taken, also those of one matrix."""
    wide = torch.zeros(40, 96, dtype=BF)
    x, w, r, y = (wide[:32, 24 * i:24 * i + 24] for i in range(4))
    w, other = w[:24], torch.zeros(32, 24, dtype=BF)
    run = lambda out, r=r, x=x, b=None: ops.linear_act(x, w, b, "gelu", r, out=out)
    flat = torch.zeros(2000, dtype=BF)
    for out, res in ((y, r), (r, r), (other, r), (other, other), (y, None), (wide[32:, :24], None),
                     (flat[100:868].view(32, 24), flat[868:1636].view(32, 24))):
        with pytest.raises(Launched):
            run(out, res, x if out.shape[0] == 32 else x[:8])
    for out in (x, wide[1:33, :24], wide[:32, 8:32], wide[:32, 40:64], wide.as_strided((32, 24), (24, 1), 23 * 96)):
        with pytest.raises(ValueError, match="not x or weight"):
            run(out, None)
    r2 = flat[100:868].view(32, 24)
    for out, res in ((wide[1:33, 48:72], r), (wide[:32, 50:74], r), (wide[:32, 49:73], r),
                     (flat.as_strided((32, 24), (25, 1), 100), r2), (flat[124:892].view(32, 24), r2)):
        with pytest.raises(ValueError, match="residual itself"):
            run(out, res)
    with pytest.raises(Launched):                      # one row: whatever its stride
        run(wide[:1, 48:72], wide[:1, 48:72], x[:1])
    b = torch.zeros(24)
    with pytest.raises(ValueError, match="bias"):
        run(b.view(BF).view(2, 24), None, x[:2], b)


def test_outputs_that_share_memory_with_q_or_k(host):
    """In place in this order, and into other heads and tokens of the same rows; nothing that is yet to be read."""
    M, h, hd = 12, 4, 16
    packed = torch.zeros(M, 5 * h * hd, dtype=BF)
    q, k, v, a, b = (packed[:, i * h * hd:(i + 1) * h * hd].view(M, h, hd) for i in range(5))
    other, more = torch.zeros(M, h, hd, dtype=BF), torch.zeros(M, h, hd, dtype=BF)
    woven = torch.zeros(M, h, 3, hd, dtype=BF)          # the heads of q, k and v in turn
    run = lambda out, q=q, k=k, **more: ops.qk_norm_rope(q, k, out=out, **more)
    for out in ((q, k), (a, b), (b, other), (q, b), (a, k), (other, more)):
        with pytest.raises(Launched):
            run(out)
    for out in ((woven[:, :, 0], woven[:, :, 1]), (woven[:, :, 2], woven[:, :, 1]), (other, more)):
        with pytest.raises(Launched):
            run(out, woven[:, :, 0], woven[:, :, 1])
    with pytest.raises(Launched):
        run((q[:, :1], k[:, 3:]), q[:, :1], k[:, 3:])
    step = packed[1:, :h * hd].view(M - 1, h, hd)
    square = torch.zeros(h, h, hd, dtype=BF)
    for out, x in (((k, q), (q, k)), ((k, a), (q, k)), ((a, q), (q, k)), ((a, a), (q, k)), ((q, q), (q, k)),
                   ((other, packed[:, 8:72].view(M, h, hd)), (q, k)), ((step, a[1:]), (q[:-1], k[:-1])),
                   ((a[1:], step), (q[:-1], k[:-1])), ((a, other), (q, a[:, :, :])), ((q, other), (q, q)),
                   ((square.transpose(0, 1), other[:h]), (square, k[:h])),
                   ((woven[:, :, 1], woven[:, :, 0]), (woven[:, :, 0], woven[:, :, 1]))):
        with pytest.raises(ValueError, match="themselves"):
            run(out, *x)
    w = torch.zeros(hd)
    with pytest.raises(ValueError, match="weights"):
        ops.qk_norm_rope(q[:1, :2], k[:1, :2], w, out=(w.view(BF).view(1, 2, hd), other[:1, :2]))


def test_a_table_that_asks_for_a_gradient(cuda):
    from strata_b200 import torch_ops  # noqa: F401  (registers the operators)
    op = torch.ops.strata_b200.qk_norm_rope
    q, k, cs = cuda(5, 4, 64), cuda(5, 2, 64), cuda(5, 32, 2, dtype=torch.float32)
    op(q.requires_grad_(), k, None, None, cs)
    cs.requires_grad_()
    for one in (q, q.detach()):
        with pytest.raises(NotImplementedError, match="rope_cs"):
            op(one, k, None, None, cs)
    with torch.no_grad():
        op(q, k, None, None, cs)
    op(q, k, None, None, cs.detach())


@pytest.mark.parametrize("N,K", [(0, 16), (8, 0), (0, 0)])
def test_widths_of_zero(cuda, N, K):
    for lead in ((4,), (0,), (2, 3)):
        x, w, dy = cuda(*lead, K), cuda(N, K), cuda(*lead, N)
        with pytest.raises(ValueError, match="at least one"):
            ops.linear_act(x, w)
        with pytest.raises(ValueError, match="at least one"):
            ops.linear_act_backward(dy, x, w)


def test_more_heads_than_are_counted(cuda):
    for hq, hk in ((65537, 1), (1, 65537)):
        with pytest.raises(ValueError, match="65536 heads"):
            ops.qk_norm_rope(cuda(0, hq, 8), cuda(0, hk, 8))
