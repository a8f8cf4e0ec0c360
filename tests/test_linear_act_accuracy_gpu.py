"""The dense layer's activations where their values are small: errors relative to the value itself, in every form of the
product (dot products, mma.sync, tiles, split sums, pairs of CTAs).

Tolerance beside the result's own rounding u |y| (u = finfo.eps / 2):
  gelu   Phi(-a) = 2^q(a) with a fitted q. The formula in 64 bits on 800001 points: bf16 off by 8.1e-5 of |y| for
         z > -4, 2.2e-4 for z > -6, 3.8e-3 for z > -8, 5.2 % for z > -9, 25 % for z > -10 and 4.5e-23 below; fp16 by
         6.2e-6 of |y| for z > -4 and 4e-10 below. Evaluated in fp32 (seven steps, |q| up to 17 at -4, 29 at -6 and 50 at
         -8, each 2^-24 |q| ln 2 at most, and exp2 to 2^-22): 6e-6 more at -4, 1e-5 at -6, 2e-5 at -8
  gelu_tanh, silu   z / (1 + 2^-w): four roundings or rounded constants in w, 2^-24 |w| ln 2 each, below 2^-22 |w| in
         all; exp2 to 2^-22, the reciprocal to 2^-23, four more roundings: below 2^-20 together. They stand still below
         -7.5 (at 4.017e-18; with its rounding to bf16, 2^-8 of it, 4.033e-18) and -40 (1.7e-16)
and what the type cannot hold: half of fp16's smallest step, 2^-25; in bf16, whose smallest normal number is fp32's,
what lies below 13 2^-126 (a value times a power of two that is flushed to zero)."""
import math

import pytest
import torch

from tests.test_linear_act_gpu import BF, HF

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from strata_b200 import ops
    return ops


def act64(z, act):
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":        # (torch.special.ndtr takes 1 + erf, whose 2^-53 is 5 % of Phi(-8))
        return z * torch.special.erfc(z * -(0.5 ** 0.5)) / 2
    return z / (1 + torch.exp(-2 * (2 / math.pi) ** 0.5 * (z + 0.044715 * z ** 3)))


def forms(ops, z, act):
    """act(z) by every form of the product: z [P] of a 16-bit type against a weight of ones on the diagonal."""
    one = torch.ones(1, 1, device="cuda", dtype=z.dtype)
    eye = lambda n, k: torch.eye(n, k, device="cuda", dtype=z.dtype)
    P = z.numel()
    assert P % 2000 == 0
    yield ops.linear_act(z[:, None], one, None, act)[:, 0]                                        # tiles
    yield torch.cat([ops.linear_act(part.view(4, -1), eye(P // 8, P // 8), None, act).flatten()
                     for part in z.view(2, -1)])                                                  # four rows
    yield torch.cat([ops.linear_act(part.view(20, -1), eye(P // 40, P // 40), None, act).flatten()
                     for part in z.view(2, -1)])                                                  # mma.sync
    wide = torch.cat([z.view(40, -1), torch.zeros(40, 8192 - P // 40, device="cuda", dtype=z.dtype)], 1)
    yield ops.linear_act(wide, eye(P // 40, 8192), None, act).flatten()                           # split sums
    big = z.view(-1, 100)
    big = big.repeat(40000 // len(big), 1)
    y = ops.linear_act(big, eye(600, 100), None, act)[:, :100]                                    # pairs of CTAs
    yield y[:P // 100].flatten()


def near(got, z, act, rel, rest=0.0):
    t, z = got.dtype, z.double()
    want = act64(z, act)
    u = torch.finfo(t).eps / 2
    least = 2.0 ** -25 if t == HF else 13 * 2.0 ** -126
    over = (got.double() - want).abs() - ((rel + u * (1 + rel)) * want.abs() + least + rest)
    i = int(over.argmax())
    assert float(over.max()) <= 0, f"{act}({float(z[i]):.5g}) = {float(got[i]):.5g}, not {float(want[i]):.5g}"


@pytest.mark.parametrize("t", [BF, HF])
def test_gelu_in_its_tail(ops, t):
    z = torch.cat([torch.linspace(-14, 0, 12001)[:-1], torch.linspace(0, 8, 2000), -torch.logspace(-5, 1.14, 2000)])
    z = z.to(t).cuda()
    steps = [(-4, 1e-4), (-6, 2.5e-4), (-8, 4e-3), (-9, 6e-2), (-10, 0.3)] if t == BF else [(-4, 1.3e-5)]
    rel = torch.zeros(z.shape, dtype=torch.float64, device="cuda")
    for above, r in reversed(steps):
        rel[z > above] = r
    rest = 5e-23 if t == BF else 5e-10
    for y in forms(ops, z, "gelu"):
        near(y, z, "gelu", rel, rest)


@pytest.mark.parametrize("act,far,least", [("gelu_tanh", -9, 4.05e-18), ("silu", -50, 1.72e-16)])
@pytest.mark.parametrize("t", [BF, HF])
def test_logistic_forms_in_their_tail(ops, act, far, least, t):
    z = torch.cat([torch.linspace(far, 0, 12001)[:-1], torch.linspace(0, 8, 2000), -torch.logspace(-5, 4, 2000)])
    z = z.to(t).cuda()
    d = z.double()
    w = (d if act == "silu" else 2 * (2 / math.pi) ** 0.5 * (d + 0.044715 * d ** 3)) / math.log(2)
    for y in forms(ops, z, act):
        near(y, z, act, 2.0 ** -20 + w.abs().clamp(max=100) * 2.0 ** -22, least)


@pytest.mark.parametrize("act,low", [("silu", -50.0), ("gelu", -6.0), ("gelu_tanh", -5.0)])
@pytest.mark.parametrize("M,N,K", [(3, 40, 64), (20, 40, 512), (64, 72, 4096), (200, 72, 64), (40000, 512, 64)])
def test_a_large_value_beside_a_small_one(ops, act, low, M, N, K):
    """Two columns share a reciprocal: the finite result of the one does not depend on the other's denominator. (silu
    keeps the value of -40 below that: 2e-16.)"""
    x, w = (torch.zeros(s, K, device="cuda", dtype=BF) for s in (M, N))
    for big in (1e25, 1e37):
        for first in (0, 1):
            b = torch.full((N,), low, device="cuda")
            b[first::2] = big
            want = act64(b.double(), act).to(BF)
            y = ops.linear_act(x, w, b, act)
            assert torch.equal(y[:, first::2], want[first::2].expand(M, -1))
            small = (y[:, 1 - first::2].double() - want[1 - first::2].double()).abs()
            assert bool((small <= 2 * torch.finfo(BF).eps * want[1 - first::2].double().abs() + 2e-16).all())
