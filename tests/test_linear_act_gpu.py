"""The dense layer with its epilogue and gradients against the formulas in 64 bits, element by element.

Tolerances (u: half a step of the type, finfo.eps / 2; e = 2^-23 bounds a step of an fp32 sum, two roundings):
  z   |x| |w|^T (K + 2) e + |b| e
  y   that times the activation's largest slope (1.13), + the activation's own error, + u |y|; the activation's error is
      2^-20 |z| (exp2, reciprocal and products, a few steps each), for gelu_tanh 2^-12 |z| (the hardware's tanh: 2^-11 of
      (1 + tanh) / 2 <= 1), for gelu besides its fit's: 1.1e-4 (bf16), 4.6e-6 (fp16) of max(|y|, 0.01), the maximum over
      [-12, 12] of the polynomial's formula evaluated in 64 bits, and 1e-8 below -6, where it stands still
  dz  slope error 1e-6 + its own rounding u |dz|
  dx, dW  sums of |dz error| |w| and |dz| |w| (N + 2) e, + u |result|;  db: without the rounding of dz
and a smallest step of the type (fp16: 2^-25, bf16: nothing that shows) where results are subnormal."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
E = 2.0 ** -23
BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ops():
    from strata_b200 import ops
    return ops


def act64(z, act):
    c = (2 / math.pi) ** 0.5
    return {"none": lambda: z, "relu": lambda: z.clamp(min=0), "silu": lambda: z * torch.sigmoid(z),
            "gelu": lambda: z * torch.special.ndtr(z),
            "gelu_tanh": lambda: 0.5 * z * (1 + torch.tanh(c * (z + 0.044715 * z ** 3)))}[act]()


def slope64(z, act):
    z = z.clamp(-40, 40)
    c = (2 / math.pi) ** 0.5
    if act == "none":
        return torch.ones_like(z)
    if act == "relu":
        return (z > 0).double()
    if act == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    if act == "gelu":
        return torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    t = torch.tanh(c * (z + 0.044715 * z ** 3))
    return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)


def act_error(z, y, act, t):
    if act in ("none", "relu"):
        return 0.0
    rounding = z.abs() * 2.0 ** (-12 if act == "gelu_tanh" else -20)
    return rounding + (y.abs().clamp(min=0.01) * (1.1e-4 if t == BF else 4.6e-6) + 1e-8 if act == "gelu" else 0.0)


def near(got, want, slack, t):
    u = torch.finfo(t).eps / 2
    tiny = 2.0 ** -25 if t == HF else 0.0
    assert got.shape == want.shape and got.dtype == t
    over = (got.double() - want).abs() - (slack + u * (want.abs() + slack) + tiny)
    assert float(over.max()) <= 0, f"{float(over.max()):.3e} beyond the tolerance at {int(over.argmax())}"


def data(M, N, K, t, seed=0, bias=True, residual=True):
    g = torch.Generator("cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")
    return dict(x=n(M, K).to(t), w=(n(N, K) * K ** -0.5).to(t), b=n(N) if bias else None,
                r=n(M, N).to(t) if residual else None, dy=n(M, N).to(t))


def check_forward(y, z, d, act):
    t = d["x"].dtype
    x, w = d["x"].double(), d["w"].double()
    z64 = x @ w.T
    ez = x.abs() @ w.abs().T * ((x.shape[-1] + 2) * E)
    if d["b"] is not None:
        z64 = z64 + d["b"].double()
        ez = ez + (z64.abs() + d["b"].double().abs()) * E
    if z is not None:
        near(z, z64, ez, t)
    y64 = act64(z64, act)
    ey = 1.13 * ez + act_error(z64, y64, act, t)
    if d["r"] is not None:
        y64 = y64 + d["r"].double()
        ey = ey + y64.abs() * E
    near(y, y64, ey, t)


def check_backward(got, d, z, act):
    t = d["x"].dtype
    x, w, dy = d["x"].double(), d["w"].double(), d["dy"].double()
    u = torch.finfo(t).eps / 2
    dz = dy * slope64(z.double(), act) if act != "none" else dy
    e_slope = 1e-6 * dy.abs() if act not in ("none", "relu") else 0 * dy
    e_dz = e_slope + (u * dz.abs() + (2.0 ** -25 if t == HF else 0.0) if act != "none" else 0.0)
    dx, dw, db = got
    M, N = dy.shape
    if dx is not None:
        near(dx, dz @ w, e_dz @ w.abs() + dz.abs() @ w.abs() * ((N + 2) * E), t)
    if dw is not None:
        near(dw, dz.T @ x, e_dz.T @ x.abs() + dz.abs().T @ x.abs() * ((M + 2) * E), t)
    if db is not None:
        assert db.dtype == torch.float32
        assert bool(((db.double() - dz.sum(0)).abs() <= e_slope.sum(0) + dz.abs().sum(0) * ((M + 2) * E)).all())


# one row and the few-row form's edges; a 128-row tile's edges; widths that are no multiple of 8; one column, one
# contraction value; several turns of the chip; split sums (few tiles, long contraction) with and without a ragged end
SIZES = [(1, 64, 64), (1, 4096, 1024), (2, 130, 77), (5, 33, 520), (8, 650, 207), (9, 64, 64), (24, 1024, 4096),
         (127, 72, 8), (128, 256, 64), (129, 257, 65), (300, 1, 40), (77, 40, 1), (2500, 650, 207), (1100, 1536, 384),
         (20011, 384, 640), (333, 520, 4104), (40000, 264, 72)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("t", [BF, HF])
def test_forward(ops, M, N, K, t):
    for i, act in enumerate(ops.ACTIVATIONS):
        d = data(M, N, K, t, seed=M + i, bias=i != 1, residual=i % 2 == 0)
        y, z = ops.linear_act(d["x"], d["w"], d["b"], act, d["r"], save_preact=True)
        check_forward(y, z, d, act)
        y2 = ops.linear_act(d["x"], d["w"], d["b"], act, d["r"])
        assert torch.equal(y, y2)               # the same sums in the same order, with and without z


@pytest.mark.parametrize("M,N,K", SIZES + [(70001, 128, 128), (3000, 2048, 264), (64, 4096, 512)])
@pytest.mark.parametrize("t", [BF, HF])
def test_backward(ops, M, N, K, t):
    from strata_b200 import _lib
    for i, act in enumerate(ops.ACTIVATIONS):
        d = data(M, N, K, t, seed=M + i)
        z = ops.linear_act(d["x"], d["w"], d["b"], "none")
        got = ops.linear_act_backward(d["dy"], d["x"], d["w"], act, z)
        check_backward(got, d, z, act)
        again = ops.linear_act_backward(d["dy"], d["x"], d["w"], act, z)
        assert all(torch.equal(a, b) for a, b in zip(got, again))       # no order of additions is left to chance
        for need in ((1, 0, 0), (0, 1, 0), (0, 0, 1)):
            one = ops.linear_act_backward(d["dy"], d["x"], d["w"], act, z, need_x=bool(need[0]),
                                          need_weight=bool(need[1]), need_bias=bool(need[2]))
            assert all((a is None) if not n else torch.equal(a, b) for a, b, n in zip(one, got, need))
    assert _lib.device_status() == 0


# db where one block of rows has it whole, in the blocks of a product, and where the product has too few of them
@pytest.mark.parametrize("M,N,K", [(2, 472, 16), (64, 4000, 8), (600, 472, 16), (3000, 4001, 8), (3000, 40, 8)])
def test_bias_gradient_with_few_blocks(ops, M, N, K):
    d = data(M, N, K, BF, seed=M)
    for act in ("none", "silu"):
        z = ops.linear_act(d["x"], d["w"], d["b"], "none")
        got = ops.linear_act_backward(d["dy"], d["x"], d["w"], act, z)
        check_backward(got, d, z, act)
        for nx, nw in ((False, False), (True, False), (False, True)):
            part = ops.linear_act_backward(d["dy"], d["x"], d["w"], act, z, need_x=nx, need_weight=nw)
            assert torch.equal(part[2], got[2])


def test_out_may_not_be_an_operand(ops):
    d = data(64, 64, 64, BF)
    for out in (d["x"], d["w"]):
        with pytest.raises(ValueError, match="not x or weight"):
            ops.linear_act(d["x"], d["w"], d["b"], "gelu", out=out)


def test_gradients_are_the_forward_pass_differences():
    """The 64-bit gradients that the kernels are held to, against central differences of the 64-bit forward formula."""
    g = torch.Generator("cuda").manual_seed(0)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda", dtype=torch.float64)
    x, w, b, dy = n(7, 5), n(3, 5), n(3), n(7, 3)
    for act in ("gelu", "gelu_tanh", "silu", "relu"):
        f = lambda x, w, b: (act64(x @ w.T + b, act) * dy).sum()
        dz = dy * slope64(x @ w.T + b, act)
        for grad, at in ((dz @ w, 0), (dz.T @ x, 1), (dz.sum(0), 2)):
            args, v = [x, w, b], n(*(x, w, b)[at].shape)
            h = 1e-6
            args[at] = (x, w, b)[at] + h * v
            up = f(*args)
            args[at] = (x, w, b)[at] - h * v
            # (error of a central difference: h^2 |f'''| / 6 + rounding 2^-52 |f| / h, below 1e-8 here)
            assert abs(float((up - f(*args)) / (2 * h) - (grad * v).sum())) < 1e-7


@pytest.mark.parametrize("t", [BF, HF])
def test_activations_over_their_whole_range(ops, t):
    """z swept through everything the type holds, on every path of the epilogue (one row form, tiles, split sums)."""
    z = torch.cat([torch.linspace(-12, 12, 40961), torch.linspace(-300, 300, 4001), torch.logspace(-6, 4.7, 2000),
                   -torch.logspace(-6, 4.7, 2000)]).cuda().to(t)[:, None]
    one = torch.ones(1, 1, device="cuda", dtype=t)
    for act in ops.ACTIVATIONS:
        d = dict(x=z, w=one, b=None, r=None)
        check_forward(ops.linear_act(z, one, None, act), None, d, act)
        few = z[-2000:, 0].view(-1, 8).T.contiguous()                   # 8 rows of 250 diagonal columns
        w = torch.eye(250, device="cuda", dtype=t)
        check_forward(ops.linear_act(few, w, None, act), None, dict(x=few, w=w, b=None, r=None), act)
        wide = torch.cat([z[:40000].view(40, 1000), torch.zeros(40, 7192, device="cuda", dtype=t)], 1)
        w = torch.eye(1000, 8192, device="cuda", dtype=t)
        check_forward(ops.linear_act(wide, w, None, act), None, dict(x=wide, w=w, b=None, r=None), act)
        big = z[:40000].view(400, 100).repeat(8, 1)                     # pairs of CTAs
        w = torch.eye(600, 100, device="cuda", dtype=t)
        check_forward(ops.linear_act(big, w, None, act), None, dict(x=big, w=w, b=None, r=None), act)


@pytest.mark.parametrize("t", [BF, HF])
def test_strides_and_alignments(ops, t):
    """Column slices, rows off the 16-byte grid, transposed and expanded operands, a contiguous copy's results."""
    M, N, K = 190, 72, 96
    d = data(M, N, K, t)
    for make in (lambda a: torch.cat([a, a], 1)[:, :a.shape[1]],                        # wider rows
                 lambda a: torch.cat([a[:, :3], a, a[:, :2]], 1)[:, 3:3 + a.shape[1]],  # 6 bytes off, odd row stride
                 lambda a: torch.cat([a[:, :8], a], 1)[:, 8:],                          # 16-byte steps
                 lambda a: a.t().contiguous().t(),                                      # unit stride the other way
                 lambda a: torch.stack([a, a], 2)[:, :, 1]):                            # every other element
        v = {k: make(a) if k != "b" else torch.cat([a[:1], a])[1:] for k, a in d.items()}
        assert torch.equal(v["x"], d["x"])
        for m in (M, 3):
            y, z = ops.linear_act(v["x"][:m], v["w"], v["b"], "silu", v["r"][:m], save_preact=True)
            check_forward(y, z, {**d, "x": d["x"][:m], "r": d["r"][:m]}, "silu")
        z = make(ops.linear_act(d["x"], d["w"], d["b"]))
        check_backward(ops.linear_act_backward(v["dy"], v["x"], v["w"], "silu", z), d, z, "silu")
        check_backward(ops.linear_act_backward(v["dy"], v["x"], v["w"]), d, None, "none")
    one = d["dy"][:1, :1].expand(M, N)                       # what sum().backward() hands over
    check_backward(ops.linear_act_backward(one, d["x"], d["w"]), {**d, "dy": one}, None, "none")
    same = d["x"][:1].expand(M, K)
    check_forward(ops.linear_act(same, d["w"], d["b"]), None, {**d, "x": same, "r": None}, "none")
    y3 = ops.linear_act(d["x"].view(2, 95, K), d["w"], d["b"], "relu", d["r"].view(2, 95, N))
    assert y3.shape == (2, 95, N) and torch.equal(y3.view(M, N), ops.linear_act(d["x"], d["w"], d["b"], "relu", d["r"]))


@pytest.mark.parametrize("K,N", [(77, 65), (80, 97), (74, 90)])
def test_what_lies_behind_the_last_column_does_not_count(ops, K, N):
    """Views whose rows go on with NaN."""
    nan = lambda a: torch.cat([a, torch.full((len(a), 104 - a.shape[1]), float("nan"), device="cuda", dtype=a.dtype)],
                              1)[:, :a.shape[1]]
    d = data(300, N, K, BF)
    v = {k: a if k == "b" else nan(a) for k, a in d.items()}
    y, z = ops.linear_act(v["x"], v["w"], v["b"], "gelu", v["r"], save_preact=True)
    check_forward(y, z, d, "gelu")
    check_backward(ops.linear_act_backward(v["dy"], v["x"], v["w"], "gelu", nan(z)), d, z, "gelu")
    check_backward(ops.linear_act_backward(v["dy"], v["x"], v["w"]), d, None, "none")


@pytest.mark.parametrize("M", [4, 64, 1500])
@pytest.mark.parametrize("N", [96, 97])
def test_out_may_be_the_residual_and_leaves_the_rest_alone(ops, M, N):
    d = data(M, N, 80, BF)
    want = ops.linear_act(d["x"], d["w"], d["b"], "gelu", d["r"])
    wide = torch.full((M + 2, N + 15), 7.0, device="cuda", dtype=BF)
    out = wide[1:M + 1, 8:8 + N]
    out.copy_(d["r"])
    got = ops.linear_act(d["x"], d["w"], d["b"], "gelu", out, out=out)
    assert got.data_ptr() == out.data_ptr() and torch.equal(out, want)
    wide[1:M + 1, 8:8 + N] = 7.0
    assert bool((wide == 7.0).all())


# every tile, one and several turns, with and without other operands that have to be copied, split sums
@pytest.mark.parametrize("M,N,K", [(40, 17, 64), (300, 65, 64), (24000, 105, 40), (2500, 650, 207),
                                   (40000, 97, 128), (9000, 1001, 64), (9000, 1002, 77), (64, 130, 4096)])
@pytest.mark.parametrize("t", [BF, HF])
def test_residual_rows_off_the_grid(ops, M, N, K, t):
    """Contiguous, one element off, and in place between NaN; out leaves what lies around it alone. (Every result against
    64 bits: kernels for different rows may contract the activation's products differently.)"""
    d = data(M, N, K, t)
    check_forward(ops.linear_act(d["x"], d["w"], d["b"], "silu", d["r"]), None, d, "silu")
    for lead in (1, 2, 8):
        wide = torch.full((M + 2, N + lead + 5), float("nan"), device="cuda", dtype=t)
        r = wide[1:M + 1, lead:lead + N]
        r.copy_(d["r"])
        check_forward(ops.linear_act(d["x"], d["w"], d["b"], "silu", r), None, d, "silu")
        assert ops.linear_act(d["x"], d["w"], d["b"], "silu", r, out=r) is r
        check_forward(r, None, d, "silu")
        assert int(wide.isnan().sum()) == wide.numel() - M * N


def test_no_rows(ops):
    d = data(0, 24, 16, HF)
    assert ops.linear_act(d["x"], d["w"], d["b"], "gelu", d["r"]).shape == (0, 24)
    dx, dw, db = ops.linear_act_backward(d["dy"], d["x"], d["w"])
    assert dx.shape == (0, 16) and not dw.any() and not db.any() and dw.shape == (24, 16) and db.shape == (24,)


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu", "relu"])
def test_infinite_and_nan_preactivations(ops, act):
    """A z that has left fp16 has the slope of a far z; NaN stays NaN, in its row and column only."""
    d = data(40, 16, 24, HF)
    z = torch.randn(40, 16, device="cuda").to(HF)
    z[3, 4], z[5, 6] = float("inf"), float("-inf")
    got = ops.linear_act_backward(d["dy"], d["x"], d["w"], act, z)
    check_backward(got, d, z, act)
    z[7, 8] = float("nan")
    dx, dw, db = ops.linear_act_backward(d["dy"], d["x"], d["w"], act, z)
    assert dx[7].isnan().all() and dw[8].isnan().all() and db[8].isnan()
    assert int(dx.isnan().sum()) == 24 and int(dw.isnan().sum()) == 24 and int(db.isnan().sum()) == 1
    x = d["x"].clone()
    x[2, 1] = float("nan")
    y = ops.linear_act(x, d["w"], d["b"], act)
    assert y[2].isnan().all() and int(y.isnan().sum()) == 16


@pytest.mark.parametrize("act", ["none", "gelu", "gelu_tanh", "silu", "relu"])
@pytest.mark.parametrize("M,N,K", [(3, 40, 64), (20, 40, 512), (64, 72, 4096), (200, 72, 64), (2048, 1024, 64)])
def test_nan_stays_in_its_column(ops, act, M, N, K):
    """A NaN or an infinity in one output's weights or bias reaches no other output, in any form of the product."""
    d = data(M, N, K, BF)
    want = ops.linear_act(d["x"], d["w"], d["b"], act, d["r"])
    w, b = d["w"].clone(), d["b"].clone()
    w[5], b[10], b[17], b[22] = float("nan"), float("nan"), float("inf"), float("-inf")
    y, z = ops.linear_act(d["x"], w, b, act, d["r"], save_preact=True)
    clean = torch.ones(N, dtype=torch.bool, device="cuda")
    clean[[5, 10, 17, 22]] = False
    # (two neighbours share a reciprocal, so a neighbour may move within the formula's rounding, 2^-20 |z|, and then by a step)
    step = torch.finfo(BF).eps * want[:, clean].float().abs() + 2.0 ** -19 * z[:, clean].float().abs()
    assert bool(((y[:, clean].float() - want[:, clean].float()).abs() <= step).all())
    assert y[:, [5, 10]].isnan().all() and (y[:, 17] == float("inf")).all() and not z[:, clean].isnan().any()


def test_offsets_beyond_32_bits(ops):
    """4.3e9 outputs and inputs: the rows behind 2^32 elements are their own."""
    M, N = 1_048_800, 4104
    d = data(M, 8, N, BF, residual=False)
    at = torch.tensor([0, 1, M // 2, M - 130, M - 1], device="cuda")
    check_forward(ops.linear_act(d["x"], d["w"], d["b"], "relu")[at], None, {**d, "x": d["x"][at]}, "relu")
    w = torch.randn(N, 8, device="cuda").to(BF)
    x = torch.randn(M, 8, device="cuda").to(BF)
    y = d["x"]                                           # 8.6 GB, written over
    ops.linear_act(x, w, None, out=y)
    check_forward(y[at], None, dict(x=x[at], w=w, b=None, r=None), "none")
    dx = ops.linear_act_backward(y, x, w, need_weight=False, need_bias=False)[0]
    check_backward((dx[at], None, None), dict(x=x[at], w=w, dy=y[at]), None, "none")


def test_captured_and_replayed(ops):
    """Two graphs that share a memory pool, replayed in turn on new inputs, on a stream of their own."""
    from strata_b200 import _lib
    d, e = data(500, 136, 1032, BF, seed=1), data(500, 136, 1032, BF, seed=2)
    s = {k: v.clone() for k, v in d.items()}

    def step():
        y, z = ops.linear_act(s["x"], s["w"], s["b"], "gelu", s["r"], save_preact=True)
        return y, z, *ops.linear_act_backward(s["dy"], s["x"], s["w"], "gelu", z)

    step()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0].pool() if graphs else None):
            outs.append(step())
        graphs.append(g)
    for v in (d, e, d):
        for k in s:
            s[k].copy_(v[k])
        want = step()
        for g, out in zip(graphs, outs):
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))
    assert _lib.device_status() == 0


def test_two_streams_at_once(ops):
    d = [data(700, 264, 2056, HF, seed=i) for i in range(2)]
    run = lambda v: ops.linear_act_backward(v["dy"], v["x"], v["w"])
    want = [run(v) for v in d]
    streams = [torch.cuda.Stream() for _ in d]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, v in enumerate(d):
            with torch.cuda.stream(streams[i]):
                got[i].append(run(v))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for i in range(2) for one in got[i] for a, b in zip(one, want[i]))


# ------------------------------------------------------------------ the differentiable form
def test_autograd_is_the_backward_call(ops):
    from strata_b200 import torch_ops  # noqa: F401  (registers the operators)
    op = torch.ops.strata_b200.linear_act
    d = data(60, 24, 40, BF)
    for act in ops.ACTIVATIONS:
        for keep in (False, True):
            x, w, b, r = (d[k].clone().requires_grad_() for k in "xwbr")
            y, z = op(x, w, b, act, r, keep)
            assert torch.equal(y, ops.linear_act(d["x"], d["w"], d["b"], act, d["r"])) and not z.requires_grad
            y.backward(d["dy"])
            z = ops.linear_act(d["x"], d["w"], d["b"])
            want = ops.linear_act_backward(d["dy"], d["x"], d["w"], act, z)
            assert all(torch.equal(a.grad, v) for a, v in zip((x, w, b), want)) and torch.equal(r.grad, d["dy"])
    # only what asks for a gradient gets one
    w = d["w"].clone().requires_grad_()
    op(d["x"], w, d["b"], "silu")[0].sum().backward()
    assert w.grad is not None


@pytest.mark.parametrize("N", [24, 27])
def test_operator_registration(ops, N):
    """Schema, shape-only implementation (strides of odd widths included) and gradients as torch checks them."""
    from strata_b200 import torch_ops  # noqa: F401
    d = data(40, N, 32, BF)
    x, w, b, r = (d[k].clone().requires_grad_() for k in "xwbr")
    torch.library.opcheck(torch.ops.strata_b200.linear_act, (x, w, b, "silu", r, True),
                          test_utils=("test_schema", "test_faketensor", "test_autograd_registration"))
    f = torch.compile(lambda x, w, b, r: torch.ops.strata_b200.linear_act(x, w, b, "silu", r, True)[0] * 2, fullgraph=True)
    y = f(x, w, b, r)
    assert torch.equal(y, 2 * ops.linear_act(d["x"], d["w"], d["b"], "silu", d["r"]))
    y.backward(d["dy"])
    want = ops.linear_act_backward(2 * d["dy"], d["x"], d["w"], "silu", ops.linear_act(d["x"], d["w"], d["b"]))
    assert all(torch.equal(t.grad, v) for t, v in zip((x, w, b, r), (*want, 2 * d["dy"])))


def test_captured_training_step(ops):
    """Forward and backward in one graph: refused while an eager graph of the same leaves lives, right once it is gone."""
    from strata_b200 import torch_ops  # noqa: F401
    op = torch.ops.strata_b200.linear_act
    d = data(256, 64, 48, BF)
    w, b = d["w"].clone().requires_grad_(), d["b"].clone().requires_grad_()

    def step():
        y = op(d["x"], w, b, "gelu", None, True)[0]
        return torch.autograd.grad(y, (w, b), d["dy"])

    want = step()
    alive = op(d["x"], w, b, "gelu", None, True)[0]
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="alive on another stream"):
        with torch.cuda.graph(g):
            op(d["x"], w, b, "gelu", None, True)
    del alive
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, v) for a, v in zip(got, want))
