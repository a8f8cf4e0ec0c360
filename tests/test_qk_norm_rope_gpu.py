"""Norm and rotation of q and k heads, forward and backward, against the formulas in 64 bits, element by element.

Tolerances (u: half a step of the type; everything else is fp32, a handful of roundings and rsqrt to 2^-22): forward 2^-19 of
|n w| summed over a pair (the rotation mixes two channels) + u |y|; backward 2^-18 of the terms' absolute sum + u |dx|; dw
(rows + 64) 2^-23 of the sum of absolute terms."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ops():
    from strata_b200 import ops
    return ops


def data(M, hq, hk, hd, t, *, rot=None, rows=None, f32=False, weights=True, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")
    qkv = (n(M, (hq + 2 * hk) * hd) * (0.1 + 3 * torch.rand(M, 1, generator=g, device="cuda"))).to(t)
    d = dict(q=qkv[:, :hq * hd].view(M, hq, hd), k=qkv[:, hq * hd:(hq + hk) * hd].view(M, hk, hd), qkv=qkv,
             dq=n(M, hq, hd).to(t), dk=n(M, hk, hd).to(t), qw=None, kw=None, cs=None)
    if weights:
        d["qw"], d["kw"] = n(hd), n(hd)
    if rot:
        a = torch.rand(rows, rot // 2, generator=g, device="cuda", dtype=torch.float64) * 100
        cs = torch.stack([a.cos(), a.sin()], -1)
        d["cs"] = cs.float() if f32 else cs.half()
    return d


def rotation64(cs, at, live, hd, adjacent):
    """[M, hd, hd] would be the matrix; returns a function that applies it, or its transpose, to [M, heads, hd]."""
    if cs is None:
        return lambda v, back=False: v
    cs = cs.double().reshape(-1, cs.shape[-2], 2)[at.clamp(min=0)]
    half = cs.shape[1]
    i = torch.arange(half, device="cuda")
    a, b = (2 * i, 2 * i + 1) if adjacent else (i, i + half)

    def turn(v, back=False):
        c, s = cs[:, None, :, 0], cs[:, None, :, 1] * (-1 if back else 1)
        out = v.clone()
        out[..., a] = v[..., a] * c - v[..., b] * s
        out[..., b] = v[..., a] * s + v[..., b] * c
        return out * live[:, None, None]
    return turn


def spread(v, cs, adjacent):
    """Upper bound of what a rotation makes of absolute values: each channel with its partner's added."""
    if cs is None:
        return v
    half = cs.shape[-2]
    i = torch.arange(half, device="cuda")
    a, b = (2 * i, 2 * i + 1) if adjacent else (i, i + half)
    out = v.clone()
    out[..., a] = out[..., b] = v[..., a] + v[..., b]
    return out


def near(got, want, slack, t):
    u = torch.finfo(t).eps / 2
    over = (got.double() - want).abs() - (slack + u * (want.abs() + slack) + (2.0 ** -25 if t == HF else 0.0))
    assert got.shape == want.shape and got.dtype == t
    assert float(over.max()) <= 0, f"{float(over.max()):.3e} beyond the tolerance at {int(over.argmax())}"


def check(ops, d, adjacent, at=None, live=None, eps=1e-6, **table):
    M, _, hd = d["q"].shape
    if at is None:
        at = torch.zeros(M, dtype=torch.int64, device="cuda")
    if live is None:
        live = torch.ones(M, dtype=torch.bool, device="cuda")
    turn = rotation64(d["cs"], at, live, hd, adjacent)
    kw = dict(rope_cs=d["cs"], eps=eps, interleaved=adjacent, **table)
    ys = ops.qk_norm_rope(d["q"], d["k"], d["qw"], d["kw"], **kw)
    gs = ops.qk_norm_rope_backward(d["dq"], d["dk"], d["q"], d["k"], d["qw"], d["kw"], **kw)
    assert all(torch.equal(a, b) if a is not None else b is None for a, b in
               zip(gs, ops.qk_norm_rope_backward(d["dq"], d["dk"], d["q"], d["k"], d["qw"], d["kw"], **kw)))
    for i, (x, w, dy) in enumerate(((d["q"], d["qw"], d["dq"]), (d["k"], d["kw"], d["dk"]))):
        t, x = x.dtype, x.double()
        w64 = 1.0 if w is None else w.double()
        r = ((x * x).mean(-1, keepdim=True) + eps).rsqrt()
        n = x * r
        near(ys[i], turn(n * w64), spread((n * w64).abs(), d["cs"], adjacent) * 2.0 ** -19, t)
        g = turn(dy.double(), True)
        ag = spread(dy.double().abs(), d["cs"], adjacent) if d["cs"] is not None else g.abs()
        h = g * w64
        terms = r * (ag * abs(w64) + n.abs() * (ag * abs(w64) * n.abs()).mean(-1, keepdim=True))
        near(gs[i], (r * (h - n * (h * n).mean(-1, keepdim=True))) * live[:, None, None], terms * 2.0 ** -18, t)
        if w is not None:
            dw, rows = (g * n).sum((0, 1)), M * x.shape[1]
            slack = (ag * n.abs() * live[:, None, None]).sum((0, 1)) * ((rows + 64) * 2.0 ** -23)
            assert gs[2 + i].dtype == torch.float32 and bool(((gs[2 + i].double() - dw).abs() <= slack).all())
    return ys, gs


# one token, odd counts, a head narrower than 16 bytes times two lanes, heads that fill no power of two, more heads than a
# warp's rounds hold, shared key heads
@pytest.mark.parametrize("M,hq,hk,hd,rot", [(1, 1, 1, 8, 8), (1, 16, 2, 128, 128), (5, 3, 1, 64, 64), (33, 12, 12, 64, 32),
                                            (257, 2, 2, 32, 16), (100, 5, 5, 48, 48), (513, 12, 3, 80, 32),
                                            (61, 4, 2, 96, 96), (40, 40, 8, 128, 64), (19, 2, 1, 256, 256),
                                            (3, 7, 3, 200, 96), (9001, 8, 8, 64, 64), (1000, 1, 1, 16, 16)])
@pytest.mark.parametrize("adjacent", [True, False])
@pytest.mark.parametrize("t,f32,weights", [(BF, False, True), (HF, True, False), (HF, False, True)])
def test_by_position(ops, M, hq, hk, hd, rot, adjacent, t, f32, weights):
    from strata_b200 import _lib
    if not adjacent and rot % 16:
        rot = 0
    d = data(M, hq, hk, hd, t, rot=rot, rows=77, f32=f32, weights=weights, seed=M)
    if not rot:
        check(ops, d, adjacent)
        return
    pos = torch.randint(0, 77, (M,), device="cuda", dtype=torch.int64 if f32 else torch.int32)
    pos[M // 2:M // 2 + 2] = torch.tensor([0, 76], device="cuda", dtype=pos.dtype)[:M - M // 2]
    check(ops, d, adjacent, pos.long(), positions=pos)
    assert _lib.device_status() == 0


# few tokens: a token's heads over several blocks, also where the last ones have no k heads, or no whole share
@pytest.mark.parametrize("M,hq,hk,hd", [(1, 48, 12, 256), (44, 48, 12, 256), (5, 48, 1, 128), (9, 3, 40, 64), (300, 13, 7, 64),
                                        (1100, 17, 3, 200), (2, 1000, 999, 8)])
@pytest.mark.parametrize("adjacent", [True, False])
def test_heads_over_several_blocks(ops, M, hq, hk, hd, adjacent):
    d = data(M, hq, hk, hd, BF, rot=hd if adjacent else hd // 16 * 16 or None, rows=M, f32=True, seed=M + hq)
    at = torch.arange(M - 1, -1, -1, device="cuda")
    live = at != M // 2 if M > 2 else torch.ones_like(at, dtype=torch.bool)
    if d["cs"] is None:
        check(ops, d, adjacent)
    else:
        check(ops, d, adjacent, at, live, positions=torch.where(live, at, -1))


@pytest.mark.parametrize("tiles,depth,hw", [(1, 1, 1), (3, 4, 50), (2, 16, 33)])
def test_by_tile_and_cell(ops, tiles, depth, hw):
    M = tiles * depth * hw
    d = data(M, 4, 4, 64, BF, rot=64, rows=tiles * hw)
    m = torch.arange(M, device="cuda")
    check(ops, d, True, m // (depth * hw) * hw + m % hw, tokens_per_tile=depth * hw, hw=hw)
    if depth == 1:
        check(ops, d, True, m)                       # token m has row m


@pytest.mark.parametrize("weights", [True, False])
def test_norm_alone(ops, weights):
    check(ops, data(301, 6, 2, 64, BF, weights=weights), True)
    check(ops, data(301, 6, 2, 72, HF, weights=weights), False, eps=0.5)


def test_same_as_the_norm_of_packed_rows(ops):
    d = data(1000, 4, 4, 64, BF, weights=False)
    packed = d["qkv"].clone()
    ops.qk_norm_rows_(packed, 256)
    q, k = ops.qk_norm_rope(d["q"], d["k"])
    # (both are the formula within half a step: they may differ by one)
    for a, b in ((q, packed[:, :256]), (k, packed[:, 256:512])):
        a, b = a.reshape(-1, 256).float(), b.float()
        assert bool(((a - b).abs() <= 2 * torch.finfo(BF).eps * b.abs()).all())


def test_in_place_leaves_the_values_alone(ops):
    d = data(777, 6, 2, 64, BF, rot=64, rows=777)
    want = ops.qk_norm_rope(d["q"], d["k"], d["qw"], d["kw"], rope_cs=d["cs"])
    v = d["qkv"][:, 8 * 64:].clone()
    got = ops.qk_norm_rope(d["q"], d["k"], d["qw"], d["kw"], rope_cs=d["cs"], out=(d["q"], d["k"]))
    assert got[0] is d["q"] and torch.equal(d["q"], want[0]) and torch.equal(d["k"], want[1])
    assert torch.equal(d["qkv"][:, 8 * 64:], v)
    with pytest.raises(ValueError):                  # overlapping rows cannot be written to
        ops.qk_norm_rope(d["q"], d["k"], out=(d["q"][:1].expand(777, 6, 64), d["k"]))


def test_layouts(ops):
    """Heads outermost, every second token, a grid of tokens, and addresses off the 16-byte grid."""
    M, h, hd = 96, 4, 64
    d = data(M, h, h, hd, HF, rot=hd, rows=M)
    want = ops.qk_norm_rope(d["q"], d["k"], d["qw"], d["kw"], rope_cs=d["cs"])
    grads = ops.qk_norm_rope_backward(d["dq"], d["dk"], d["q"], d["k"], d["qw"], d["kw"], rope_cs=d["cs"])
    for make in (lambda a: a.transpose(0, 1).contiguous().transpose(0, 1),
                 lambda a: torch.stack([a, a], 1)[:, 1],
                 lambda a: torch.cat([a.reshape(-1)[:3], a.reshape(-1)])[3:].view(a.shape),
                 lambda a: a.transpose(1, 2).contiguous().transpose(1, 2)):
        v = {k: make(d[k]) for k in ("q", "k", "dq", "dk")}
        got = ops.qk_norm_rope(v["q"], v["k"], d["qw"], d["kw"], rope_cs=d["cs"])
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        got = ops.qk_norm_rope_backward(v["dq"], v["dk"], v["q"], v["k"], d["qw"], d["kw"], rope_cs=d["cs"])
        assert all(torch.equal(a, b) for a, b in zip(got, grads))
    grid = lambda a: a.reshape(2, 3, 4, 4, h, hd)
    got = ops.qk_norm_rope(grid(d["q"]), grid(d["k"]), d["qw"], d["kw"], rope_cs=d["cs"].view(2, 48, hd // 2, 2))
    assert got[0].shape == (2, 3, 4, 4, h, hd) and torch.equal(got[0].view(M, h, hd), want[0])
    one = d["dq"][:1, :1, :1].expand(M, h, hd)
    a = ops.qk_norm_rope_backward(one, one, d["q"], d["k"])
    b = ops.qk_norm_rope_backward(one.contiguous(), one.contiguous(), d["q"], d["k"])
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("wide", [torch.int32, torch.int64])
def test_padding_tokens(ops, wide):
    """Negative positions: zero outputs and gradients and no part in dw, whatever stands in the rows."""
    d = data(90, 6, 2, 64, BF, rot=64, rows=50)
    pos = torch.randint(0, 50, (90,), device="cuda").to(wide)
    pos[30:45] = -1
    pos[89] = -(2 ** 31)
    dead = pos < 0
    for x in ("q", "k", "dq", "dk"):
        d[x] = d[x].clone()
        d[x][40], d[x][41], d[x][89] = float("nan"), float("inf"), float("-inf")
    ys = ops.qk_norm_rope(d["q"], d["k"], d["qw"], d["kw"], rope_cs=d["cs"], positions=pos)
    gs = ops.qk_norm_rope_backward(d["dq"], d["dk"], d["q"], d["k"], d["qw"], d["kw"], rope_cs=d["cs"], positions=pos)
    assert all(not bool(t[dead].any()) for t in (*ys, *gs[:2]))
    for x in ("q", "k", "dq", "dk"):
        d[x][dead] = 0
    clean = ops.qk_norm_rope_backward(d["dq"], d["dk"], d["q"], d["k"], d["qw"], d["kw"], rope_cs=d["cs"], positions=pos)
    assert all(torch.equal(a, b) for a, b in zip(gs, clean))
    check(ops, d, True, pos.long(), ~dead, positions=pos)


def test_positions_behind_the_table(ops):
    from strata_b200 import _lib
    d = data(20, 2, 1, 64, BF, rot=64, rows=10)
    pos = torch.arange(20, device="cuda") % 10
    pos[7], pos[12] = 10, 2 ** 40
    assert _lib.device_status() == 0
    q, k = ops.qk_norm_rope(d["q"], d["k"], d["qw"], d["kw"], rope_cs=d["cs"], positions=pos)
    assert _lib.device_status() == 107
    bad = torch.zeros(20, dtype=torch.bool, device="cuda")
    bad[7] = bad[12] = True
    for t in (q, k):
        assert t[bad].isnan().all() and not t[~bad].isnan().any()
    g = ops.qk_norm_rope_backward(d["dq"], d["dk"], d["q"], d["k"], rope_cs=d["cs"], positions=pos)
    assert _lib.device_status() == 107 and g[0][7].isnan().all() and not g[0][~bad].isnan().any()
    assert _lib.device_status() == 0


def test_no_tokens(ops):
    d = data(0, 4, 2, 64, BF)
    gs = ops.qk_norm_rope_backward(d["dq"], d["dk"], d["q"], d["k"], d["qw"], d["kw"])
    assert gs[0].shape == (0, 4, 64) and not gs[2].any() and not gs[3].any()


def test_offsets_beyond_32_bits(ops):
    M, h, hd = 1_100_000, 16, 256
    q = torch.randn(M, h, hd, device="cuda", dtype=BF)
    k = q[:, :1]
    a = torch.rand(M, hd // 2, device="cuda")
    cs = torch.stack([a.cos(), a.sin()], -1).half()
    yq, yk = ops.qk_norm_rope(q, k, rope_cs=cs)
    at = torch.tensor([0, M // 2, M - 1], device="cuda")
    wq, wk = ops.qk_norm_rope(q[at], k[at], rope_cs=cs[at])
    assert torch.equal(yq[at], wq) and torch.equal(yk[at], wk)


def test_captured_replayed_and_on_two_streams(ops):
    d, e = (data(4000, 8, 2, 64, BF, rot=64, rows=4000, seed=i) for i in range(2))
    s = {k: v.clone() for k, v in d.items() if k != "qkv"}
    run = lambda v: (*ops.qk_norm_rope(v["q"], v["k"], v["qw"], v["kw"], rope_cs=v["cs"]), *ops.qk_norm_rope_backward(
        v["dq"], v["dk"], v["q"], v["k"], v["qw"], v["kw"], rope_cs=v["cs"]))
    wants = [run(d), run(e)]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run(s)
    for v, want in zip((d, e), wants):
        for k in s:
            s[k].copy_(v[k])
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(10):
        for i, v in enumerate((d, e)):
            with torch.cuda.stream(streams[i]):
                got[i].append(run(v))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for i in range(2) for one in got[i] for a, b in zip(one, wants[i]))


# ------------------------------------------------------------------ together, and differentiable
def test_projection_norm_attention_projection(ops):
    """The attention half of a block from the pieces, as block_forward computes it: same values to bf16's rounding of the
    intermediate q and k (one more than the fused projection makes)."""
    tiles, D, H, W, C, heads = 2, 3, 8, 8, 128, 2
    T, M = D * H * W, 2 * D * H * W
    d = data(M, heads, heads, 64, BF, rot=64, rows=tiles * H * W, weights=False)
    g = torch.Generator("cuda").manual_seed(3)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x, wqkv, bqkv = n(M, C).to(BF), (n(3 * C, C) * C ** -0.5).to(BF), n(3 * C) * 0.1
    wp, bp = (n(C, C) * C ** -0.5).to(BF), n(C) * 0.1
    cs = d["cs"].view(tiles, H * W, 32, 2)
    grid = lambda t: t.reshape(tiles, D, H, W, heads, 64)

    def half(q, k, v):
        a = ops.na3d(grid(q), grid(k), grid(v), (3, 3, 3))
        return ops.linear_act(a.view(M, C), wp, bp, "none", x)

    qkv = ops.linear_act(x, wqkv, bqkv)
    q, k = ops.qk_norm_rope(*(t.view(M, heads, 64) for t in (qkv[:, :C], qkv[:, C:2 * C])), rope_cs=cs, tokens_per_tile=T,
                            hw=H * W)
    got = half(q, k, qkv[:, 2 * C:])
    fused = ops.qkv_rope(x, wqkv, bqkv, 64, None, None, T, H * W, qk_norm=True, rope_cs=cs)
    want = half(*(fused[:, i * C:(i + 1) * C].contiguous() for i in range(3)))
    # q and k carry one more rounding (2^-8 at most); their scores, and so the result, move by a few times that
    assert float((got.float() - want.float()).abs().max() / want.float().abs().max()) < 2e-2


def test_operator_registration(ops):
    from strata_b200 import torch_ops  # noqa: F401
    d = data(30, 4, 2, 64, BF, rot=64, rows=30)
    q, k, qw, kw = (d[n].clone().requires_grad_() for n in ("q", "k", "qw", "kw"))
    pos = torch.arange(30, device="cuda").flip(0)
    torch.library.opcheck(torch.ops.strata_b200.qk_norm_rope, (q, k, qw, kw, d["cs"], pos),
                          test_utils=("test_schema", "test_faketensor", "test_autograd_registration"))
    f = torch.compile(lambda q, k, qw, kw: torch.ops.strata_b200.qk_norm_rope(q, k, qw, kw, d["cs"], pos), fullgraph=True)
    torch.autograd.backward(f(q, k, qw, kw), (d["dq"], d["dk"]))
    want = ops.qk_norm_rope_backward(d["dq"], d["dk"], d["q"], d["k"], d["qw"], d["kw"], rope_cs=d["cs"], positions=pos)
    assert all(torch.equal(t.grad, v) for t, v in zip((q, k, qw, kw), want))


def test_gradients_through_projection_norm_and_mlp(ops):
    """A training step over the differentiable operators against autograd in 64 bits on the same bf16 weights: bf16 keeps 8
    bits of every intermediate value and gradient, four roundings in a row of 2^-9 rms each at most."""
    from strata_b200 import torch_ops  # noqa: F401
    S = torch.ops.strata_b200
    M, C, heads, hd = 500, 96, 3, 32
    g = torch.Generator("cuda").manual_seed(5)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")
    a = torch.rand(M, hd // 2, generator=g, device="cuda", dtype=torch.float64) * 6
    cs = torch.stack([a.cos(), a.sin()], -1).half()
    x = n(M, C).to(BF)
    p = dict(wqkv=(n(2 * C, C) * C ** -0.5).to(BF), bqkv=n(2 * C) * 0.1, qw=1 + 0.1 * n(hd), kw=1 + 0.1 * n(hd),
             w1=(n(4 * C, C) * C ** -0.5).to(BF), b1=n(4 * C) * 0.1, w2=(n(C, 4 * C) * (4 * C) ** -0.5).to(BF), b2=n(C) * 0.1)
    up = n(M, C).to(BF)

    def kernels(x, p):
        qk = S.linear_act(x, p["wqkv"], p["bqkv"])[0]
        q, k = S.qk_norm_rope(qk[:, :C].view(M, heads, hd), qk[:, C:].view(M, heads, hd), p["qw"], p["kw"], cs)
        h = (q + k).reshape(M, C)
        h1 = S.linear_act(h, p["w1"], p["b1"], "gelu", None, True)[0]
        return S.linear_act(h1, p["w2"], p["b2"], "none", h)[0]

    def plain(x, p):
        qk = x @ p["wqkv"].T + p["bqkv"]
        c, s = cs.double()[:, None, :, 0], cs.double()[:, None, :, 1]

        def one(v, w):
            v = v.view(M, heads, hd)
            v = v * ((v * v).mean(-1, keepdim=True) + 1e-6).rsqrt() * w
            e, o = v[..., 0::2], v[..., 1::2]
            return torch.stack([e * c - o * s, e * s + o * c], -1).flatten(-2)
        h = (one(qk[:, :C], p["qw"]) + one(qk[:, C:], p["kw"])).reshape(M, C)
        return torch.nn.functional.gelu(h @ p["w1"].T + p["b1"]) @ p["w2"].T + p["b2"] + h

    leaves = {k: v.clone().requires_grad_() for k, v in p.items()}
    xl = x.clone().requires_grad_()
    kernels(xl, leaves).backward(up)
    doubles = {k: v.double().requires_grad_() for k, v in p.items()}
    xd = x.double().requires_grad_()
    plain(xd, doubles).backward(up.double())
    for name, got, want in [("x", xl.grad, xd.grad)] + [(k, leaves[k].grad, doubles[k].grad) for k in p]:
        assert float((got.double() - want).norm() / want.norm()) < 1.5e-2, name
