"""Operators that are measured one by one: a dense layer with its epilogue and the norm-and-rotation of query and key
heads, each forward and backward.

A case is a dict of plain values with an "op":

  linear        y = residual + act(x W^T + b), optionally with the pre-activation z = x W^T + b besides
  linear_grad   dx, dW and db of it from dy, x, W and the stored z
  qk            per-head RMS norm of q and k (learned weights or none) and the rotary turn, in one pass
  qk_grad       the gradients of that in q, k and the two weights

Sums of many terms are taken in 64 bits in the plain form where the output has 32.
"""
from __future__ import annotations

import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------- the cases
def _linear(name, op, rows, k, n, act, *, dtype="bf16", bias=True, residual=False, preact=False):
    return dict(name=name, op=op, rows=rows, k=k, n=n, act=act, dtype=dtype, bias=bias, residual=residual,
                preact=preact)


def _qk(name, op, rows, hq, hk, hd, rot, table, *, dtype="bf16", weights=True, adjacent=True, tiles=0, hw=0):
    return dict(name=name, op=op, rows=rows, hq=hq, hk=hk, hd=hd, rot=rot, table=table, dtype=dtype, weights=weights,
                adjacent=adjacent, tiles=tiles, hw=hw)


def listed():
    return [
        # one token through a wide layer: nothing but the weights' way through the chip and the launch
        _linear("linear_token", "linear", 1, 1024, 4096, "gelu_tanh"),
        # a handful of tokens back into the residual stream: few rows, few output tiles, a long sum
        _linear("linear_few", "linear", 24, 4096, 1024, "none", dtype="fp16", residual=True),
        # field channels into a narrow model: a width that is no multiple of 8, rows that fill no tile
        _linear("linear_ragged", "linear", 10473, 207, 650, "silu", dtype="fp16", residual=True),
        # the first MLP layer of a training step on one production tile's tokens (24 x 64 x 64), z kept
        _linear("linear_keep", "linear", 98304, 512, 2048, "gelu", preact=True),
        # the widest call: four tiles of 16 x 64 x 64 tokens, inference
        _linear("linear_tiles", "linear", 262144, 512, 2048, "silu"),
        # gradients on one small tile: a fine-tuning step of the test-suite's size
        _linear("grad_small", "linear_grad", 1024, 128, 512, "gelu_tanh"),
        # gradients of the ragged layer
        _linear("grad_ragged", "linear_grad", 10473, 207, 650, "relu", dtype="fp16"),
        # both gradients of a wide second MLP layer (no activation): the largest product
        _linear("grad_wide", "linear_grad", 98304, 4096, 1024, "none"),
        # a few tokens, shared key heads, float table by position
        _qk("qk_tokens", "qk", 5, 16, 2, 128, 128, "position", adjacent=False),
        # the benchmark's four tiles: 8 heads of 64, half table by horizontal cell, packed qkv rows
        _qk("qk_tiles", "qk", 262144, 8, 8, 64, 64, "tile", tiles=4, hw=4096),
        # gradients of a batch of padded sequences, part of each head turned, a head that is no power of two wide
        _qk("qk_grad_ragged", "qk_grad", 9973, 12, 3, 80, 32, "position", dtype="fp16", adjacent=False),
        # gradients on one production tile: 12 heads of 64
        _qk("qk_grad_tile", "qk_grad", 98304, 12, 12, 64, 64, "tile", tiles=1, hw=4096),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("linear", "linear", "linear_grad", "qk", "qk_grad"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    while True:
        if op.startswith("linear"):
            width = lambda: (8 * _log_int(rng, 2, 512)) if rng.random() < 0.7 else _log_int(rng, 9, 4096)
            c = _linear("", op, _log_int(rng, 1, 262144), width(), width(),
                        rng.choice(("none", "gelu", "gelu_tanh", "silu", "relu")), dtype=dtype,
                        bias=rng.random() < 0.8)
            if op == "linear":
                c["residual"] = rng.random() < 0.5
                c["preact"] = rng.random() < 0.3
        else:
            hd = rng.choice((32, 48, 64, 64, 80, 96, 128, 128, 256))
            hk = rng.choice((1, 2, 3, 4, 8, 12))
            hq = hk * rng.choice((1, 1, 2, 4))
            rows = _log_int(rng, 1, 262144)
            table = rng.choice(("none", "position", "tile"))
            c = _qk("", op, rows, hq, hk, hd, rng.choice((hd, hd, hd // 16 * 8)), table, dtype=dtype,
                    weights=rng.random() < 0.7, adjacent=rng.random() < 0.5)
            if c["rot"] % 16:
                c["adjacent"] = True
            if table == "tile":
                depth, tiles = rng.choice((1, 4, 16)), rng.choice((1, 2, 4))
                hw = max(1, rows // (depth * tiles))
                c["tiles"], c["hw"], c["rows"] = tiles, hw, depth * tiles * hw
        w = work(c)
        if w["flops"] <= 1.6e12 and w["bytes"] <= 1.3e9:
            del c["name"]
            return c


# ------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(int(seed))
    t = _TYPES[case["dtype"]]
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda")
    M = case["rows"]
    s = dict(case)
    if case["op"].startswith("linear"):
        K, N = case["k"], case["n"]
        s["x"] = normal(M, K).to(t)                                   # normalised tokens
        s["w"] = (normal(N, K) * K ** -0.5).to(t)
        s["b"] = normal(N) * 0.3 if case["bias"] else None
        s["r"] = normal(M, N).to(t) if case["residual"] else None
        if case["op"] == "linear_grad":
            z = (s["x"] @ s["w"].t()).float()
            s["z"] = (z + s["b"] if case["bias"] else z).to(t) if case["act"] != "none" else None
            s["dy"] = (normal(M, N) * 0.05).to(t)
        return s
    hq, hk, hd = case["hq"], case["hk"], case["hd"]
    packed = normal(M, (hq + 2 * hk) * hd)
    packed *= 0.5 + 2 * torch.rand(M, 1, generator=g, device="cuda")      # tokens of different size
    packed = packed.to(t)
    s["q"] = packed[:, :hq * hd].view(M, hq, hd)
    s["k"] = packed[:, hq * hd:(hq + hk) * hd].view(M, hk, hd)
    s["qw"], s["kw"] = ((1 + 0.2 * normal(hd), 1 + 0.2 * normal(hd)) if case["weights"] else (None, None))
    s["cs"], s["pos"], s["per_tile"], s["cells"] = None, None, None, None
    half = case["rot"] // 2
    if case["table"] == "position":
        # sequences one behind the other, the last one padded
        rows = max(16, 2 * M)
        f = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
        a = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * f
        s["cs"] = torch.stack([a.cos(), a.sin()], -1).float()
        pos = torch.randint(0, rows - M + 1, (1,), generator=g, device="cuda") + torch.arange(M, device="cuda")
        if M >= 16:
            pos[M // 2:] -= pos[M // 2].clone()
            pos[M - M // 16:] = -1
        s["pos"] = pos
    elif case["table"] == "tile":
        f = 100.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
        where = torch.rand(case["tiles"], case["hw"], 1, generator=g, device="cuda", dtype=torch.float64) * 64 - 32
        a = where * f
        s["cs"] = torch.stack([a.cos(), a.sin()], -1).half()
        s["per_tile"], s["cells"] = M // case["tiles"], case["hw"]
    if case["op"] == "qk_grad":
        s["dq"], s["dk"] = (normal(M, hq, hd) * 0.05).to(t), (normal(M, hk, hd) * 0.05).to(t)
    return s


# ------------------------------------------------------------------------------- one pass
def run(state):
    s = state
    if own:
        from strata_b200 import ops
        if s["op"] == "linear":
            return ops.linear_act(s["x"], s["w"], s["b"], s["act"], s["r"], save_preact=s["preact"])
        if s["op"] == "linear_grad":
            return ops.linear_act_backward(s["dy"], s["x"], s["w"], s["act"], s["z"], need_bias=s["bias"])
        table = dict(rope_cs=s["cs"], positions=s["pos"], tokens_per_tile=s["per_tile"], hw=s["cells"], eps=1e-6,
                     interleaved=s["adjacent"])
        if s["op"] == "qk":
            return ops.qk_norm_rope(s["q"], s["k"], s["qw"], s["kw"], **table)
        return ops.qk_norm_rope_backward(s["dq"], s["dk"], s["q"], s["k"], s["qw"], s["kw"], **table)
    if s["op"] == "linear":
        return _plain_linear(s)
    if s["op"] == "linear_grad":
        return _plain_linear_grad(s)
    turn = _plain_turn(s)
    if s["op"] == "qk":
        return _plain_qk(s["q"], s["qw"], s, turn), _plain_qk(s["k"], s["kw"], s, turn)
    dq, dqw = _plain_qk_grad(s["dq"], s["q"], s["qw"], s, turn)
    dk, dkw = _plain_qk_grad(s["dk"], s["k"], s["kw"], s, turn)
    return dq, dk, dqw, dkw


def _act(z, act):
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh((2 / math.pi) ** 0.5 * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z * (z > 0) if act == "relu" else z


def _act_slope(z, act):
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * 0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    if act == "gelu_tanh":
        c = (2 / math.pi) ** 0.5
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    if act == "silu":
        q = 1 / (1 + torch.exp(-z))
        return q * (1 + z * (1 - q))
    return (z > 0).to(z.dtype)


def _plain_linear(s):
    z = s["x"].float() @ s["w"].float().t()
    if s["b"] is not None:
        z = z + s["b"]
    y = _act(z, s["act"])
    if s["r"] is not None:
        y = y + s["r"].float()
    y = y.to(s["x"].dtype)
    return (y, z.to(s["x"].dtype)) if s["preact"] else y


def _plain_linear_grad(s):
    t = s["x"].dtype
    dz = s["dy"].float()
    if s["act"] != "none":
        dz = dz * _act_slope(s["z"].float(), s["act"])
    db = dz.double().sum(0).float() if s["bias"] else None
    return (dz @ s["w"].float()).to(t), (dz.t() @ s["x"].float()).to(t), db


def _plain_turn(s):
    """(cos, sin, live) of every token: [rows, 1, rot / 2] each and [rows, 1, 1]; None without a table."""
    if s["cs"] is None:
        return None
    cs = s["cs"].float().reshape(-1, s["rot"] // 2, 2)
    m = torch.arange(s["rows"], device="cuda")
    if s["pos"] is not None:
        at, live = s["pos"].clamp(min=0), s["pos"] >= 0
    else:
        at, live = m // s["per_tile"] * s["cells"] + m % s["cells"], m >= 0
    cs = cs[at][:, None]
    return cs[..., 0], cs[..., 1], live[:, None, None]


def _rotate(x, turn, s, sign):
    cos, sin, _ = turn
    half = s["rot"] // 2
    sin = sin * sign
    y = x.clone()
    if s["adjacent"]:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        y[..., :half], y[..., half:2 * half] = a * cos - b * sin, a * sin + b * cos
    return y


def _plain_qk(x, w, s, turn):
    t = x.dtype
    x = x.float()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    if w is not None:
        y = y * w
    if turn is not None:
        y = _rotate(y, turn, s, 1.0) * turn[2]
    return y.to(t)


def _plain_qk_grad(dy, x, w, s, turn):
    t = x.dtype
    x, g = x.float(), dy.float()
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    n = x * r
    if turn is not None:
        g = _rotate(g, turn, s, -1.0) * turn[2]
    dw = (g * n).double().sum((0, 1)).float() if w is not None else None
    if w is not None:
        g = g * w
    return (r * (g - n * (g * n).mean(-1, keepdim=True))).to(t), dw


# ------------------------------------------------------------------------------- work and the definition
def work(case):
    """Every input and output once; two operations for each multiply-add of the products, a few for each value of a
    row operator."""
    c, M = case, case["rows"]
    if c["op"] == "linear":
        K, N = c["k"], c["n"]
        return {"bytes": 2 * (M * K + N * K + M * N * (1 + c["residual"] + c["preact"])) + 4 * N * c["bias"],
                "flops": 2 * M * N * K}
    if c["op"] == "linear_grad":
        K, N = c["k"], c["n"]
        return {"bytes": 2 * (M * N * (1 + (c["act"] != "none")) + 2 * M * K + 2 * N * K) + 4 * N * c["bias"],
                "flops": 4 * M * N * K}
    values = M * (c["hq"] + c["hk"]) * c["hd"]
    if c["table"] == "tile":
        table = c["tiles"] * c["hw"] * c["rot"] * 2
    else:
        table = (M * c["rot"] * 4 + 8 * M) if c["table"] == "position" else 0
    grad = c["op"] == "qk_grad"
    return {"bytes": 2 * values * (3 if grad else 2) + table + 4 * c["hd"] * c["weights"] * (4 if grad else 2),
            "flops": values * (16 if grad else 8)}


def exact(case, seed):
    s = prepare(case, seed)
    d = lambda v: None if v is None else v.to(torch.float64)
    if case["op"].startswith("linear"):
        x, w, z = d(s["x"]), d(s["w"]), d(s.get("z"))
        if case["op"] == "linear":
            z = torch.einsum("mk,nk->mn", x, w)
            if case["bias"]:
                z += d(s["b"])
        a = slope = None
        kind = case["act"]
        if kind == "none":
            a, slope = z, 1.0
        elif kind == "relu":
            a, slope = z.clamp(min=0), torch.where(z > 0, 1.0, 0.0).double()
        elif kind == "silu":
            p = torch.sigmoid(z)
            a, slope = z * p, p + z * p * torch.sigmoid(-z)
        elif kind == "gelu":
            p = torch.special.ndtr(z)
            a, slope = z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        else:
            # z sigma(v), v = 2 sqrt(2 / pi) (z + 0.044715 z^3)
            c = 2 * math.sqrt(2 / math.pi)
            p = torch.sigmoid(c * (z + 0.044715 * z ** 3))
            a, slope = z * p, p + z * p * (1 - p) * c * (1 + 0.134145 * z ** 2)
        if case["op"] == "linear":
            y = a + d(s["r"]) if case["residual"] else a
            return (y, z) if case["preact"] else y
        dz = d(s["dy"]) * slope
        db = torch.einsum("mn->n", dz) if case["bias"] else None
        return torch.einsum("mn,nk->mk", dz, w), torch.einsum("mn,mk->nk", dz, x), db
    M, hd, half = case["rows"], case["hd"], case["rot"] // 2
    unit = live = None
    if s["cs"] is not None:
        unit = torch.view_as_complex(d(s["cs"]).reshape(-1, half, 2).contiguous())
        if s["pos"] is not None:
            live = s["pos"] >= 0
            unit = unit[torch.where(live, s["pos"], 0)]
        else:
            unit = unit.reshape(case["tiles"], 1, case["hw"], half).expand(-1, M // (case["tiles"] * case["hw"]), -1, -1)
            unit = unit.reshape(M, half)

    def turned(v, back):
        if unit is None:
            return v
        part = v[..., :2 * half]
        pairs = part.unflatten(-1, (half, 2)) if case["adjacent"] else part.unflatten(-1, (2, half)).transpose(-1, -2)
        c = torch.view_as_complex(pairs.contiguous()) * (unit.conj() if back else unit)[:, None]
        c = torch.view_as_real(c)
        c = c.flatten(-2) if case["adjacent"] else c.transpose(-1, -2).flatten(-2)
        v = torch.cat([c, v[..., 2 * half:]], -1)
        return v if live is None else v * live[:, None, None]

    def of(x, w, dy):
        x, w = d(x), d(w)
        size = (x.square().sum(-1, keepdim=True) / hd + 1e-6).sqrt()
        n = x / size
        if dy is None:
            return turned(n if w is None else n * w, False)
        g = turned(d(dy), True)
        dw = None if w is None else torch.einsum("mhc,mhc->c", g, n)
        h = g if w is None else g * w
        return (h - n * (h * n).sum(-1, keepdim=True) / hd) / size, dw

    if case["op"] == "qk":
        return of(s["q"], s["qw"], None), of(s["k"], s["kw"], None)
    (dq, dqw), (dk, dkw) = of(s["q"], s["qw"], s["dq"]), of(s["k"], s["kw"], s["dk"])
    return dq, dk, dqw, dkw
