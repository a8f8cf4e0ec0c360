"""torch.library registration of the model boundary, so that `torch.compile(network)` works.

The reference compiles the whole network before a rollout
(screamcast/earth2studio_wrappers.py:412-413, called at scripts/ace/run_screamcast_nudged.py:
639-641) and runs it under `torch.inference_mode()` (:452). The kernels of this package are
reached through ctypes on raw device pointers - nothing a tracing compiler can look into. The
whole network forward is therefore ONE custom operator,

    strata_b200::network_forward(x, lat, lon, handle) -> y

with a fake (shape / dtype only) implementation for tracing: Dynamo records a single opaque
call, `fullgraph=True` holds, Inductor has nothing to fuse across and launches the eager
implementation. `handle` names the module in a registry of live wrapper modules (weak
references); its weights are read from the module when the operator runs, they are not operator
arguments (inference only: there is no backward).

Finer-grained operators over the C ABI (`strata_b200::block_forward`, `::na3d`, `::linear`,
`::layernorm`) are registered the same way for callers that assemble their own graphs. Two of
them have gradients, for fine-tuning: `::linear_act` (a dense layer with its activation and residual) and
`::qk_norm_rope` (the norm and rotation of query and key heads).

Capturing a training step in a CUDA graph: torch ties a leaf's gradient accumulation to the stream on which its first
living graph was built, and a captured backward pass that meets an accumulation of another stream ends the
process. The two operators refuse the case they can see: a forward pass under capture whose leaves still have an
accumulation that a pass of these operators met on another stream. Delete the losses and outputs of warm-up steps
first; where something keeps the accumulations themselves (data-parallel wrappers do, as long as the module lives),
warm up and capture on one stream: `torch.cuda.graph(g, stream=s)`.
"""
from __future__ import annotations

import itertools
import weakref
from typing import Optional, Sequence

import torch

_MODULES: "weakref.WeakValueDictionary[int, torch.nn.Module]" = weakref.WeakValueDictionary()
_next_handle = itertools.count(1)


def register_module(module: torch.nn.Module) -> int:
    """Give a wrapper module a handle for `strata_b200::network_forward`."""
    h = next(_next_handle)
    _MODULES[h] = module
    return h


def _module(handle: int) -> torch.nn.Module:
    try:
        return _MODULES[handle]
    except KeyError:
        raise RuntimeError(f"strata_b200::network_forward: no live module with handle {handle}") from None


def _transform_probe():
    """A function that says whether a dispatch mode or a functorch transform (vmap, grad, jvp) is
    active. torch has no public call for either; without the private ones the answer is always yes."""
    modes = getattr(torch._C, "_len_torch_dispatch_stack", None)
    transforms = getattr(getattr(torch._C, "_functorch", None), "peek_interpreter_stack", None)
    if modes is None or transforms is None:
        return lambda: True
    return lambda: modes() != 0 or transforms() is not None


_transformed = _transform_probe()


def plain_call(x: torch.Tensor) -> bool:
    """Nothing is tracing or transforming this call - no compiler, no dispatch mode, no functorch
    transform, a plain CUDA tensor that asks for no gradient: the module's forward may then run
    directly, without the ~50 us the operator's Python dispatch takes."""
    return (type(x) is torch.Tensor and x.is_cuda and not torch.compiler.is_compiling()
            and not _transformed() and not (x.requires_grad and torch.is_grad_enabled()))


@torch.library.custom_op("strata_b200::network_forward", mutates_args=())
def network_forward(x: torch.Tensor, lat: torch.Tensor, lon: torch.Tensor, handle: int) -> torch.Tensor:
    return _module(handle)._forward_eager(x, lat, lon)


@network_forward.register_fake
def _network_forward_fake(x, lat, lon, handle):
    m = _module(handle)
    return x.new_empty((x.shape[0], m._out_chans, x.shape[2], x.shape[3], x.shape[4]))


# ------------------------------------------------------------------ operators over the C ABI
@torch.library.custom_op("strata_b200::layernorm", mutates_args=())
def layernorm(x: torch.Tensor, eps: float) -> torch.Tensor:
    from . import ops
    return ops.layernorm(x, eps)


@layernorm.register_fake
def _layernorm_fake(x, eps):
    return torch.empty_like(x)


@torch.library.custom_op("strata_b200::linear", mutates_args=())
def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], epilogue: int,
           aux: Optional[torch.Tensor]) -> torch.Tensor:
    from . import ops
    return ops.linear(x, weight, bias, epilogue, aux)


@linear.register_fake
def _linear_fake(x, weight, bias, epilogue, aux):
    return x.new_empty((*x.shape[:-1], weight.shape[0]))


@torch.library.custom_op("strata_b200::na3d", mutates_args=())
def na3d(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, kernel: Sequence[int]) -> torch.Tensor:
    from . import ops
    return ops.na3d(q, k, v, tuple(kernel))


@na3d.register_fake
def _na3d_fake(q, k, v, kernel):
    return q.new_empty(q.shape)


@torch.library.custom_op("strata_b200::block_forward", mutates_args=())
def block_forward(x: torch.Tensor, weights: Sequence[torch.Tensor], biases: Sequence[torch.Tensor],
                  grid: Sequence[int], num_heads: int, kernel: Sequence[int],
                  rope_cs: Optional[torch.Tensor], qk_norm: bool) -> torch.Tensor:
    """One backbone block. weights / biases: (qkv, proj, fc1, fc2[, gate]) in that order."""
    from . import ops
    names = ("qkv", "proj", "fc1", "fc2", "gate")
    w = {f"w_{n}": t for n, t in zip(names, weights)}
    w.update({f"b_{n}": t for n, t in zip(names, biases)})
    return ops.block_forward(x, w, grid=tuple(grid), num_heads=num_heads, kernel=tuple(kernel),
                             rope_cos=None, rope_sin=None, rope_cs=rope_cs, qk_norm=qk_norm)


@block_forward.register_fake
def _block_forward_fake(x, weights, biases, grid, num_heads, kernel, rope_cs, qk_norm):
    return torch.empty_like(x)


# ------------------------------------------------------------------ operators with gradients
_STREAM_TAG = "strata_b200.stream"


def claim_leaves(next_functions, stream: int, capturing: bool) -> None:
    """next_functions: those of a node of the graph that is being built. Notes with each leaf's gradient accumulation on
    which stream this forward pass runs, as long as a graph keeps the accumulation alive; refuses a captured pass over
    leaves whose accumulation belongs to another stream."""
    for node, _ in next_functions:
        if not hasattr(node, "variable"):         # only accumulations have one
            continue
        if node.metadata.setdefault(_STREAM_TAG, stream) != stream and capturing:
            raise RuntimeError(
                "this forward pass is being captured, but an eager graph of the same leaves is alive on another stream: "
                "its backward pass could not be captured. Delete what the eager passes returned (outputs, losses), "
                "or capture on their stream where something else keeps the leaves' gradient accumulation")


def _claim(ctx, x) -> None:
    from . import _lib
    if x.is_cuda and not isinstance(x, torch._subclasses.FakeTensor):
        claim_leaves(getattr(ctx, "next_functions", ()), _lib.stream_of(x), torch.cuda.is_current_stream_capturing())


@torch.library.custom_op("strata_b200::linear_act", mutates_args=())
def linear_act(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: str = "none",
               residual: Optional[torch.Tensor] = None, save_preact: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """(y, z) of ops.linear_act; z has no elements unless save_preact. Differentiable in x, weight, bias and residual;
    without save_preact the backward pass computes z again. z itself is not differentiable."""
    from . import ops
    if save_preact:
        return ops.linear_act(x, weight, bias, activation, residual, save_preact=True)
    return ops.linear_act(x, weight, bias, activation, residual), x.new_empty(0)


def _padded(x, width):
    """Rows as ops.linear_act lays them out: a view of whole 16-byte pieces."""
    if width % 8 == 0:
        return x.new_empty((*x.shape[:-1], width))
    return x.new_empty((*x.shape[:-1], (width + 7) // 8 * 8))[..., :width]


@linear_act.register_fake
def _linear_act_fake(x, weight, bias=None, activation="none", residual=None, save_preact=False):
    new = lambda: _padded(x, weight.shape[0])
    return new(), new() if save_preact else x.new_empty(0)


@torch.library.custom_op("strata_b200::linear_act_backward", mutates_args=())
def linear_act_backward(grad: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, activation: str,
                        preact: Optional[torch.Tensor], need_x: bool, need_weight: bool,
                        need_bias: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """ops.linear_act_backward; gradients that are not needed have no elements."""
    from . import ops
    got = ops.linear_act_backward(grad, x, weight, activation, preact, need_x=need_x, need_weight=need_weight,
                                  need_bias=need_bias)
    return tuple(x.new_empty(0) if t is None else t for t in got)


@linear_act_backward.register_fake
def _linear_act_backward_fake(grad, x, weight, activation, preact, need_x, need_weight, need_bias):
    return (_padded(x, x.shape[-1]) if need_x else x.new_empty(0), weight.new_empty(weight.shape if need_weight else 0),
            weight.new_empty(weight.shape[0] if need_bias else 0, dtype=torch.float32 if need_bias else x.dtype))


def _linear_act_context(ctx, inputs, output):
    x, weight, bias, activation, residual, save_preact = inputs
    _claim(ctx, x)
    ctx.set_materialize_grads(False)
    ctx.mark_non_differentiable(output[1])
    again = activation != "none" and not save_preact
    ctx.save_for_backward(x, weight, bias if again else None, output[1] if save_preact else None)
    ctx.activation, ctx.again = activation, again


def _each(ctx, grads):
    """One gradient for each argument that the call gave (defaults it left out have none)."""
    need = ctx.needs_input_grad
    return tuple(g if n else None for g, n in zip(grads, need)) + (None,) * (len(need) - len(grads))


def _linear_act_grad(ctx, dy, _dz):
    if dy is None:
        return _each(ctx, ())
    x, weight, bias, z = ctx.saved_tensors
    if ctx.again:
        z = torch.ops.strata_b200.linear_act(x, weight, bias, "none", None, False)[0]
    need = (*ctx.needs_input_grad, False)
    dx = dw = db = None
    if need[0] or need[1] or need[2]:
        dx, dw, db = torch.ops.strata_b200.linear_act_backward(
            dy, x, weight, ctx.activation, None if ctx.activation == "none" else z, need[0], need[1], need[2])
    return _each(ctx, (dx, dw, db, None, dy))


linear_act.register_autograd(_linear_act_grad, setup_context=_linear_act_context)


@torch.library.custom_op("strata_b200::qk_norm_rope", mutates_args=())
def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor] = None,
                 k_weight: Optional[torch.Tensor] = None, rope_cs: Optional[torch.Tensor] = None,
                 positions: Optional[torch.Tensor] = None, tokens_per_tile: Optional[int] = None,
                 hw: Optional[int] = None, eps: float = 1e-6,
                 interleaved: bool = True) -> tuple[torch.Tensor, torch.Tensor]:
    """ops.qk_norm_rope, differentiable in q, k and the two weights; a rope_cs that asks for a gradient is refused."""
    from . import ops
    return ops.qk_norm_rope(q, k, q_weight, k_weight, rope_cs=rope_cs, positions=positions,
                            tokens_per_tile=tokens_per_tile, hw=hw, eps=eps, interleaved=interleaved)


@qk_norm_rope.register_fake
def _qk_norm_rope_fake(q, k, q_weight=None, k_weight=None, rope_cs=None, positions=None, tokens_per_tile=None, hw=None,
                       eps=1e-6, interleaved=True):
    return q.new_empty(q.shape), k.new_empty(k.shape)


@torch.library.custom_op("strata_b200::qk_norm_rope_backward", mutates_args=())
def qk_norm_rope_backward(dq: torch.Tensor, dk: torch.Tensor, q: torch.Tensor, k: torch.Tensor,
                          q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor],
                          rope_cs: Optional[torch.Tensor], positions: Optional[torch.Tensor],
                          tokens_per_tile: Optional[int], hw: Optional[int], eps: float,
                          interleaved: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """ops.qk_norm_rope_backward; the gradient of a weight that is not there has no elements."""
    from . import ops
    got = ops.qk_norm_rope_backward(dq, dk, q, k, q_weight, k_weight, rope_cs=rope_cs, positions=positions,
                                    tokens_per_tile=tokens_per_tile, hw=hw, eps=eps, interleaved=interleaved)
    return tuple(q.new_empty(0, dtype=torch.float32) if t is None else t for t in got)


@qk_norm_rope_backward.register_fake
def _qk_norm_rope_backward_fake(dq, dk, q, k, q_weight, k_weight, rope_cs, positions, tokens_per_tile, hw, eps,
                                interleaved):
    w = lambda t: q.new_empty(0 if t is None else q.shape[-1], dtype=torch.float32)
    return q.new_empty(q.shape), k.new_empty(k.shape), w(q_weight), w(k_weight)


def _qk_norm_rope_context(ctx, inputs, output):
    q, k, q_weight, k_weight, rope_cs, positions, *ctx.rest = inputs
    if rope_cs is not None and rope_cs.requires_grad:
        raise NotImplementedError("rope_cs has no gradient: detach it")
    _claim(ctx, q)
    ctx.save_for_backward(q, k, q_weight, k_weight, rope_cs, positions)


def _qk_norm_rope_grad(ctx, dq, dk):
    q, k, q_weight, k_weight, rope_cs, positions = ctx.saved_tensors
    got = torch.ops.strata_b200.qk_norm_rope_backward(dq, dk, q, k, q_weight, k_weight, rope_cs, positions, *ctx.rest)
    return _each(ctx, got)


qk_norm_rope.register_autograd(_qk_norm_rope_grad, setup_context=_qk_norm_rope_context)
