"""Routed experts on libkmc.so: rows go to their k best experts and get a weighted sum of the experts' products.

The reference (kakollu/mlx-kmeans) answers with the one nearest center of a row; these operators carry fitted
centers (or any gate's scores) on to a mixture of experts:

    ids, weights = route(logits, top_k)            # the k best experts of every row, and their weights
    groups = group_rows(ids, n_experts)            # the (row, choice) pairs grouped by expert
    y = expert_matmul(x, w, groups)                # each group times its expert's matrix
    out = combine_rows(y, groups, weights)         # a row's results summed with its weights

All arguments are CUDA tensors; work is enqueued on the current stream and nothing synchronises.  route,
expert_matmul and combine_rows are differentiable through torch.autograd, once: their gradients have no derivative of
their own, and asking for one (create_graph) is a RuntimeError, as is forward-mode differentiation.  route_grad,
expert_matmul_grad and combine_rows_grad are the same gradients as plain calls.  group_rows takes labels too, as an int32
CUDA tensor -- KMeans.labels_ is a NumPy array on the host: torch.as_tensor(km.labels_).to("cuda", torch.int32) -- to run
one product per cluster.  Errors: ValueError for bad arguments, RuntimeError for a device failure.
Calls can be captured in a CUDA graph.
"""
import os
from typing import NamedTuple, Optional

import torch

from . import _lib

_SCORES = {"softmax": 0, "sigmoid": _lib.KMC_ROUTE_SIGMOID}
_module = None


def _ext():
    """The compiled module _experts.so beside this file (built by mlx_kmeans_b200/build.py); there is no fallback."""
    global _module
    if _module is None:
        path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_experts.so")
        if not os.path.exists(path):
            raise RuntimeError(f"{path} is missing: build it with `python -m mlx_kmeans_b200.build`")
        from . import _experts
        _module = _experts
    return _module


class RowGroups(NamedTuple):
    """The grouping of (row, choice) pairs by expert (group_rows), int32 CUDA tensors.

    offsets (n_experts + 1): expert e has the positions offsets[e] .. offsets[e + 1] - 1.
    rows (pairs): the row each position reads, -1 past offsets[-1].
    slot (rows, choices) or (rows,): the position of each pair, -1 for a pair that was left out.  A caller may set
    further ones to -1 before the first use (experts over their capacity): combine_rows leaves those pairs out, and its
    gradient at their positions is 0, so nothing of them reaches the gradients of expert_matmul.
    """
    offsets: torch.Tensor
    rows: torch.Tensor
    slot: torch.Tensor


def _tensors(*named):
    for t, name in named:
        if not isinstance(t, torch.Tensor):
            raise ValueError(f"{name} must be a CUDA tensor")


def _plan(groups):
    """offsets, rows and slot of a RowGroups (or a tuple of the three)."""
    if not isinstance(groups, (tuple, list)) or len(groups) != 3 or not all(isinstance(t, torch.Tensor) for t in groups):
        raise ValueError("groups must be a RowGroups (group_rows)")
    return groups


def expert_status(device=None):
    """Raise RuntimeError if an expert_matmul (or its gradient) on `device` gave up waiting on a barrier and no call has
    raised it yet, which leaves its result incomplete: a fault of the library or the device, since no wait depends on the
    data.  Waits for the device's current stream.  A later expert_matmul or gradient on the device raises it too, once the
    kernel has ended."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    _ext().status(device.index if device.index is not None else torch.cuda.current_device())


class _Once(torch.autograd.Function):
    """A function with a backward pass alone."""
    @staticmethod
    def jvp(ctx, *_):
        raise RuntimeError("route, expert_matmul and combine_rows have no forward-mode derivative")


class _Last(torch.autograd.Function):
    """Gradients tied to everything they depend on, so that a derivative taken through them is refused, whichever of
    those it is asked for."""
    @staticmethod
    def forward(ctx, n, *tensors):
        return tuple(t.view_as(t) for t in tensors[:n])

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("route, expert_matmul and combine_rows have no second derivative")


def _last(grads, *sources):
    """The gradients of a backward pass (None where there is none), made from `sources`."""
    if not torch.is_grad_enabled():                            # create_graph is not set
        return grads
    some = [g for g in grads if g is not None]
    done = iter(_Last.apply(len(some), *some, *sources)) if some else iter(())
    return tuple(None if g is None else next(done) for g in grads)


# ---------------------------------------------------------------- routing

def _route_flags(score, renormalize):
    if score not in _SCORES:
        raise ValueError(f"score must be 'softmax' or 'sigmoid', got {score!r}")
    return _SCORES[score] | (_lib.KMC_ROUTE_RENORM if renormalize else 0)


class _Route(_Once):
    @staticmethod
    def forward(ctx, logits, top_k, flags, bias, groups, top_groups, scale, mask):
        ids, weights = _ext().route(logits, top_k, flags, bias, groups, top_groups, scale, mask)
        ctx.save_for_backward(logits, ids)
        ctx.flags, ctx.scale = flags, scale
        ctx.mark_non_differentiable(ids)
        return ids, weights

    @staticmethod
    def backward(ctx, _dids, dweights):
        logits, ids = ctx.saved_tensors
        dl = _ext().route_grad(dweights.float(), logits, ids, ctx.flags, ctx.scale)
        return (*_last((dl,), dweights, logits), None, None, None, None, None, None, None)


def route(logits, top_k, *, score="softmax", bias=None, groups=1, top_groups=1, renormalize=True, scale=1.0, mask=None):
    """The top_k best experts of every row of logits (rows, n_experts) and their weights.

    logits: float32, bfloat16 or float16, up to 1024 experts, rows any distance apart.  Returns ids (rows, top_k)
    int32, best first (lowest index on ties), and weights (rows, top_k) float32.
    score: "softmax" over the experts, or each expert's "sigmoid".  renormalize: over the chosen experts only.
    scale multiplies the weights.
    bias (n_experts float32): added to the logits (softmax) or scores (sigmoid) for the choice, not for the weights.
    groups, top_groups: of `groups` groups of consecutive experts only the top_groups with the largest sum of their
    two best keys are chosen from.
    mask (rows, bool): rows that are False get no expert.
    An expert whose logit or biased key is -inf or NaN is not chosen; where fewer than top_k are left, the id is -1
    and the weight 0.
    """
    _tensors((logits, "logits"))
    flags = _route_flags(score, renormalize)
    if bias is not None:
        _tensors((bias, "bias"))
        bias = bias.detach()
    if mask is not None:
        _tensors((mask, "mask"))
    args = (logits, top_k, flags, bias, groups, top_groups, scale, mask)
    if logits.requires_grad and torch.is_grad_enabled():
        return _Route.apply(*args)
    return _ext().route(*args)


def route_grad(dweights, logits, ids, *, score="softmax", renormalize=True, scale=1.0):
    """The gradient of route's weights with respect to the logits: dlogits (rows, n_experts) in the logits' type, from
    dweights (rows, top_k) and the ids that route gave for these logits, score, renormalize and scale."""
    _tensors((logits, "logits"), (ids, "ids"), (dweights, "dweights"))
    return _ext().route_grad(dweights, logits, ids, _route_flags(score, renormalize), scale)


# ---------------------------------------------------------------- grouping

def group_rows(ids, n_experts):
    """Group (row, choice) pairs by expert: RowGroups of ids (rows, choices) or (rows,) int32, up to 4096 experts.

    Labels are the (rows,) form.  Other integer types and host arrays are refused, not converted.
    Stable: an expert's pairs keep their order.  ids outside [0, n_experts) are left out (slot -1)."""
    _tensors((ids, "ids"))
    return RowGroups(*_ext().group_rows(ids, n_experts))


# ---------------------------------------------------------------- products per expert

class _ExpertMatmul(_Once):
    @staticmethod
    def forward(ctx, x, w, offsets, rows, slot, gather):
        ctx.save_for_backward(x, w, offsets, rows, slot)
        ctx.gather = gather
        return _ext().expert_matmul(x, w, offsets, rows, slot, gather)

    @staticmethod
    def backward(ctx, dy):
        x, w, offsets, rows, slot = ctx.saved_tensors
        dx = _ext().expert_dx(dy, w, offsets, rows, slot, ctx.gather) if ctx.needs_input_grad[0] else None
        dw = _ext().expert_dw(dy, x, offsets, rows, slot, ctx.gather) if ctx.needs_input_grad[1] else None
        return (*_last((dx, dw), dy, x, w), None, None, None, None)


def expert_matmul(x, w, groups, *, gather=True):
    """Each position's row times its expert's matrix: y (positions, n) with y[p] = w[e] @ x[row of p].

    x: (rows, d) and every position reads its row (gather=True), or (positions, d) already grouped (gather=False).
    w: (n_experts, n, d), bfloat16 or float16 as x; sums are float32.  Positions past groups.offsets[-1] are zero."""
    _tensors((x, "x"), (w, "w"))
    if (x.requires_grad or w.requires_grad) and torch.is_grad_enabled():
        return _ExpertMatmul.apply(x, w, *_plan(groups), bool(gather))
    return _ext().expert_matmul(x, w, *_plan(groups), bool(gather))


def expert_matmul_grad(dy, x, w, groups, *, gather=True):
    """The gradients of expert_matmul for dy (positions, n): dx in x's shape (with gather=True the positions of a row's
    slots are summed in float32 and the sum is rounded) and dw in w's; an expert with no position gets a dw of zeros."""
    _tensors((dy, "dy"), (x, "x"), (w, "w"))
    if x.ndim == 2 and w.ndim == 3 and x.shape[1] != w.shape[2]:
        raise ValueError(f"x has {x.shape[1]} columns, the matrices {w.shape[2]}")
    ext, groups, gather = _ext(), _plan(groups), bool(gather)
    return ext.expert_dx(dy, w, *groups, gather), ext.expert_dw(dy, x, *groups, gather)


# ---------------------------------------------------------------- combination

class _Combine(_Once):
    @staticmethod
    def forward(ctx, y, weights, offsets, rows, slot):
        ctx.save_for_backward(y, weights, offsets, rows, slot)
        return _ext().combine(y, offsets, rows, slot, weights)

    @staticmethod
    def backward(ctx, dout):
        y, weights, offsets, rows, slot = ctx.saved_tensors
        dy, dw = _ext().combine_grad(dout, y, offsets, rows, slot, weights)
        return (*_last((dy, dw), dout, y, *(() if weights is None else (weights,))), None, None, None)


def combine_rows(y, groups, weights: Optional[torch.Tensor] = None):
    """A row's results summed: out (rows, features) with out[t] = sum over its choices of weight * y[slot].

    y: (positions, features), float32, bfloat16 or float16; weights float32 in the shape of the ids, or None for 1.
    The sum is float32, rounded once; a pair that was left out adds nothing."""
    _tensors((y, "y"), (weights if weights is not None else y, "weights"))
    groups = _plan(groups)
    if (y.requires_grad or (weights is not None and weights.requires_grad)) and torch.is_grad_enabled():
        return _Combine.apply(y, weights, *groups)
    return _ext().combine(y, *groups, weights)


def combine_rows_grad(dout, y, groups, weights: Optional[torch.Tensor] = None):
    """The gradients of combine_rows for dout (rows, features): dy in y's shape and type (zeros where no pair points)
    and dweights (None without weights)."""
    _tensors((dout, "dout"), (y, "y"), (weights if weights is not None else y, "weights"))
    return _ext().combine_grad(dout, y, *_plan(groups), weights)
