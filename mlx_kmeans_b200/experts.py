"""Routed experts on libkmc.so: rows go to their k best experts and get a weighted sum of the experts' products.

The reference (kakollu/mlx-kmeans) answers with the one nearest center of a row; these operators carry fitted
centers (or any gate's scores) on to a mixture of experts:

    ids, weights = route(logits, top_k)            # the k best experts of every row, and their weights
    groups = group_rows(ids, n_experts)            # the (row, choice) pairs grouped by expert
    y = expert_matmul(x, w, groups)                # each group times its expert's matrix
    out = combine_rows(y, groups, weights)         # a row's results summed with its weights

All arguments are CUDA tensors; work is enqueued on the current stream and nothing synchronises.  route,
expert_matmul and combine_rows are differentiable through torch.autograd; route_grad, expert_matmul_grad and
combine_rows_grad are the same gradients as plain calls.  group_rows takes labels too (KMeans.labels_ on the device),
to run one product per cluster.  Errors: ValueError for bad arguments, RuntimeError for a device failure.
"""
from typing import NamedTuple, Optional

import torch

from . import _lib
from .core import _ptr

_DTYPES = {torch.float32: _lib.KMC_F32, torch.bfloat16: _lib.KMC_BF16, torch.float16: _lib.KMC_F16}
_SCORES = {"softmax": 0, "sigmoid": _lib.KMC_ROUTE_SIGMOID}
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_fns = {}                           # entry points of libkmc.so, looked up once
_errors = {}                        # per device: the int32 a kernel sets when it gave up on a barrier


class RowGroups(NamedTuple):
    """The grouping of (row, choice) pairs by expert (group_rows), int32 CUDA tensors.

    offsets (n_experts + 1): expert e has the positions offsets[e] .. offsets[e + 1] - 1.
    rows (pairs): the row each position reads, -1 past offsets[-1].
    slot (rows, choices) or (rows,): the position of each pair, -1 for a pair that was left out.
    """
    offsets: torch.Tensor
    rows: torch.Tensor
    slot: torch.Tensor


def _check(t, name, ndim=None, dtypes=None, device=None):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if ndim is not None and t.ndim != ndim:
        raise ValueError(f"{name} must be {ndim}-D, got {t.ndim}-D")
    if dtypes is not None and t.dtype not in dtypes:
        raise ValueError(f"{name} must be {' or '.join(str(d)[6:] for d in dtypes)}, got {str(t.dtype)[6:]}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")
    return t


def _run(name, device, *args):
    """kmc_<name>(*args, stream) on the device's current stream, the device made current for the call if it is not."""
    fn = _fns.get(name)
    if fn is None:
        fn = _fns[name] = getattr(_lib.load(), name)
    if device.index == torch.cuda.current_device():
        status = fn(*args, _raw_stream(device.index))
    else:
        with torch.cuda.device(device):
            status = fn(*args, _raw_stream(device.index))
    if status:
        _lib.check(status, name)


def _rows_of(t):
    """t (2-D) with unit stride along its rows, copied if it has none; rows may lie any distance apart."""
    return t if (t.stride(1) == 1 or t.shape[1] == 1) and t.stride(0) >= t.shape[1] else t.contiguous()


def _error_word(device):
    e = _errors.get(device)
    if e is None:
        e = _errors[device] = torch.zeros(1, dtype=torch.int32, device=device)
        torch.cuda.current_stream(device).synchronize()      # zero before any stream's kernel can set it
    return e.data_ptr()


def expert_status(device=None):
    """Raise RuntimeError if an expert_matmul (or its gradient) on `device` gave up waiting on a barrier since the last
    call, which leaves its result incomplete.  Waits for the device's current stream."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    e = _errors.get(device)
    if e is not None and int(e.item()) != 0:
        e.zero_()
        raise RuntimeError("expert_matmul: a kernel gave up waiting on a barrier; its result is incomplete")


# ---------------------------------------------------------------- routing

def _route_flags(score, renormalize):
    if score not in _SCORES:
        raise ValueError(f"score must be 'softmax' or 'sigmoid', got {score!r}")
    return _SCORES[score] | (_lib.KMC_ROUTE_RENORM if renormalize else 0)


def _route(logits, top_k, flags, bias, groups, top_groups, scale, mask):
    T, E = logits.shape
    ids = torch.empty((T, top_k), dtype=torch.int32, device=logits.device)
    weights = torch.empty((T, top_k), dtype=torch.float32, device=logits.device)
    _run("kmc_route", logits.device, logits.data_ptr(), _DTYPES[logits.dtype], T, E, max(logits.stride(0), E), _ptr(bias),
         _ptr(mask), top_k, groups, top_groups, scale, flags, ids.data_ptr(), weights.data_ptr())
    return ids, weights


def _route_grad(dweights, logits, ids, flags, scale):
    T, E = logits.shape
    dlogits = torch.empty((T, E), dtype=logits.dtype, device=logits.device)
    _run("kmc_route_grad", logits.device, dweights.data_ptr(), logits.data_ptr(), _DTYPES[logits.dtype], T, E,
         max(logits.stride(0), E), ids.data_ptr(), ids.shape[1], scale, flags, dlogits.data_ptr())
    return dlogits


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, top_k, flags, bias, groups, top_groups, scale, mask):
        ids, weights = _route(logits, top_k, flags, bias, groups, top_groups, scale, mask)
        ctx.save_for_backward(logits, ids)
        ctx.flags, ctx.scale = flags, scale
        ctx.mark_non_differentiable(ids)
        return ids, weights

    @staticmethod
    def backward(ctx, _dids, dweights):
        logits, ids = ctx.saved_tensors
        dl = _route_grad(dweights.float().contiguous(), logits, ids, ctx.flags, ctx.scale)
        return dl, None, None, None, None, None, None, None


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
    _check(logits, "logits", 2, _DTYPES)
    flags = _route_flags(score, renormalize)
    if bias is not None:
        _check(bias, "bias", 1, (torch.float32,), logits.device)
        if bias.shape[0] != logits.shape[1]:
            raise ValueError(f"bias has {bias.shape[0]} values for {logits.shape[1]} experts")
        bias = bias.detach().contiguous()
    if mask is not None:
        _check(mask, "mask", 1, (torch.bool,), logits.device)
        if mask.shape[0] != logits.shape[0]:
            raise ValueError(f"mask has {mask.shape[0]} values for {logits.shape[0]} rows")
        mask = mask.contiguous()
    logits = _rows_of(logits)
    args = (logits, int(top_k), flags, bias, int(groups), int(top_groups), float(scale), mask)
    if logits.requires_grad and torch.is_grad_enabled():
        return _Route.apply(*args)
    return _route(*args)


def route_grad(dweights, logits, ids, *, score="softmax", renormalize=True, scale=1.0):
    """The gradient of route's weights with respect to the logits: dlogits (rows, n_experts) in the logits' type, from
    dweights (rows, top_k) and the ids that route gave for these logits, score, renormalize and scale."""
    _check(logits, "logits", 2, _DTYPES)
    _check(ids, "ids", 2, (torch.int32,), logits.device)
    _check(dweights, "dweights", 2, (torch.float32,), logits.device)
    if ids.shape != dweights.shape or ids.shape[0] != logits.shape[0]:
        raise ValueError(f"dweights {tuple(dweights.shape)}, ids {tuple(ids.shape)} and logits {tuple(logits.shape)} "
                         f"do not belong together")
    return _route_grad(dweights.contiguous(), _rows_of(logits), ids.contiguous(), _route_flags(score, renormalize),
                       float(scale))


# ---------------------------------------------------------------- grouping

def group_rows(ids, n_experts):
    """Group (row, choice) pairs by expert: RowGroups of ids (rows, choices) or (rows,) int32, up to 4096 experts.

    Stable: an expert's pairs keep their order.  ids outside [0, n_experts) are left out (slot -1)."""
    _check(ids, "ids", None, (torch.int32,))
    if ids.ndim not in (1, 2):
        raise ValueError(f"ids must be 1-D or 2-D, got {ids.ndim}-D")
    ids = ids.contiguous()
    T, k = ids.shape[0], (ids.shape[1] if ids.ndim == 2 else 1)
    dev, E = ids.device, int(n_experts)
    nb = int(_lib.load().kmc_group_bytes(T * k, E))
    ws = torch.empty(nb, dtype=torch.uint8, device=dev) if nb else None
    offsets = torch.empty(max(E, 0) + 1, dtype=torch.int32, device=dev)
    rows = torch.empty(T * k, dtype=torch.int32, device=dev)
    slot = torch.empty(ids.shape, dtype=torch.int32, device=dev)
    _run("kmc_group_rows", dev, ids.data_ptr(), T, k, E, offsets.data_ptr(), rows.data_ptr(), slot.data_ptr(),
         _ptr(ws), nb)
    return RowGroups(offsets, rows, slot)


def _check_groups(groups, device):
    offsets, rows, slot = groups
    _check(offsets, "groups.offsets", 1, (torch.int32,), device)
    _check(rows, "groups.rows", 1, (torch.int32,), device)
    _check(slot, "groups.slot", None, (torch.int32,), device)
    if not (offsets.is_contiguous() and rows.is_contiguous() and slot.is_contiguous()):
        raise ValueError("groups must hold contiguous tensors (as group_rows gives them)")
    if slot.ndim not in (1, 2) or slot.numel() != rows.numel() or offsets.numel() < 2:
        raise ValueError(f"groups of {offsets.numel() - 1} experts, {rows.numel()} positions and slots of shape "
                         f"{tuple(slot.shape)} do not belong together")
    return slot.shape[0], (slot.shape[1] if slot.ndim == 2 else 1)


# ---------------------------------------------------------------- products per expert

_HALF = (torch.bfloat16, torch.float16)


def _check_expert(x, w, groups, gather):
    _check(w, "w", 3, _HALF)
    _check(x, "x", 2, (w.dtype,), w.device)
    T, k = _check_groups(groups, w.device)
    if groups.offsets.numel() - 1 != w.shape[0]:
        raise ValueError(f"w has {w.shape[0]} matrices for {groups.offsets.numel() - 1} experts")
    if x.shape[1] != w.shape[2]:
        raise ValueError(f"x has {x.shape[1]} columns, the matrices {w.shape[2]}")
    want = T if gather else T * k
    if x.shape[0] != want:
        raise ValueError(f"x has {x.shape[0]} rows, the groups want {want} ({'rows' if gather else 'positions'})")
    return T, k


def _workspace(x, rows, w, dy, P, E, N, D, device):
    """The workspace of an expert product: for x in grouped order, and for padded copies of unaligned operands."""
    x_rows, ldx = (x.shape[0], max(x.stride(0), D)) if x is not None else (0, D)
    nb = _lib.load().kmc_expert_bytes(_ptr(x), x_rows, ldx, _ptr(rows), _ptr(w), _ptr(dy), P, E, N, D)
    return (torch.empty(nb, dtype=torch.uint8, device=device) if nb else None), nb


def _expert(x, w, groups, gather):
    (E, N, D), P, dev = w.shape, groups.rows.numel(), w.device
    y = torch.empty((P, N), dtype=w.dtype, device=dev)
    rows = groups.rows if gather else None
    ws, nb = _workspace(x, rows, w, None, P, E, N, D, dev)
    _run("kmc_expert_matmul", dev, x.data_ptr(), x.shape[0], max(x.stride(0), D),
         _ptr(rows), w.data_ptr(), groups.offsets.data_ptr(), P, E, N, D,
         _DTYPES[w.dtype], y.data_ptr(), _ptr(ws), nb, _error_word(dev))
    return y


def _expert_dx(dy, w, groups, gather):
    (E, N, D), P, dev = w.shape, groups.rows.numel(), w.device
    dx = torch.empty((P, D), dtype=w.dtype, device=dev)
    ws, nb = _workspace(None, None, w, dy, P, E, N, D, dev)
    _run("kmc_expert_matmul_dx", dev, dy.data_ptr(), w.data_ptr(), groups.offsets.data_ptr(), P, E, N, D,
         _DTYPES[w.dtype], dx.data_ptr(), _ptr(ws), nb, _error_word(dev))
    # a row with several choices: the float32 sum of its positions' gradients, which are in w's type by now (each
    # rounded once; the error of the sum stays within that of one more rounding of its result)
    return _combine(dx, groups, None) if gather else dx


def _expert_dw(dy, x, groups, E, gather):
    (N, D), P, dev = (dy.shape[1], x.shape[1]), groups.rows.numel(), dy.device
    dw = torch.empty((E, N, D), dtype=x.dtype, device=dev)
    rows = groups.rows if gather else None
    ws, nb = _workspace(x, rows, None, dy, P, E, N, D, dev)
    _run("kmc_expert_matmul_dw", dev, dy.data_ptr(), x.data_ptr(), x.shape[0], max(x.stride(0), D),
         _ptr(rows), groups.offsets.data_ptr(), P, E, N, D,
         _DTYPES[x.dtype], dw.data_ptr(), _ptr(ws), nb, _error_word(dev))
    return dw


class _ExpertMatmul(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, offsets, rows, slot, gather):
        ctx.save_for_backward(x, w, offsets, rows, slot)
        ctx.gather = gather
        return _expert(x, w, RowGroups(offsets, rows, slot), gather)

    @staticmethod
    def backward(ctx, dy):
        x, w, offsets, rows, slot = ctx.saved_tensors
        groups, dy = RowGroups(offsets, rows, slot), dy.contiguous()
        dx = _expert_dx(dy, w, groups, ctx.gather) if ctx.needs_input_grad[0] else None
        dw = _expert_dw(dy, x, groups, w.shape[0], ctx.gather) if ctx.needs_input_grad[1] else None
        return dx, dw, None, None, None, None


def expert_matmul(x, w, groups, *, gather=True):
    """Each position's row times its expert's matrix: y (positions, n) with y[p] = w[e] @ x[row of p].

    x: (rows, d) and every position reads its row (gather=True), or (positions, d) already grouped (gather=False).
    w: (n_experts, n, d), bfloat16 or float16 as x; sums are float32.  Positions past groups.offsets[-1] are zero."""
    _check_expert(x, w, groups, gather)
    x, w = _rows_of(x), w.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or w.requires_grad):
        return _ExpertMatmul.apply(x, w, *groups, bool(gather))
    return _expert(x, w, groups, gather)


def expert_matmul_grad(dy, x, w, groups, *, gather=True):
    """The gradients of expert_matmul for dy (positions, n): dx in x's shape (with gather=True a row's positions are
    summed) and dw in w's; an expert with no position gets a dw of zeros."""
    _check_expert(x, w, groups, gather)
    _check(dy, "dy", 2, (w.dtype,), w.device)
    if tuple(dy.shape) != (groups.rows.numel(), w.shape[1]):
        raise ValueError(f"dy is {tuple(dy.shape)}, the products {(groups.rows.numel(), w.shape[1])}")
    x, w, dy = _rows_of(x), w.contiguous(), dy.contiguous()
    return _expert_dx(dy, w, groups, gather), _expert_dw(dy, x, groups, w.shape[0], gather)


# ---------------------------------------------------------------- combination

def _check_combine(y, groups, weights):
    _check(y, "y", 2, _DTYPES)
    T, k = _check_groups(groups, y.device)
    if y.shape[0] != T * k:
        raise ValueError(f"y has {y.shape[0]} rows for {T * k} positions")
    if weights is not None:
        _check(weights, "weights", None, (torch.float32,), y.device)
        if weights.shape != groups.slot.shape:
            raise ValueError(f"weights are {tuple(weights.shape)}, the groups' pairs {tuple(groups.slot.shape)}")
    return T, k


def _combine(y, groups, weights):
    slot = groups.slot
    T, k = slot.shape[0], (slot.shape[1] if slot.ndim == 2 else 1)
    out = torch.empty((T, y.shape[1]), dtype=y.dtype, device=y.device)
    _run("kmc_combine", y.device, y.data_ptr(), _DTYPES[y.dtype], T, k, y.shape[1], slot.data_ptr(), _ptr(weights),
         out.data_ptr())
    return out


def _combine_grad(dout, y, groups, weights):
    slot = groups.slot
    T, k = slot.shape[0], (slot.shape[1] if slot.ndim == 2 else 1)
    dy = torch.empty_like(y)
    dw = torch.empty_like(weights) if weights is not None else None
    _run("kmc_combine_grad", y.device, dout.data_ptr(), y.data_ptr(), _DTYPES[y.dtype], T, k, y.shape[1],
         slot.data_ptr(), _ptr(weights), groups.offsets.data_ptr() + 4 * (groups.offsets.numel() - 1), dy.data_ptr(), _ptr(dw))
    return dy, dw


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, offsets, rows, slot):
        ctx.save_for_backward(y, weights, offsets, rows, slot)
        return _combine(y, RowGroups(offsets, rows, slot), weights)

    @staticmethod
    def backward(ctx, dout):
        y, weights, offsets, rows, slot = ctx.saved_tensors
        dy, dw = _combine_grad(dout.contiguous(), y, RowGroups(offsets, rows, slot), weights)
        return dy, dw, None, None, None


def combine_rows(y, groups, weights: Optional[torch.Tensor] = None):
    """A row's results summed: out (rows, features) with out[t] = sum over its choices of weight * y[slot].

    y: (positions, features), float32, bfloat16 or float16; weights float32 in the shape of the ids, or None for 1.
    The sum is float32, rounded once; a pair that was left out adds nothing."""
    _check_combine(y, groups, weights)
    y = y.contiguous()
    weights = weights.contiguous() if weights is not None else None
    if torch.is_grad_enabled() and (y.requires_grad or (weights is not None and weights.requires_grad)):
        return _Combine.apply(y, weights, *groups)
    return _combine(y, groups, weights)


def combine_rows_grad(dout, y, groups, weights: Optional[torch.Tensor] = None):
    """The gradients of combine_rows for dout (rows, features): dy in y's shape and type (zeros where no pair points)
    and dweights (None without weights)."""
    T, _ = _check_combine(y, groups, weights)
    _check(dout, "dout", 2, (y.dtype,), y.device)
    if tuple(dout.shape) != (T, y.shape[1]):
        raise ValueError(f"dout is {tuple(dout.shape)}, the result {(T, y.shape[1])}")
    return _combine_grad(dout.contiguous(), y.contiguous(), groups, weights.contiguous() if weights is not None else None)
