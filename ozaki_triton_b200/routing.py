"""The router of an expert layer, and the tokens' rows on their way to the experts and back.

``route`` picks each token's experts from its scores and says where each pick's
row lies among the rows sorted by expert; ``dispatch`` puts the tokens' rows
there, in the groups that ``grouped_matmul`` and ``matmul_w4`` take, and
``combine`` adds the experts' results up for each token.

    routing = oz.route(scores, 2)
    rows = oz.dispatch(x, routing)
    rows = oz.grouped_matmul(rows, w, routing.offsets)
    y = oz.combine(rows, routing)

Nothing waits for the routing: all numbers stay on the device.  All calls
enqueue their work on the current stream of their tensors' device.
"""

from __future__ import annotations

import ctypes
import math
from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .api import _OZ_DTYPE
from .experts import _LEVEL, _Plan, _Plans, _check_places, _check_tangents, _launch, _make_plan

ROUTE_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
MAX_EXPERTS, MAX_PICKS = 1024, 32


class Routing(NamedTuple):
    """What ``route`` returns for T tokens, E experts and k picks a token.

    A pick that there is not (of a row of -inf, or of an expert at -inf) has
    weight 0, expert -1 and slot -1 and counts nowhere.  A Routing made by hand
    whose fields contradict each other gives undefined values, never an invalid
    access.
    """

    weights: torch.Tensor        # (T, k) fp32, differentiable
    experts: torch.Tensor        # (T, k) int32
    slots: torch.Tensor          # (T, k) int32, each pick's row
    offsets: torch.Tensor        # (E + 1,) int32, each expert's first row; offsets[E] rows in all
    counts: torch.Tensor         # (E,) int32, each expert's rows
    tokens: torch.Tensor         # () int32, tokens with a pick
    balance_loss: torch.Tensor   # () fp32, differentiable


_PLANS = _Plans()


def _check_logits(logits: torch.Tensor, picks: int) -> None:
    assert logits.dim() == 2, f"logits must have 2 dimensions, got shape {tuple(logits.shape)}"
    assert logits.dtype in ROUTE_DTYPES, f"unsupported dtype of logits: {logits.dtype}"
    experts = logits.shape[1]
    assert 1 <= experts <= MAX_EXPERTS, f"there must be 1 to {MAX_EXPERTS} experts, got {experts}"
    assert 1 <= picks <= min(experts, MAX_PICKS), \
        f"picks must be in [1, {min(experts, MAX_PICKS)}], got {picks}"


def _strides(*shape: int) -> Tuple[int, ...]:
    return tuple(math.prod(max(n, 1) for n in shape[i + 1:]) for i in range(len(shape)))


def _plan_route(key, logits, picks, normalize) -> _Plan:
    _check_logits(logits, picks)
    device = _check_places(logits)
    rows, experts = logits.shape
    size = _lib.load().oz_route_workspace_bytes(rows, experts)
    if size < 0:
        _lib.check(size)
    args = _lib.RouteArgs(None, None, None, None, None, None, None, None, None, rows, *logits.stride(), size, experts,
                          picks, bool(normalize), _OZ_DTYPE[logits.dtype])
    return _PLANS.keep(key, _make_plan("oz_route", args, (rows, picks), logits.dtype, device, False, False, size))


def _route(logits: torch.Tensor, picks: int, normalize: bool) -> Routing:
    key = ("route", logits.shape, logits.stride(), logits.dtype, logits.get_device(), picks, normalize)
    plan = _PLANS.kept.get(key) or _plan_route(key, logits, picks, normalize)
    shape, strides, args, new = plan.shape, plan.strides, plan.args, logits.new_empty_strided
    experts, whole, real = args.experts, torch.int32, torch.float32
    out = Routing(new(shape, strides, dtype=real), new(shape, strides, dtype=whole), new(shape, strides, dtype=whole),
                  new((experts + 1,), (1,), dtype=whole), new((experts,), (1,), dtype=whole), new((), (), dtype=whole),
                  new((), (), dtype=real))
    args.logits, args.weights, args.chosen = logits.data_ptr(), out[0].data_ptr(), out[1].data_ptr()
    args.slots, args.offsets, args.counts = out[2].data_ptr(), out[3].data_ptr(), out[4].data_ptr()
    args.tokens, args.loss = out[5].data_ptr(), out[6].data_ptr()
    if plan.workspace:
        workspace = new((plan.workspace,), (1,), dtype=torch.uint8)
        args.workspace = workspace.data_ptr()
    _launch(plan)
    return out


def _plan_route_gradient(key, dweights, dloss, logits, weights, experts, counts, tokens, normalize) -> _Plan:
    assert experts.dim() == 2, f"routing.experts must have 2 dimensions, got shape {tuple(experts.shape)}"
    _check_logits(logits, experts.shape[1])
    shape = (logits.shape[0], experts.shape[1])
    for name, t, dtype, want in (("dweights", dweights, torch.float32, shape), ("dloss", dloss, torch.float32, ()),
                                 ("routing.weights", weights, torch.float32, shape),
                                 ("routing.experts", experts, torch.int32, shape),
                                 ("routing.counts", counts, torch.int32, (logits.shape[1],)),
                                 ("routing.tokens", tokens, torch.int32, ())):
        if t is not None:
            assert t.dtype is dtype, f"{name} must be {dtype}, got {t.dtype}"
            assert t.shape == want, f"{name} must have shape {want}, got {tuple(t.shape)}"
    device = _check_places(logits, dweights, dloss, weights, experts, counts, tokens)
    args = _lib.RouteBackwardArgs(None, None, None, None, None, None, None, None, logits.shape[0], *logits.stride(),
                                  logits.shape[1], experts.shape[1], bool(normalize), _OZ_DTYPE[logits.dtype])
    copy = not all(t is None or t.is_contiguous() for t in (dweights, weights, experts, counts))
    return _PLANS.keep(key, _make_plan("oz_route_backward", args, tuple(logits.shape), logits.dtype, device,
                                       logits.shape[0] == 0, copy))


def _signature(t: Optional[torch.Tensor]):
    return None if t is None else (t.shape, t.stride(), t.dtype, t.get_device())


def _route_gradient(dweights, dloss, logits, weights, experts, counts, tokens, normalize) -> torch.Tensor:
    key = ("gradient", logits.shape, logits.stride(), logits.dtype, logits.get_device(), normalize, _signature(dweights),
           _signature(dloss), _signature(weights), _signature(experts), _signature(counts), _signature(tokens))
    plan = _PLANS.kept.get(key) or _plan_route_gradient(key, dweights, dloss, logits, weights, experts, counts, tokens,
                                                        normalize)
    if plan.copy:
        return _route_gradient(None if dweights is None else dweights.contiguous(), dloss, logits, weights.contiguous(),
                               experts.contiguous(), counts.contiguous(), tokens, normalize)
    out = logits.new_empty_strided(plan.shape, plan.strides)
    if not plan.empty:
        args = plan.args
        args.logits, args.weights, args.chosen = logits.data_ptr(), weights.data_ptr(), experts.data_ptr()
        args.counts, args.tokens, args.dlogits = counts.data_ptr(), tokens.data_ptr(), out.data_ptr()
        args.dweights = None if dweights is None else dweights.data_ptr()
        args.dloss = None if dloss is None else dloss.data_ptr()
        _launch(plan)
    return out


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, picks, normalize):
        out = _route(logits, picks, normalize)
        ctx.save_for_backward(logits, out.weights, out.experts, out.counts, out.tokens)
        ctx.normalize = normalize
        ctx.mark_non_differentiable(*out[1:6])
        ctx.set_materialize_grads(False)
        return tuple(out)

    @staticmethod
    @once_differentiable
    def backward(ctx, dweights, *rest):
        dloss = rest[-1]
        if dweights is None and dloss is None:
            return None, None, None
        logits, weights, experts, counts, tokens = ctx.saved_tensors
        return (_route_gradient(dweights, dloss, logits, weights, experts, counts, tokens, ctx.normalize), None, None)


def route(logits: torch.Tensor, picks: int, *, normalize: bool = False) -> Routing:
    """Each token's experts, where its rows go, and how evenly the experts are used.

    logits (T, E) fp32, bf16 or fp16, any strides; p = softmax(logits) in fp32.
    A token's picks are the ``picks`` experts with the largest logits, the
    largest first and the lowest index first among equals (a NaN counts as the
    largest); their weights are p, or with ``normalize`` p over the picks' sum.
    Rows are numbered by expert, and by token within one.  An expert at -inf is
    not picked, and a row of -inf throughout (padding) has no picks and takes no
    part in the loss

        balance_loss = E sum_e (counts[e] / sum of counts) (sum_t p[t, e] / tokens)

    (1 where all experts are used alike; 0 without tokens).  Differentiable in
    the weights and the loss (once; forward-mode derivatives are refused).  At most
    1024 experts and 32 picks.
    """
    if _LEVEL._current_level >= 0:
        _check_tangents(logits)
    if logits.requires_grad and torch.is_grad_enabled():
        return Routing(*_Route.apply(logits, picks, normalize))
    return _route(logits, picks, normalize)


def route_backward(dweights: Optional[torch.Tensor], dloss: Optional[torch.Tensor], logits: torch.Tensor,
                   routing: Routing, *, normalize: bool = False) -> torch.Tensor:
    """Gradient of ``route`` in the logits, in their dtype and contiguous.

    dweights (T, k) fp32 and dloss () fp32 are the gradients of the weights and of
    the balance loss, either None for zero; ``normalize`` as in the forward call.
    With dL/dp[e] = dloss E counts[e] / (sum of counts, tokens) plus, without
    ``normalize``, the pick's dweights: dlogits = p (dL/dp - sum p dL/dp); with
    ``normalize`` a pick adds w (dw - sum w dw).
    """
    if _LEVEL._current_level >= 0:
        _check_tangents(dweights, dloss, logits, routing.weights)
    return _route_gradient(dweights, dloss, logits, routing.weights, routing.experts, routing.counts, routing.tokens,
                           normalize)


# ---------------------------------------------------------------------------
# rows
# ---------------------------------------------------------------------------
def _check_routing(slots: torch.Tensor, offsets: torch.Tensor, weights: Optional[torch.Tensor]) -> None:
    assert slots.dim() == 2 and slots.dtype is torch.int32, \
        f"routing.slots must be (tokens, picks) int32, got {tuple(slots.shape)} {slots.dtype}"
    assert 1 <= slots.shape[1] <= MAX_PICKS, f"picks must be in [1, {MAX_PICKS}], got {slots.shape[1]}"
    assert slots.is_contiguous(), "routing.slots must be contiguous"
    assert offsets.dim() == 1 and offsets.shape[0] >= 2 and offsets.dtype is torch.int32, \
        f"routing.offsets must be (experts + 1,) int32, got {tuple(offsets.shape)} {offsets.dtype}"
    assert offsets.is_contiguous(), "routing.offsets must be contiguous"
    if weights is not None:
        assert weights.dtype is torch.float32 and weights.shape == slots.shape, \
            f"routing.weights must be {tuple(slots.shape)} torch.float32, got {tuple(weights.shape)} {weights.dtype}"


def _check_matrix(t: torch.Tensor, rows: int, what: str) -> None:
    assert t.dim() == 2, f"{what} must have 2 dimensions, got shape {tuple(t.shape)}"
    assert t.dtype in ROUTE_DTYPES, f"unsupported dtype of {what}: {t.dtype}"
    assert t.shape[0] == rows, f"{what} must have {rows} rows, got {t.shape[0]}"


def _plan_rows(key, call, x, rows, slots, offsets, weights) -> _Plan:
    """x: of tokens, rows: of picks; the one that a call does not read is None."""
    _check_routing(slots, offsets, weights)
    (tokens, picks), given = slots.shape, x if rows is None else rows
    if rows is not None:
        _check_matrix(rows, tokens * picks, "rows")
    if x is not None:
        _check_matrix(x, tokens, "x" if rows is None else "dy")
        assert x.dtype is given.dtype and x.shape[1] == given.shape[1], \
            f"dy must be {(tokens, given.shape[1])} {given.dtype}, got {tuple(x.shape)} {x.dtype}"
    device = _check_places(given, x, slots, offsets, weights)
    d = given.shape[1]
    shape = (tokens, d) if call == "oz_combine" else (tokens * picks, d)
    # (a tensor without elements has no copy of other strides, and needs none)
    copy = not all(t is None or t.stride(1) == 1 or t.shape[1] == 1 or t.numel() == 0 for t in (x, rows)) \
        or (weights is not None and not weights.is_contiguous())
    args = _lib.RowsArgs(None, None, None, None, None, None, None, None, tokens, d, 0 if x is None else x.stride(0),
                         0 if rows is None else rows.stride(0), offsets.shape[0] - 1, picks,
                         _OZ_DTYPE[given.dtype], 0)
    return _PLANS.keep(key, _make_plan(call, args, shape, given.dtype, device, tokens == 0, copy))


def _rows(call, x, rows, slots, offsets, weights):
    """The result of a call in rows or tokens; of ``oz_combine_backward`` (drows, dweights)."""
    key = (call, _signature(x), _signature(rows), _signature(slots), _signature(offsets), _signature(weights))
    plan = _PLANS.kept.get(key) or _plan_rows(key, call, x, rows, slots, offsets, weights)
    if plan.copy:
        return _rows(call, None if x is None else x.contiguous(), None if rows is None else rows.contiguous(), slots,
                     offsets, None if weights is None else weights.contiguous())
    given = x if rows is None else rows
    out = given.new_empty_strided(plan.shape, plan.strides)
    gradient = call == "oz_combine_backward"
    dweights = slots.new_empty(slots.shape, dtype=torch.float32) if gradient else None
    if not plan.empty:
        args = plan.args
        args.x = None if x is None else x.data_ptr()
        args.rows = None if rows is None else rows.data_ptr()
        args.slots = slots.data_ptr()
        args.offsets = offsets.data_ptr()
        args.weights = None if weights is None else weights.data_ptr()
        if call == "oz_combine":
            args.x_out = out.data_ptr()
        else:
            args.rows_out = out.data_ptr()
        if gradient:
            args.dweights = dweights.data_ptr()
        _launch(plan)
    return (out, dweights) if gradient else out


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, slots, offsets):
        ctx.save_for_backward(slots, offsets)
        return _rows("oz_dispatch", x, None, slots, offsets, None)

    @staticmethod
    @once_differentiable
    def backward(ctx, drows):
        return _rows("oz_combine", None, drows, *ctx.saved_tensors, None), None, None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, slots, offsets):
        ctx.save_for_backward(rows, weights, slots, offsets)
        return _rows("oz_combine", None, rows, slots, offsets, weights)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        rows, weights, slots, offsets = ctx.saved_tensors
        drows, dweights = _rows("oz_combine_backward", dy, rows, slots, offsets, weights)
        return (drows if ctx.needs_input_grad[0] else None, dweights if ctx.needs_input_grad[1] else None, None, None)


def dispatch(x: torch.Tensor, routing: Routing) -> torch.Tensor:
    """Each token's row once for each of its picks, in the order of the experts.

    x (T, D) fp32, bf16 or fp16.  Returns (T k, D) rows with
    rows[routing.slots[t, j]] = x[t], the groups of ``routing.offsets``; rows after
    the last group are 0.  Differentiable in x (once): a token's gradients are
    added in fp32 and rounded once.  Forward-mode derivatives are refused.
    """
    if _LEVEL._current_level >= 0:
        _check_tangents(x)
    if x.requires_grad and torch.is_grad_enabled():
        return _Dispatch.apply(x, routing.slots, routing.offsets)
    return _rows("oz_dispatch", x, None, routing.slots, routing.offsets, None)


def dispatch_backward(drows: torch.Tensor, routing: Routing) -> torch.Tensor:
    """Gradient of ``dispatch``: dx[t] = the sum over j of drows[routing.slots[t, j]]."""
    if _LEVEL._current_level >= 0:
        _check_tangents(drows)
    return _rows("oz_combine", None, drows, routing.slots, routing.offsets, None)


def combine(rows: torch.Tensor, routing: Routing) -> torch.Tensor:
    """y[t] = the sum over j of routing.weights[t, j] rows[routing.slots[t, j]].

    rows (T k, D) fp32, bf16 or fp16; returns (T, D) in that dtype, summed in fp32
    in the order of j and rounded once, 0 for a token without picks.
    Differentiable in rows and routing.weights (once); forward-mode derivatives are
    refused.
    """
    if _LEVEL._current_level >= 0:
        _check_tangents(rows, routing.weights)
    weights = routing.weights
    if (rows.requires_grad or weights.requires_grad) and torch.is_grad_enabled():
        return _Combine.apply(rows, weights, routing.slots, routing.offsets)
    return _rows("oz_combine", None, rows, routing.slots, routing.offsets, weights)


def combine_backward(dy: torch.Tensor, rows: torch.Tensor, routing: Routing) -> Tuple[torch.Tensor, torch.Tensor]:
    """Gradients of ``combine``: (drows, dweights).

    drows[routing.slots[t, j]] = weights[t, j] dy[t] in rows' dtype, 0 after the
    last group; dweights[t, j] = dy[t] . rows[routing.slots[t, j]] in fp32, 0 where there
    is no pick.  dy (T, D) has rows' dtype.
    """
    if _LEVEL._current_level >= 0:
        _check_tangents(dy, rows, routing.weights)
    return _rows("oz_combine_backward", dy, rows, routing.slots, routing.offsets, routing.weights)
