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
from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .api import _OZ_DTYPE
from .experts import _CURRENT_DEVICE, _LEVEL, _OnDevice, _check_places, _check_tangents, _stream_of

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


def _call(name: str, args: ctypes.Structure, device: int) -> None:
    call = getattr(_lib.load(), name)
    if _CURRENT_DEVICE() == device:
        status = call(ctypes.byref(args), _stream_of(device))
    else:
        with _OnDevice(device):
            status = call(ctypes.byref(args), _stream_of(device))
    if status:
        _lib.check(status)


def _check_logits(logits: torch.Tensor, picks: int) -> None:
    assert logits.dim() == 2, f"logits must have 2 dimensions, got shape {tuple(logits.shape)}"
    assert logits.dtype in ROUTE_DTYPES, f"unsupported dtype of logits: {logits.dtype}"
    experts = logits.shape[1]
    assert 1 <= experts <= MAX_EXPERTS, f"there must be 1 to {MAX_EXPERTS} experts, got {experts}"
    assert 1 <= picks <= min(experts, MAX_PICKS), \
        f"picks must be in [1, {min(experts, MAX_PICKS)}], got {picks}"


def _route(logits: torch.Tensor, picks: int, normalize: bool) -> Routing:
    _check_logits(logits, picks)
    device = _check_places(logits)
    rows, experts = logits.shape
    lib = _lib.load()

    def whole(*shape):
        return logits.new_empty(shape, dtype=torch.int32)

    out = Routing(logits.new_empty((rows, picks), dtype=torch.float32), whole(rows, picks), whole(rows, picks),
                  whole(experts + 1), whole(experts), whole(), logits.new_empty((), dtype=torch.float32))
    size = lib.oz_route_workspace_bytes(rows, experts)
    workspace = logits.new_empty((size,), dtype=torch.uint8) if size else None
    args = _lib.RouteArgs(logits.data_ptr(), out.weights.data_ptr(), out.balance_loss.data_ptr(), out.experts.data_ptr(),
                          out.slots.data_ptr(), out.offsets.data_ptr(), out.counts.data_ptr(), out.tokens.data_ptr(),
                          None if workspace is None else workspace.data_ptr(), rows, *logits.stride(), size, experts,
                          picks, bool(normalize), _OZ_DTYPE[logits.dtype])
    _call("oz_route", args, device)
    return out


def _route_gradient(dweights, dloss, logits, weights, experts, counts, tokens, normalize) -> torch.Tensor:
    out = logits.new_empty(logits.shape)
    args = _lib.RouteBackwardArgs(logits.data_ptr(), None if dweights is None else dweights.data_ptr(),
                                  None if dloss is None else dloss.data_ptr(), weights.data_ptr(), experts.data_ptr(),
                                  counts.data_ptr(), tokens.data_ptr(), out.data_ptr(), logits.shape[0],
                                  *logits.stride(), logits.shape[1], experts.shape[1], bool(normalize),
                                  _OZ_DTYPE[logits.dtype])
    _call("oz_route_backward", args, logits.get_device())
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
        dweights = None if dweights is None else dweights.float().contiguous()
        return (_route_gradient(dweights, None if dloss is None else dloss.float(), logits, weights, experts, counts,
                                tokens, ctx.normalize), None, None)


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
    experts = routing.experts
    assert experts.dim() == 2, f"routing.experts must have 2 dimensions, got shape {tuple(experts.shape)}"
    _check_logits(logits, experts.shape[1])
    shape = (logits.shape[0], experts.shape[1])
    for name, t, dtype, want in (("dweights", dweights, torch.float32, shape), ("dloss", dloss, torch.float32, ()),
                                 ("routing.weights", routing.weights, torch.float32, shape),
                                 ("routing.experts", experts, torch.int32, shape),
                                 ("routing.counts", routing.counts, torch.int32, (logits.shape[1],)),
                                 ("routing.tokens", routing.tokens, torch.int32, ())):
        if t is not None:
            assert t.dtype is dtype, f"{name} must be {dtype}, got {t.dtype}"
            assert t.shape == want, f"{name} must have shape {want}, got {tuple(t.shape)}"
    _check_places(logits, dweights, dloss, *routing[:2], routing.counts, routing.tokens)
    return _route_gradient(None if dweights is None else dweights.contiguous(), dloss, logits,
                           routing.weights.contiguous(), experts.contiguous(), routing.counts.contiguous(),
                           routing.tokens, normalize)


# ---------------------------------------------------------------------------
# rows
# ---------------------------------------------------------------------------
def _check_routing(routing: Routing, weights: bool) -> None:
    slots, offsets = routing.slots, routing.offsets
    assert slots.dim() == 2 and slots.dtype is torch.int32, \
        f"routing.slots must be (tokens, picks) int32, got {tuple(slots.shape)} {slots.dtype}"
    assert 1 <= slots.shape[1] <= MAX_PICKS, f"picks must be in [1, {MAX_PICKS}], got {slots.shape[1]}"
    assert offsets.dim() == 1 and offsets.shape[0] >= 2 and offsets.dtype is torch.int32, \
        f"routing.offsets must be (experts + 1,) int32, got {tuple(offsets.shape)} {offsets.dtype}"
    assert slots.is_contiguous() and offsets.is_contiguous(), "routing.slots and offsets must be contiguous"
    if weights:
        w = routing.weights
        assert w.dtype is torch.float32 and w.shape == slots.shape, \
            f"routing.weights must be {tuple(slots.shape)} torch.float32, got {tuple(w.shape)} {w.dtype}"


def _check_matrix(t: torch.Tensor, rows: int, what: str) -> None:
    assert t.dim() == 2, f"{what} must have 2 dimensions, got shape {tuple(t.shape)}"
    assert t.dtype in ROUTE_DTYPES, f"unsupported dtype of {what}: {t.dtype}"
    assert t.shape[0] == rows, f"{what} must have {rows} rows, got {t.shape[0]}"


def _rowwise(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _dispatch(x: torch.Tensor, slots: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    x = _rowwise(x)
    (tokens, d), picks = x.shape, slots.shape[1]
    out = x.new_empty((tokens * picks, d))
    _call("oz_dispatch", _lib.RowsArgs(x.data_ptr(), None, None, out.data_ptr(), slots.data_ptr(), offsets.data_ptr(),
                                       None, None, tokens, d, x.stride(0), 0, offsets.shape[0] - 1, picks,
                                       _OZ_DTYPE[x.dtype], 0), x.get_device())
    return out


def _combine(rows: torch.Tensor, slots: torch.Tensor, weights: Optional[torch.Tensor]) -> torch.Tensor:
    rows = _rowwise(rows)
    (tokens, picks), d = slots.shape, rows.shape[1]
    out = rows.new_empty((tokens, d))
    if weights is not None:
        weights = weights.contiguous()
    _call("oz_combine", _lib.RowsArgs(None, rows.data_ptr(), out.data_ptr(), None, slots.data_ptr(), None,
                                      None if weights is None else weights.data_ptr(), None, tokens, d, 0,
                                      rows.stride(0), 1, picks, _OZ_DTYPE[rows.dtype], 0), rows.get_device())
    return out


def _combine_gradient(dy, rows, slots, offsets, weights):
    dy, rows, weights = _rowwise(dy), _rowwise(rows), weights.contiguous()
    (tokens, picks), d = slots.shape, rows.shape[1]
    drows, dweights = rows.new_empty(rows.shape), weights.new_empty(weights.shape)
    _call("oz_combine_backward", _lib.RowsArgs(dy.data_ptr(), rows.data_ptr(), None, drows.data_ptr(), slots.data_ptr(),
                                               offsets.data_ptr(), weights.data_ptr(), dweights.data_ptr(), tokens, d,
                                               dy.stride(0), rows.stride(0), offsets.shape[0] - 1, picks,
                                               _OZ_DTYPE[rows.dtype], 0), rows.get_device())
    return drows, dweights


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, slots, offsets):
        ctx.save_for_backward(slots)
        return _dispatch(x, slots, offsets)

    @staticmethod
    @once_differentiable
    def backward(ctx, drows):
        return _combine(drows, ctx.saved_tensors[0], None), None, None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, slots, offsets):
        ctx.save_for_backward(rows, weights, slots, offsets)
        return _combine(rows, slots, weights)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        rows, weights, slots, offsets = ctx.saved_tensors
        drows, dweights = _combine_gradient(dy, rows, slots, offsets, weights)
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
    _check_routing(routing, False)
    _check_matrix(x, routing.slots.shape[0], "x")
    _check_places(x, routing.slots, routing.offsets)
    if x.requires_grad and torch.is_grad_enabled():
        return _Dispatch.apply(x, routing.slots, routing.offsets)
    return _dispatch(x, routing.slots, routing.offsets)


def dispatch_backward(drows: torch.Tensor, routing: Routing) -> torch.Tensor:
    """Gradient of ``dispatch``: dx[t] = the sum over j of drows[routing.slots[t, j]]."""
    if _LEVEL._current_level >= 0:
        _check_tangents(drows)
    _check_routing(routing, False)
    _check_matrix(drows, routing.slots.numel(), "drows")
    _check_places(drows, routing.slots)
    return _combine(drows, routing.slots, None)


def combine(rows: torch.Tensor, routing: Routing) -> torch.Tensor:
    """y[t] = the sum over j of routing.weights[t, j] rows[routing.slots[t, j]].

    rows (T k, D) fp32, bf16 or fp16; returns (T, D) in that dtype, summed in fp32
    in the order of j and rounded once, 0 for a token without picks.
    Differentiable in rows and routing.weights (once); forward-mode derivatives are
    refused.
    """
    if _LEVEL._current_level >= 0:
        _check_tangents(rows, routing.weights)
    _check_routing(routing, True)
    _check_matrix(rows, routing.slots.numel(), "rows")
    weights = routing.weights
    _check_places(rows, *routing[:4])
    if (rows.requires_grad or weights.requires_grad) and torch.is_grad_enabled():
        return _Combine.apply(rows, weights, routing.slots, routing.offsets)
    return _combine(rows, routing.slots, weights)


def combine_backward(dy: torch.Tensor, rows: torch.Tensor, routing: Routing) -> Tuple[torch.Tensor, torch.Tensor]:
    """Gradients of ``combine``: (drows, dweights).

    drows[routing.slots[t, j]] = weights[t, j] dy[t] in rows' dtype, 0 after the
    last group; dweights[t, j] = dy[t] . rows[routing.slots[t, j]] in fp32, 0 where there
    is no pick.  dy (T, D) has rows' dtype.
    """
    if _LEVEL._current_level >= 0:
        _check_tangents(dy, rows, routing.weights)
    _check_routing(routing, True)
    _check_matrix(rows, routing.slots.numel(), "rows")
    _check_matrix(dy, routing.slots.shape[0], "dy")
    assert dy.dtype is rows.dtype and dy.shape[1] == rows.shape[1], \
        f"dy must be {(routing.slots.shape[0], rows.shape[1])} {rows.dtype}, got {tuple(dy.shape)} {dy.dtype}"
    _check_places(rows, dy, *routing[:4])
    return _combine_gradient(dy, rows, routing.slots, routing.offsets, routing.weights)
