"""Products with what follows them: bias, activation and residual, and the gradients.

``fused_matmul`` computes act(x w + bias) + residual in one pass over the
result; ``fused_matmul_backward`` gives the gradients.  The dense layer beside
an expert layer, a router's scores, a projection added to the residual stream.

All calls enqueue their work on the current stream of their tensors' device.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Tuple, Union

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .api import _OZ_DTYPE
from .experts import (_LEVEL, _Plan, _Plans, _check_places, _check_rows, _check_tangents, _copied, _launch, _make_plan,
                      _out_dtype, _readable, _unit)

_PLANS = _Plans()


def _along(w: torch.Tensor) -> torch.Tensor:
    """(K, N) weights with the dimension they are stored along last."""
    return w.t() if w.stride(0) == 1 and w.stride(1) != 1 else w


def _copy_bytes(t: torch.Tensor) -> int:
    """Workspace of the library's copy of a matrix, none where it can be read as it is."""
    return 0 if _readable(t) else (t.shape[0] * ((t.shape[1] + 7) // 8 * 8) * 2 + 255) // 256 * 256


def _check_product(x: torch.Tensor, w: torch.Tensor, activation: Optional[str]) -> None:
    _check_rows(x, "x")
    assert w.dim() == 2, f"w must have 2 dimensions, got shape {tuple(w.shape)}"
    assert w.dtype == x.dtype, f"x/w dtype mismatch: {x.dtype} vs {w.dtype}"
    assert w.shape[0] == x.shape[1], f"contraction dim mismatch: x K={x.shape[1]}, w K={w.shape[0]}"
    assert activation in _lib.ACTIVATIONS, \
        f"unknown activation {activation!r} (one of {', '.join(repr(a) for a in _lib.ACTIVATIONS)})"


def _plan_forward(key, x, w, bias, activation, residual, out_dtype, want_pre) -> _Plan:
    _check_product(x, w, activation)
    out_dtype = _out_dtype(out_dtype, x.dtype)
    rows, k = x.shape
    n = w.shape[1]
    if bias is not None:
        assert bias.dtype in (x.dtype, torch.float32), f"bias must be {x.dtype} or torch.float32, not {bias.dtype}"
        assert bias.shape == (n,), f"bias must have shape {(n,)}, got {tuple(bias.shape)}"
    if residual is not None:
        assert residual.dtype == out_dtype, f"residual must have the result's dtype {out_dtype}, not {residual.dtype}"
        assert residual.shape == (rows, n), f"residual must have shape {(rows, n)}, got {tuple(residual.shape)}"
    device = _check_places(x, w, bias, residual)
    copy = (k > 0 and not (_unit(x) and _unit(_along(w)))) or (bias is not None and not _unit(bias)) \
        or (residual is not None and not _unit(residual))
    args = _lib.LinearArgs(x.data_ptr(), w.data_ptr(), None, None, None, None, None, rows, k, n, x.stride(0), *w.stride(),
                           0 if residual is None else residual.stride(0), 0, _OZ_DTYPE[x.dtype],
                           _OZ_DTYPE[out_dtype], _OZ_DTYPE[x.dtype if bias is None else bias.dtype],
                           _lib.ACTIVATIONS[activation])
    # (negative for what oz_linear will refuse)
    workspace = 0 if copy else max(0, _lib.load().oz_linear_workspace_bytes(ctypes.byref(args)))
    args.workspace_bytes = workspace
    return _PLANS.keep(key, _make_plan("oz_linear", args, (rows, n), out_dtype, device, rows == 0 or n == 0, copy,
                                       workspace))


def _forward(x, w, bias, activation, residual, out_dtype, want_pre):
    """(y, pre or None)."""
    xp, wp = x.data_ptr(), w.data_ptr()
    key = (x.shape, x.stride(), x.dtype, w.shape, w.stride(), w.dtype, x.get_device(), w.get_device(), xp % 16, wp % 16,
           None if bias is None else (bias.shape, bias.stride(), bias.dtype, bias.get_device()), activation,
           None if residual is None else (residual.shape, residual.stride(), residual.dtype, residual.get_device()),
           out_dtype, want_pre)
    plan = _PLANS.kept.get(key) or _plan_forward(key, x, w, bias, activation, residual, out_dtype, want_pre)
    if plan.copy and not plan.empty:
        return _forward(x if _unit(x) else _copied(x), w if _unit(_along(w)) else _copied(w),
                        None if bias is None else bias.contiguous(), activation,
                        residual if residual is None or _unit(residual) else residual.contiguous(), out_dtype, want_pre)
    y = x.new_empty_strided(plan.shape, plan.strides, dtype=plan.dtype)
    pre = x.new_empty_strided(plan.shape, plan.strides) if want_pre else None
    if not plan.empty:
        args = plan.args
        args.x, args.w, args.y = xp, wp, y.data_ptr()
        args.bias = None if bias is None else bias.data_ptr()
        args.residual = None if residual is None else residual.data_ptr()
        args.pre = None if pre is None else pre.data_ptr()
        if plan.workspace:
            workspace = x.new_empty((plan.workspace,), dtype=torch.uint8)
            args.workspace = workspace.data_ptr()
        _launch(plan)
    return y, pre


def _plan_backward(key, dy, x, w, pre, activation, dw_dtype, needs) -> _Plan:
    _check_product(x, w, activation)
    rows, k = x.shape
    n = w.shape[1]
    assert dy.dtype is x.dtype, f"x/dy dtype mismatch: {x.dtype} vs {dy.dtype}"
    assert dy.shape == (rows, n), f"dy must have shape {(rows, n)}, got {tuple(dy.shape)}"
    assert (pre is not None) == (activation is not None), "pre is needed with an activation, and only then"
    if pre is not None:
        assert pre.dtype is x.dtype, f"x/pre dtype mismatch: {x.dtype} vs {pre.dtype}"
        assert pre.shape == (rows, n), f"pre must have shape {(rows, n)}, got {tuple(pre.shape)}"
    dw_dtype = _out_dtype(dw_dtype, x.dtype)
    device = _check_places(x, w, dy, pre)
    copy = not (_unit(dy) and _unit(x) and _unit(_along(w)) and (pre is None or _unit(pre)))
    act, workspace = _lib.ACTIVATIONS[activation], 0
    empty = (rows == 0 or n == 0) and k == 0
    if rows > 0 and n > 0:
        workspace = _lib.load().oz_linear_backward_workspace_bytes(rows, n, act, needs[2])
        if workspace < 0:
            _lib.check(workspace)
        if k > 0 and not copy:
            workspace += (0 if act else _copy_bytes(dy)) + (_copy_bytes(_along(w)) if needs[0] else 0) \
                + (_copy_bytes(x) if needs[1] else 0)
    args = _lib.LinearBackwardArgs(None, None, None, None, None, None, None, None, rows, k, n, dy.stride(0), x.stride(0),
                                   *w.stride(), 0 if pre is None else pre.stride(0), workspace, _OZ_DTYPE[x.dtype],
                                   _OZ_DTYPE[dw_dtype], act, 0)
    return _PLANS.keep(key, _make_plan("oz_linear_backward", args, (rows, k), dw_dtype, device, empty, copy, workspace))


def _backward(dy, x, w, pre, activation, dw_dtype, needs):
    """(dx, dw, db in fp32), None where not needed."""
    dp, xp, wp = dy.data_ptr(), x.data_ptr(), w.data_ptr()
    key = (dy.shape, dy.stride(), dy.dtype, x.shape, x.stride(), x.dtype, w.shape, w.stride(), w.dtype, dy.get_device(),
           x.get_device(), w.get_device(), dp % 16, xp % 16, wp % 16, activation, dw_dtype, needs,
           None if pre is None else (pre.shape, pre.stride(), pre.dtype, pre.get_device()))
    plan = _PLANS.kept.get(key) or _plan_backward(key, dy, x, w, pre, activation, dw_dtype, needs)
    if plan.copy:
        return _backward(dy if _unit(dy) else _copied(dy), x if _unit(x) else _copied(x),
                         w if _unit(_along(w)) else _copied(w), pre if pre is None or _unit(pre) else _copied(pre),
                         activation, dw_dtype, needs)
    dx = x.new_empty_strided(plan.shape, plan.strides) if needs[0] else None
    dw = x.new_empty(w.shape, dtype=plan.dtype) if needs[1] else None
    db = x.new_empty((w.shape[1],), dtype=torch.float32) if needs[2] else None
    if not plan.empty or needs[2]:
        args = plan.args
        args.dy, args.x, args.w = dp, xp, wp
        args.pre = None if pre is None else pre.data_ptr()
        args.dx = None if dx is None else dx.data_ptr()
        args.dw = None if dw is None else dw.data_ptr()
        args.db = None if db is None else db.data_ptr()
        if plan.workspace:
            workspace = x.new_empty((plan.workspace,), dtype=torch.uint8)
            args.workspace = workspace.data_ptr()
        if plan.call is None:
            plan.call = _lib.load().oz_linear_backward
        _launch(plan)
    return dx, dw, db


class _FusedMatmul(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, activation, residual, out_dtype):
        need = any(ctx.needs_input_grad[:3])
        y, pre = _forward(x, w, bias, activation, residual, out_dtype, need and activation is not None)
        if need:
            ctx.save_for_backward(x, w, pre)
        ctx.activation, ctx.bias_dtype = activation, None if bias is None else bias.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        need_x, need_w, need_b, _, need_r, _ = ctx.needs_input_grad
        dx = dw = db = None
        if need_x or need_w or need_b:
            x, w, pre = ctx.saved_tensors
            dx, dw, db = _backward(dy.to(x.dtype), x, w, pre, ctx.activation, None, (need_x, need_w, need_b))
            if db is not None:
                db = db.to(ctx.bias_dtype)
        return dx, dw, db, None, dy if need_r else None, None


def fused_matmul(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                 activation: Optional[str] = None, residual: Optional[torch.Tensor] = None,
                 out_dtype: Optional[torch.dtype] = None, return_pre: bool = False
                 ) -> Union[torch.Tensor, Tuple[torch.Tensor, Optional[torch.Tensor]]]:
    """y = act(x @ w + bias) + residual.

    x (T, K) and w (K, N) of the same dtype (bf16 or fp16), w stored along K or
    along N (other layouts are copied first, and so are rows that do not start on
    16-byte boundaries, unless the product is small); bias (N,) in that dtype or
    fp32; ``activation`` None, "relu", "gelu" (u times the normal distribution's
    function of u) or "silu" (u / (1 + exp(-u))); residual (T, N) in the result's
    dtype.  Returns (T, N) in the operands' dtype, or fp32 with
    ``out_dtype=torch.float32``.  Sums, bias, activation and residual are held in
    fp32 and rounded once.  (For a 16-bit result the tensor cores add the whole
    contraction, cutting off: terms of one sign lose 1e-4 of their sum with 16384
    of them; for an fp32 result 2.5e-6 at any K.)

    Differentiable in x, w, bias and residual (once; second derivatives and
    forward-mode derivatives are refused).  With an activation the forward pass
    then keeps u = x @ w + bias, rounded to the operands' dtype; the gradient of an
    fp32 result is rounded to that dtype before anything else.  With
    ``return_pre`` the result is (y, u), u None without an activation, for
    ``fused_matmul_backward``; no gradient is recorded.
    """
    if _LEVEL._current_level >= 0:
        _check_tangents(x, w, bias, residual)
    if return_pre:
        with torch.no_grad():
            return _forward(x, w, bias, activation, residual, out_dtype, activation is not None)
    if torch.is_grad_enabled() and (x.requires_grad or w.requires_grad or (bias is not None and bias.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        return _FusedMatmul.apply(x, w, bias, activation, residual, out_dtype)
    return _forward(x, w, bias, activation, residual, out_dtype, False)[0]


def fused_matmul_backward(dy: torch.Tensor, x: torch.Tensor, w: torch.Tensor, pre: Optional[torch.Tensor] = None, *,
                          activation: Optional[str] = None, bias: bool = False,
                          dw_dtype: Optional[torch.dtype] = None
                          ) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """Gradients of ``fused_matmul``: du = dy act'(pre), dx = du @ w^T, dw = x^T @ du, dbias = sum of du's rows.

    pre is what ``fused_matmul(..., return_pre=True)`` returned beside y (None
    without an activation); the residual's gradient is dy itself.  Returns (dx, dw,
    dbias): dx (T, K) in the operands' dtype, dw (K, N) in it or, with
    ``dw_dtype=torch.float32``, in fp32, dbias (N,) in fp32, or None unless ``bias``.
    With an activation du is rounded to the operands' dtype before it is
    multiplied; dbias sums it unrounded.  No gradient of the gradients is recorded,
    and forward-mode derivatives are refused.
    """
    if _LEVEL._current_level >= 0:
        _check_tangents(dy, x, w, pre)
    assert dy.dim() == 2 and x.dim() == 2 and w.dim() == 2, "dy, x and w must have 2 dimensions"
    return _backward(dy, x, w, pre, activation, dw_dtype, (True, True, bool(bias)))
