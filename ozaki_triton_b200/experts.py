"""Products of an expert layer: ragged groups of rows, each with its own weights.

``grouped_matmul`` multiplies each group of rows of ``x`` by the weights of
its expert and ``grouped_matmul_backward`` gives the gradients;
``matmul_w4`` multiplies a few rows by 4-bit weights with group scales (one
matrix, or one per expert), laid out by ``quantize_w4``.

The groups are runs of rows: ``offsets`` (experts + 1 device integers) says
that rows ``offsets[e] .. offsets[e + 1] - 1`` belong to expert ``e``.  It is
read on the device only, so a call never waits for the routing that produced
it.  Offsets are clamped to ``[0, rows]``; a group may be empty, and a row
that no group holds has a zero result and adds nothing to any gradient.
Offsets that decrease give undefined values, never an invalid access.

All calls enqueue their work on the current stream of their tensors' device.
"""

from __future__ import annotations

import ctypes
import math
import threading
import types
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib
from .api import _OZ_DTYPE, _RAW_STREAM, _check_cuda

# operand types: products are exact in fp32, sums are held in fp32
GROUPED_DTYPES = (torch.bfloat16, torch.float16)

_OFFSET_DTYPES = (torch.int32, torch.int64)
_SCALE_DTYPES = (torch.float16, torch.bfloat16, torch.float32)


def _check_places(x: torch.Tensor, *ts: Optional[torch.Tensor]) -> int:
    """The index of the device that holds every tensor."""
    _check_cuda(x)
    index = x.get_device()
    for t in ts:
        if t is not None and (not t.is_cuda or t.get_device() != index):
            raise ValueError(f"tensors on different devices: {x.device} and {t.device}")
    return index


# inside a forward-mode level >= 0 (where torch does not say, tensors are always looked at)
_LEVEL = forward_ad if hasattr(forward_ad, "_current_level") else types.SimpleNamespace(_current_level=0)


def _check_tangents(*ts: Optional[torch.Tensor]) -> None:
    """Refuses tensors that carry a forward-mode derivative: it would be lost, since the
    library reads their values only."""
    for t in ts:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError("no forward-mode derivative of this operator: an argument has a tangent")


class _OnDevice:
    """Makes a device current for a call."""

    __slots__ = ("index", "other")

    def __init__(self, index: int):
        self.index = index

    def __enter__(self):
        self.other = torch.cuda.current_device()
        if self.other != self.index:
            torch.cuda.set_device(self.index)

    def __exit__(self, *_):
        if self.other != self.index:
            torch.cuda.set_device(self.other)


def _stream_of(device: int) -> int:
    return _RAW_STREAM(device) if _RAW_STREAM is not None else torch.cuda.current_stream(device).cuda_stream


def _check_offsets(offsets: torch.Tensor, groups: int) -> None:
    assert offsets.dtype in _OFFSET_DTYPES, f"offsets must be int32 or int64, got {offsets.dtype}"
    assert offsets.dim() == 1 and offsets.shape[0] == groups + 1, \
        f"offsets must have {groups + 1} entries, got shape {tuple(offsets.shape)}"
    assert offsets.is_contiguous(), "offsets must be contiguous"


def _check_rows(x: torch.Tensor, what: str) -> None:
    assert x.dim() == 2, f"{what} must have 2 dimensions, got shape {tuple(x.shape)}"
    assert x.dtype in GROUPED_DTYPES, f"unsupported dtype of {what}: {x.dtype}"


def _out_dtype(dtype: Optional[torch.dtype], operand: torch.dtype) -> torch.dtype:
    if dtype is None:
        return operand
    assert dtype is operand or dtype is torch.float32, \
        f"results are {operand} or torch.float32, not {dtype}"
    return dtype


def _copied(t: torch.Tensor) -> torch.Tensor:
    """A copy of t whose rows start on 16-byte boundaries."""
    inner = t.shape[-1]
    laid = torch.empty((*t.shape[:-1], (inner + 7) // 8 * 8), dtype=t.dtype, device=t.device)
    return laid[..., :inner].copy_(t)


def _readable(t: torch.Tensor) -> bool:
    """Whether the copy unit can read t's layout: it wants a unit stride along the
    last dimension, 16-byte boundaries and no repeated rows."""
    shape, strides = t.shape, t.stride()
    if (strides[-1] != 1 and shape[-1] != 1) or t.data_ptr() % 16:
        return False
    return all(n <= 1 or (s > 0 and s % 8 == 0) for n, s in zip(shape[:-1], strides))


def _as_operand(t: torch.Tensor) -> torch.Tensor:
    return t if _readable(t) else _copied(t)


def _along(w: torch.Tensor) -> torch.Tensor:
    """(E, K, N) weights with the dimension they are stored along last."""
    return w.transpose(1, 2) if w.stride(1) == 1 and w.stride(2) != 1 else w


def _unit(t: torch.Tensor) -> bool:
    return t.stride(-1) == 1 or t.shape[-1] == 1


def _copy_bytes(t: torch.Tensor) -> int:
    """Workspace of the library's copy of t, none where it can be read as it is."""
    if _readable(t):
        return 0
    return (t[..., 0].numel() * ((t.shape[-1] + 7) // 8 * 8) * 2 + 255) // 256 * 256


def _check_grouped(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor) -> None:
    _check_rows(x, "x")
    assert w.dim() == 3, f"w must have 3 dimensions, got shape {tuple(w.shape)}"
    assert w.dtype == x.dtype, f"x/w dtype mismatch: {x.dtype} vs {w.dtype}"
    assert w.shape[0] >= 1, "w must hold at least one expert"
    assert w.shape[1] == x.shape[1], f"contraction dim mismatch: x K={x.shape[1]}, w K={w.shape[1]}"
    _check_offsets(offsets, w.shape[0])


class _Plan:
    """What a call derives from its tensors' types, shapes, strides and devices
    alone: the checks passed, the library's arguments but for the addresses,
    and the result's shape.  Kept per distinct call signature and thread, so
    that a repeated small product pays for its allocation and one library
    call (checking and converting everything again took 5 us of 13)."""

    __slots__ = ("args", "ref", "call", "shape", "strides", "dtype", "empty", "copy", "device", "workspace")


class _Plans(threading.local):
    def __init__(self):
        self.kept = {}

    def keep(self, key, plan: _Plan) -> _Plan:
        if len(self.kept) >= 256:
            self.kept.clear()
        self.kept[key] = plan
        return plan


_PLANS = _Plans()
_CURRENT_DEVICE = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _launch(plan: _Plan) -> None:
    """The plan's library call on the current stream of its device."""
    device = plan.device
    if _CURRENT_DEVICE() == device:
        status = plan.call(plan.ref, _stream_of(device))
    else:
        with _OnDevice(device):
            status = plan.call(plan.ref, _stream_of(device))
    if status:
        _lib.check(status)


def _make_plan(call: str, args: ctypes.Structure, shape: Tuple[int, ...], dtype: torch.dtype, device: int,
               empty: bool, copy: bool, workspace: int = 0) -> _Plan:
    plan = _Plan()
    plan.args, plan.ref = args, ctypes.byref(args)
    plan.call = getattr(_lib.load(), call) if not empty else None
    plan.shape, plan.dtype, plan.device, plan.empty, plan.copy = shape, dtype, device, empty, copy
    plan.workspace = workspace
    # a result allocated by shape and strides costs 0.2 us less than by shape alone
    plan.strides = tuple(math.prod(max(n, 1) for n in shape[i + 1:]) for i in range(len(shape)))
    return plan


def _plan_product(key, x, w, offsets, out_dtype) -> _Plan:
    _check_grouped(x, w, offsets)
    out_dtype = _out_dtype(out_dtype, x.dtype)
    device = _check_places(x, w, offsets)
    rows, k = x.shape
    groups, _, n = w.shape
    copy, workspace = k > 0 and not (_unit(x) and _unit(_along(w))), 0
    if k > 0 and rows > 0 and n > 0 and not copy:
        workspace = _copy_bytes(x) + _copy_bytes(_along(w))
    args = _lib.GroupedArgs(None, None, None, None, rows, k, n, x.stride(0), *w.stride(), n, None, workspace,
                            groups, offsets.dtype is torch.int64, _OZ_DTYPE[x.dtype], _OZ_DTYPE[out_dtype])
    return _PLANS.keep(key, _make_plan("oz_grouped_matmul", args, (rows, n), out_dtype, device,
                                       rows == 0 or n == 0, copy, workspace))


def _product(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor,
             out_dtype: Optional[torch.dtype]) -> torch.Tensor:
    # the addresses' alignment is part of the signature: it decides what is copied
    xp, wp = x.data_ptr(), w.data_ptr()
    key = (x.shape, x.stride(), x.dtype, w.shape, w.stride(), w.dtype, offsets.shape, offsets.stride(),
           offsets.dtype, out_dtype, x.get_device(), w.get_device(), offsets.get_device(), xp % 16, wp % 16)
    plan = _PLANS.kept.get(key) or _plan_product(key, x, w, offsets, out_dtype)
    if plan.copy:
        return _product(x if _unit(x) else _copied(x), w if _unit(_along(w)) else _copied(w), offsets, out_dtype)
    y = x.new_empty_strided(plan.shape, plan.strides, dtype=plan.dtype)
    if not plan.empty:
        args = plan.args
        args.x, args.w, args.offsets, args.y = xp, wp, offsets.data_ptr(), y.data_ptr()
        if plan.workspace:
            workspace = x.new_empty((plan.workspace,), dtype=torch.uint8)
            args.workspace = workspace.data_ptr()
        _launch(plan)
    return y


def _plan_weight_gradient(key, x, dy, offsets, groups, out_dtype) -> _Plan:
    out_dtype = _out_dtype(out_dtype, x.dtype)
    device = _check_places(x, dy, offsets)
    rows, k = x.shape
    n = dy.shape[1]
    copy, workspace = rows > 0 and not (_unit(x) and _unit(dy)), 0
    if rows > 0 and k > 0 and n > 0 and not copy:
        workspace = _copy_bytes(x) + _copy_bytes(dy)
    args = _lib.GroupedWgradArgs(None, None, None, None, rows, k, n, x.stride(0), dy.stride(0), None, workspace,
                                 groups, offsets.dtype is torch.int64, _OZ_DTYPE[x.dtype], _OZ_DTYPE[out_dtype])
    return _PLANS.keep(key, _make_plan("oz_grouped_wgrad", args, (groups, k, n), out_dtype, device,
                                       k == 0 or n == 0, copy, workspace))


def _weight_gradient(x: torch.Tensor, dy: torch.Tensor, offsets: torch.Tensor, groups: int,
                     out_dtype: Optional[torch.dtype]) -> torch.Tensor:
    xp, dp = x.data_ptr(), dy.data_ptr()
    key = (groups, x.shape, x.stride(), x.dtype, dy.shape, dy.stride(), offsets.dtype, out_dtype,
           x.get_device(), dy.get_device(), offsets.get_device(), xp % 16, dp % 16)
    plan = _PLANS.kept.get(key) or _plan_weight_gradient(key, x, dy, offsets, groups, out_dtype)
    if plan.copy:
        return _weight_gradient(x if _unit(x) else _copied(x), dy if _unit(dy) else _copied(dy), offsets, groups,
                                out_dtype)
    dw = x.new_empty_strided(plan.shape, plan.strides, dtype=plan.dtype)
    if not plan.empty:
        args = plan.args
        args.x, args.dy, args.offsets, args.dw = xp, dp, offsets.data_ptr(), dw.data_ptr()
        if plan.workspace:
            workspace = x.new_empty((plan.workspace,), dtype=torch.uint8)
            args.workspace = workspace.data_ptr()
        _launch(plan)
    return dw


class _GroupedMatmul(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, offsets, out_dtype):
        ctx.save_for_backward(x, w, offsets)
        return _product(x, w, offsets, out_dtype)

    @staticmethod
    def backward(ctx, dy):
        x, w, offsets = ctx.saved_tensors
        # by functions that record gradients themselves: a graph of the gradient is whole
        dy = dy.to(x.dtype)
        need_x, need_w = ctx.needs_input_grad[:2]
        dx = grouped_matmul(dy, w.transpose(1, 2), offsets) if need_x else None
        dw = _differentiable_weight_gradient(x, dy, offsets, w.shape[0]) if need_w else None
        return dx, dw, None, None


class _WeightGradient(torch.autograd.Function):
    """dw[e] = sum_r x[r]^T dy[r], bilinear like the product: its gradients are products."""

    @staticmethod
    def forward(ctx, x, dy, offsets, groups):
        ctx.save_for_backward(x, dy, offsets)
        return _weight_gradient(x, dy, offsets, groups, None)

    @staticmethod
    def backward(ctx, v):
        x, dy, offsets = ctx.saved_tensors
        v = v.to(x.dtype)
        need_x, need_dy = ctx.needs_input_grad[:2]
        return (grouped_matmul(dy, v.transpose(1, 2), offsets) if need_x else None,
                grouped_matmul(x, v, offsets) if need_dy else None, None, None)


def _differentiable_weight_gradient(x, dy, offsets, groups):
    if _LEVEL._current_level >= 0:
        _check_tangents(x, dy)
    if (x.requires_grad or dy.requires_grad) and torch.is_grad_enabled():
        return _WeightGradient.apply(x, dy, offsets, groups)
    return _weight_gradient(x, dy, offsets, groups, None)


def grouped_matmul(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor, *,
                   out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """y[r] = x[r] @ w[e] for the rows r of each group e; zero rows outside the groups.

    x (T, K) and w (E, K, N) of the same dtype (bf16 or fp16), w stored along K
    or along N (other layouts, and rows that do not start on 16-byte
    boundaries, are copied first);
    offsets (E + 1,) int32 or int64.  Returns (T, N) in the operands' dtype, or
    fp32 with ``out_dtype=torch.float32``.  Sums are held in fp32 and rounded
    once.  Differentiable in x and w, to any order: a gradient is rounded to the
    operands' dtype before it is multiplied.  Forward-mode derivatives are refused.
    """
    if _LEVEL._current_level >= 0:
        _check_tangents(x, w)
    if (x.requires_grad or w.requires_grad) and torch.is_grad_enabled():
        return _GroupedMatmul.apply(x, w, offsets, out_dtype)
    return _product(x, w, offsets, out_dtype)


def grouped_matmul_backward(dy: torch.Tensor, x: torch.Tensor, w: torch.Tensor,
                            offsets: torch.Tensor, *, dw_dtype: Optional[torch.dtype] = None
                            ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Gradients of ``grouped_matmul``: dx[r] = dy[r] @ w[e]^T, dw[e] = sum_r x[r]^T dy[r].

    Returns (dx, dw): dx (T, K) in the operands' dtype, dw (E, K, N) in it or,
    with ``dw_dtype=torch.float32``, in fp32.  The gradient of an expert without
    rows is zero.  No gradient of the gradients is recorded here; autograd of
    ``grouped_matmul`` records it.  Forward-mode derivatives are refused.
    """
    if _LEVEL._current_level >= 0:
        _check_tangents(dy, x, w)
    assert dy.dim() == 2 and x.dim() == 2 and w.dim() == 3, "x and dy must have 2 dimensions, w 3"
    assert dy.dtype is x.dtype, f"x/dy dtype mismatch: {x.dtype} vs {dy.dtype}"
    assert dy.shape[0] == x.shape[0] and dy.shape[1] == w.shape[2], \
        f"dy must be {(x.shape[0], w.shape[2])}, got {tuple(dy.shape)}"
    assert x.shape[1] == w.shape[1], f"contraction dim mismatch: x K={x.shape[1]}, w K={w.shape[1]}"
    dw_dtype = _out_dtype(dw_dtype, x.dtype)
    if dy.is_cuda and not _readable(dy):
        dy = _copied(dy)                                  # once for both products
    return (_product(dy, w.transpose(1, 2), offsets, None),
            _weight_gradient(x, dy, offsets, w.shape[0], dw_dtype))


def quantize_w4(w: torch.Tensor, group_size: int = 128, *, symmetric: bool = True,
                scale_dtype: Optional[torch.dtype] = None
                ) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """4-bit form of weights (..., K, N) for ``matmul_w4``: (packed, scales, zeros).

    Each group of ``group_size`` weights along K has one scale s and value
    (q - z) s with q in 0..15: z = 8 (``symmetric``, zeros is None) or a zero
    point of its own.  packed (..., N, K / 2) holds two q a byte, the even k in
    the low half; scales (and zeros) are (..., N, K / group_size).
    """
    assert w.is_floating_point() and w.dim() >= 2, "w must be a floating-point matrix or a stack"
    k = w.shape[-2]
    assert group_size >= 32 and group_size % 32 == 0 and k % group_size == 0, \
        f"the group size must be a multiple of 32 that divides K (group_size={group_size}, K={k})"
    scale_dtype = scale_dtype or (w.dtype if w.dtype in GROUPED_DTYPES else torch.float32)
    v = w.transpose(-1, -2).float().unflatten(-1, (-1, group_size))
    if symmetric:
        scales = (v.abs().amax(-1) / 7.5).to(scale_dtype)
        zeros = None
        zero = torch.full_like(scales, 8, dtype=torch.float32)
    else:
        low, high = v.amin(-1).clamp(max=0), v.amax(-1).clamp(min=0)
        scales = ((high - low) / 15).to(scale_dtype)
        s = scales.float()
        zero = torch.where(s > 0, torch.round(-low / s), 0.0).clamp(0, 15)
        zeros = zero.to(torch.uint8)
    s = scales.float().unsqueeze(-1)
    q = torch.where(s > 0, torch.round(v / s), 0.0) + zero.unsqueeze(-1)
    q = q.clamp(0, 15).to(torch.uint8).flatten(-2)
    return (q[..., 0::2] | (q[..., 1::2] << 4)).contiguous(), scales, zeros


def _plan_w4(key, x, packed, scales, zeros, offsets, out_dtype) -> _Plan:
    _check_rows(x, "x")
    lead = 2 if offsets is None else 3
    p_shape, s_shape = packed.shape, scales.shape
    rows, k = x.shape
    assert len(p_shape) == lead, f"packed must have {lead} dimensions, got shape {tuple(p_shape)}"
    assert packed.dtype is torch.uint8, f"packed must be uint8, got {packed.dtype}"
    n = p_shape[-2]
    assert p_shape[-1] * 2 == k, f"contraction dim mismatch: x K={k}, packed K={p_shape[-1] * 2}"
    assert len(s_shape) == lead and s_shape[:-1] == p_shape[:-1], \
        f"scales of shape {tuple(s_shape)} do not fit packed {tuple(p_shape)}"
    assert scales.dtype in _SCALE_DTYPES, f"unsupported scale dtype: {scales.dtype}"
    groups = s_shape[-1]
    assert groups > 0 and k > 0 and k % groups == 0 and (k // groups) % 32 == 0, \
        f"the group size must be a multiple of 32 that divides K ({groups} scales, K={k})"
    if zeros is not None:
        assert zeros.dtype is torch.uint8, f"zeros must be uint8, got {zeros.dtype}"
        assert zeros.shape == s_shape, \
            f"zeros of shape {tuple(zeros.shape)} do not fit scales {tuple(s_shape)}"
    experts = 1 if offsets is None else p_shape[0]
    assert experts >= 1, "packed must hold at least one expert"
    out_dtype = _out_dtype(out_dtype, x.dtype)
    if offsets is not None:
        _check_offsets(offsets, experts)
    device = _check_places(x, packed, scales, zeros, offsets)
    copy = (not _readable(x) or not packed.is_contiguous() or not scales.is_contiguous()
            or packed.data_ptr() % 16 != 0 or (zeros is not None and not zeros.is_contiguous()))
    args = _lib.W4Args(None, None, None, None, None, None, rows, k, n, x.stride(0), n * (k // 2), k // 2,
                       n * groups, groups, n, experts, k // groups,
                       offsets is not None and offsets.dtype is torch.int64, _OZ_DTYPE[x.dtype],
                       _OZ_DTYPE[scales.dtype], _OZ_DTYPE[out_dtype])
    return _PLANS.keep(key, _make_plan("oz_matmul_w4", args, (rows, n), out_dtype, device,
                                       rows == 0 or n == 0, copy))


def matmul_w4(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor,
              zeros: Optional[torch.Tensor] = None, *, offsets: Optional[torch.Tensor] = None,
              out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """y = x @ W^T with W[n, k] = (q[n, k] - z[n, k / g]) s[n, k / g] held in 4 bits.

    x (T, K) bf16 or fp16; packed (N, K / 2) uint8, two values a byte, the even
    k in the low half; scales (N, K / g) fp16, bf16 or fp32; zeros (N, K / g)
    uint8 (any value), or None for 8 everywhere (the layout ``quantize_w4`` returns).
    With ``offsets`` the weights have a leading expert dimension and the rows
    of x come in groups.  Returns (T, N) in x's dtype or fp32.  Made for few
    rows a matrix (the weights' bytes bound it); any number is right.  Layouts
    that the copy unit cannot read are copied first.  For serving: no gradient
    is recorded, and forward-mode derivatives are refused.
    """
    if _LEVEL._current_level >= 0:
        _check_tangents(x, scales)
    xp, pp = x.data_ptr(), packed.data_ptr()
    key = (x.shape, x.stride(), x.dtype, packed.shape, packed.stride(), packed.dtype, scales.shape,
           scales.stride(), scales.dtype, out_dtype, x.get_device(), packed.get_device(), scales.get_device(),
           xp % 16, pp % 16,
           None if zeros is None else (zeros.shape, zeros.stride(), zeros.dtype, zeros.get_device()),
           None if offsets is None else (offsets.shape, offsets.stride(), offsets.dtype, offsets.get_device()))
    plan = _PLANS.kept.get(key) or _plan_w4(key, x, packed, scales, zeros, offsets, out_dtype)
    if plan.copy and not plan.empty:
        packed = packed.contiguous()
        return matmul_w4(_as_operand(x), packed.clone() if packed.data_ptr() % 16 else packed, scales.contiguous(),
                         None if zeros is None else zeros.contiguous(), offsets=offsets, out_dtype=out_dtype)
    y = x.new_empty_strided(plan.shape, plan.strides, dtype=plan.dtype)
    if not plan.empty:
        args = plan.args
        args.x, args.packed, args.scales, args.y = xp, pp, scales.data_ptr(), y.data_ptr()
        args.zeros = None if zeros is None else zeros.data_ptr()
        args.offsets = None if offsets is None else offsets.data_ptr()
        _launch(plan)
    return y
