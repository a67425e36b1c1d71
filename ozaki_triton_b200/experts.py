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

from typing import Optional, Tuple

import torch

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


class _OnDevice:
    """Makes a device current for a call, at no cost where it is already."""

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


def _as_operand(t: torch.Tensor) -> torch.Tensor:
    """t, or a copy where the copy unit cannot read its layout: it wants a unit
    stride along the last dimension, 16-byte boundaries and no repeated rows."""
    shape, strides = t.shape, t.stride()
    if (strides[-1] == 1 or shape[-1] == 1) and t.data_ptr() % 16 == 0:
        for n, s in zip(shape[:-1], strides):
            if n > 1 and (s <= 0 or s % 8):
                break
        else:
            return t
    return _copied(t)


def _as_weights(w: torch.Tensor) -> torch.Tensor:
    """The same for (E, K, N) weights, which may be stored along K or along N."""
    if w.stride(1) == 1 and w.stride(2) != 1:
        return _as_operand(w.transpose(1, 2)).transpose(1, 2)
    return _as_operand(w)


def _product(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor, out_dtype: torch.dtype,
             device: int) -> torch.Tensor:
    rows, k = x.shape
    groups, _, n = w.shape
    y = x.new_empty((rows, n), dtype=out_dtype)
    if rows == 0 or n == 0:
        return y
    if k > 0:
        x, w = _as_operand(x), _as_weights(w)
    w_se, w_sk, w_sn = w.stride()
    with _OnDevice(device):
        _lib.check(_lib.load().oz_grouped_matmul(
            x.data_ptr(), w.data_ptr(), offsets.data_ptr(), offsets.dtype is torch.int64,
            _OZ_DTYPE[x.dtype], _OZ_DTYPE[out_dtype], groups, rows, k, n, x.stride(0),
            w_se, w_sk, w_sn, y.data_ptr(), n, _stream_of(device)))
    return y


def _weight_gradient(x: torch.Tensor, dy: torch.Tensor, offsets: torch.Tensor, groups: int,
                     out_dtype: torch.dtype, device: int) -> torch.Tensor:
    rows, k = x.shape
    n = dy.shape[1]
    dw = x.new_empty((groups, k, n), dtype=out_dtype)
    if k == 0 or n == 0:
        return dw
    if rows > 0:
        x, dy = _as_operand(x), _as_operand(dy)
    with _OnDevice(device):
        _lib.check(_lib.load().oz_grouped_wgrad(
            x.data_ptr(), dy.data_ptr(), offsets.data_ptr(), offsets.dtype is torch.int64,
            _OZ_DTYPE[x.dtype], _OZ_DTYPE[out_dtype], groups, rows, k, n, x.stride(0),
            dy.stride(0), dw.data_ptr(), _stream_of(device)))
    return dw


def _check_grouped(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor) -> None:
    _check_rows(x, "x")
    assert w.dim() == 3, f"w must have 3 dimensions, got shape {tuple(w.shape)}"
    assert w.dtype == x.dtype, f"x/w dtype mismatch: {x.dtype} vs {w.dtype}"
    assert w.shape[0] >= 1, "w must hold at least one expert"
    assert w.shape[1] == x.shape[1], f"contraction dim mismatch: x K={x.shape[1]}, w K={w.shape[1]}"
    _check_offsets(offsets, w.shape[0])


class _GroupedMatmul(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, offsets, out_dtype):
        ctx.save_for_backward(x, w, offsets)
        return _product(x, w, offsets, out_dtype, x.get_device())

    @staticmethod
    def backward(ctx, dy):
        x, w, offsets = ctx.saved_tensors
        dy, device = dy.to(x.dtype), x.get_device()
        need_x, need_w = ctx.needs_input_grad[:2]
        dx = _product(dy, w.transpose(1, 2), offsets, x.dtype, device) if need_x else None
        dw = _weight_gradient(x, dy, offsets, w.shape[0], w.dtype, device) if need_w else None
        return dx, dw, None, None


def grouped_matmul(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor, *,
                   out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """y[r] = x[r] @ w[e] for the rows r of each group e; zero rows outside the groups.

    x (T, K) and w (E, K, N) of the same dtype (bf16 or fp16), w stored along K
    or along N (other layouts, and rows that do not start on 16-byte
    boundaries, are copied first);
    offsets (E + 1,) int32 or int64.  Returns (T, N) in the operands' dtype, or
    fp32 with ``out_dtype=torch.float32``.  Sums are held in fp32 and rounded
    once.  Differentiable in x and w.
    """
    _check_grouped(x, w, offsets)
    out_dtype = _out_dtype(out_dtype, x.dtype)
    device = _check_places(x, w, offsets)
    if torch.is_grad_enabled() and (x.requires_grad or w.requires_grad):
        return _GroupedMatmul.apply(x, w, offsets, out_dtype)
    return _product(x, w, offsets, out_dtype, device)


def grouped_matmul_backward(dy: torch.Tensor, x: torch.Tensor, w: torch.Tensor,
                            offsets: torch.Tensor, *, dw_dtype: Optional[torch.dtype] = None
                            ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Gradients of ``grouped_matmul``: dx[r] = dy[r] @ w[e]^T, dw[e] = sum_r x[r]^T dy[r].

    Returns (dx, dw): dx (T, K) in the operands' dtype, dw (E, K, N) in it or,
    with ``dw_dtype=torch.float32``, in fp32.  The gradient of an expert without
    rows is zero.
    """
    _check_grouped(x, w, offsets)
    _check_rows(dy, "dy")
    assert dy.dtype == x.dtype, f"x/dy dtype mismatch: {x.dtype} vs {dy.dtype}"
    assert tuple(dy.shape) == (x.shape[0], w.shape[2]), \
        f"dy must be {(x.shape[0], w.shape[2])}, got {tuple(dy.shape)}"
    dw_dtype = _out_dtype(dw_dtype, x.dtype)
    device = _check_places(x, w, offsets, dy)
    x, dy = _as_operand(x), _as_operand(dy)               # once for both products
    return (_product(dy, w.transpose(1, 2), offsets, x.dtype, device),
            _weight_gradient(x, dy, offsets, w.shape[0], dw_dtype, device))


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


def matmul_w4(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor,
              zeros: Optional[torch.Tensor] = None, *, offsets: Optional[torch.Tensor] = None,
              out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """y = x @ W^T with W[n, k] = (q[n, k] - z[n, k / g]) s[n, k / g] held in 4 bits.

    x (T, K) bf16 or fp16; packed (N, K / 2) uint8, two values a byte, the even
    k in the low half; scales (N, K / g) fp16, bf16 or fp32; zeros (N, K / g)
    uint8, or None for 8 everywhere (the layout ``quantize_w4`` returns).
    With ``offsets`` the weights have a leading expert dimension and the rows
    of x come in groups.  Returns (T, N) in x's dtype or fp32.  Made for few
    rows a matrix (the weights' bytes bound it); any number is right.
    """
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
    y = x.new_empty((rows, n), dtype=out_dtype)
    if rows == 0 or n == 0:
        return y
    x = _as_operand(x)
    packed, scales = packed.contiguous(), scales.contiguous()
    if packed.data_ptr() % 16:
        packed = packed.clone()
    if zeros is not None:
        zeros = zeros.contiguous()
    with _OnDevice(device):
        _lib.check(_lib.load().oz_matmul_w4(
            x.data_ptr(), packed.data_ptr(), scales.data_ptr(),
            zeros.data_ptr() if zeros is not None else None,
            offsets.data_ptr() if offsets is not None else None,
            offsets is not None and offsets.dtype is torch.int64, _OZ_DTYPE[x.dtype],
            _OZ_DTYPE[scales.dtype], _OZ_DTYPE[out_dtype], experts, rows, k, n, k // groups,
            x.stride(0), n * (k // 2), k // 2, n * groups, groups, y.data_ptr(), n,
            _stream_of(device)))
    return y
