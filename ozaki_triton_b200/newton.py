"""Orthogonalisation of matrix updates by Newton-Schulz steps."""

from __future__ import annotations

import ctypes
import math
from typing import Optional, Sequence, Union

import torch

from . import _lib
from .api import _OZ_DTYPE, _check_cuda
from .experts import _CURRENT_DEVICE, _LEVEL, _OnDevice, _Plans, _check_tangents, _stream_of

ORTHOGONALIZE_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


class _Plan:
    """What a call derives from its matrices' type, shape and strides and from
    its other arguments: the checks passed and the library's arguments."""

    __slots__ = ("matrices", "rest", "workspace", "empty", "device")


_PLANS = _Plans()


def _plan(key, g, steps, coefficients, eps, num_splits) -> _Plan:
    assert g.dim() >= 2, f"g must be a matrix or a stack of them, got shape {tuple(g.shape)}"
    assert g.dtype in ORTHOGONALIZE_DTYPES, f"unsupported dtype: {g.dtype}"
    assert steps >= 1, f"at least one step is needed, got {steps}"
    assert eps >= 0, f"eps must not be negative, got {eps}"
    if num_splits is None:
        rows, cols = sorted(g.shape[-2:])
        work = g.numel() * rows * (3 + rows / max(cols, 1))           # of a step
        num_splits = 1 if g.dtype == torch.bfloat16 and work >= 5e9 else 2
    assert num_splits in (1, 2), f"num_splits must be 1 or 2, got {num_splits}"
    rows = list(coefficients) if hasattr(coefficients[0], "__len__") else [coefficients] * steps
    assert len(rows) == steps and all(len(r) == 3 for r in rows), \
        f"coefficients must be one (a, b, c) or one for each of the {steps} steps"
    values = [float(v) for r in rows for v in r]
    assert all(math.isfinite(v) for v in values), "coefficients must be finite"
    _check_cuda(g)
    plan = _Plan()
    plan.device, plan.empty, plan.workspace = g.get_device(), g.numel() == 0, 0
    plan.matrices = plan.rest = None
    if not plan.empty:
        m, n = g.shape[-2:]
        code, batch = _OZ_DTYPE[g.dtype], g.numel() // (m * n)
        strides = g.stride() if g.dim() == 3 else (0, *g.stride()) if g.dim() == 2 else (m * n, n, 1)
        plan.matrices = (code, batch, m, n, *strides, steps, (ctypes.c_double * len(values))(*values), float(eps),
                         num_splits)
        plan.workspace = _lib.load().oz_orthogonalize_workspace_bytes(code, batch, m, n, steps, num_splits)
    return _PLANS.keep(key, plan)


def orthogonalize(g: torch.Tensor, steps: int = 5,
                  coefficients: Union[Sequence[float], Sequence[Sequence[float]]] = (
                      3.4445, -4.7750, 2.0315),
                  eps: float = 1e-7, *, num_splits: Optional[int] = None) -> torch.Tensor:
    """The (nearly) orthogonal matrix with the singular vectors of g.

    g (..., M, N) fp32, bf16 or fp16, any strides; batch members are
    independent.  X = g / (|g|_F + eps), then ``steps`` times with A = X X^T
    X <- a X + (b A + c A^2) X, which drives the singular values of X towards
    1 (``coefficients``: one (a, b, c) for all steps or one for each).  A zero
    matrix stays zero, also with eps = 0.  Returns a contiguous tensor of g's
    shape and dtype (at most 65535 matrices of at most 2^20 rows and columns).  For updates: no gradient is
    recorded, and forward-mode derivatives are refused.

    ``num_splits`` is how many fp16 slices of each matrix the products use: 1
    (11 bits, the default for bf16, whose result has 8, where the products'
    time counts: batch M N min(M, N) above 2e9 or so) or 2 (22 bits, the default
    elsewhere).  One slice leaves a bf16 result 1.15 to 1.4 times as far from the
    exact one as its rounding alone does; ask for 2 where that matters.  Sums are
    held in fp32.  The slices' scales follow from the largest singular value
    that the coefficients allow, so a schedule that lets one starting in [0, 1]
    grow past 8 before its last step is refused (OzakiError).  Small matrices (at
    most 128 rows or columns, where that fits on chip and is the faster way: up to
    16 steps, 4096 matrices and some 10^4 elements each) are worked on in fp32
    whatever ``num_splits`` is, with any coefficients.
    """
    if _LEVEL._current_level >= 0:
        _check_tangents(g)
    if not isinstance(coefficients, tuple) or hasattr(coefficients[0], "__len__"):
        coefficients = tuple(tuple(c) if hasattr(c, "__len__") else c for c in coefficients)
    if g.dim() > 3:
        g3 = g.reshape(-1, *g.shape[-2:]) if g.numel() else g
        return orthogonalize(g3, steps, coefficients, eps, num_splits=num_splits).view(g.shape) if g.numel() \
            else g.new_empty(g.shape)
    key = (g.shape, g.stride(), g.dtype, g.get_device(), steps, coefficients, eps, num_splits)
    plan = _PLANS.kept.get(key) or _plan(key, g, steps, coefficients, eps, num_splits)
    out = g.new_empty(g.shape)
    if plan.empty:
        return out
    ws = g.new_empty((plan.workspace,), dtype=torch.uint8) if plan.workspace else None
    args = (g.data_ptr(), *plan.matrices, out.data_ptr(), ws.data_ptr() if ws is not None else None, plan.workspace)
    call, device = _lib.load().oz_orthogonalize, plan.device
    if _CURRENT_DEVICE() == device:
        status = call(*args, _stream_of(device))
    else:
        with _OnDevice(device):
            status = call(*args, _stream_of(device))
    if status:
        _lib.check(status)
    return out
