"""Orthogonalisation of matrix updates by Newton-Schulz steps."""

from __future__ import annotations

import ctypes
from typing import Optional, Sequence, Union

import torch

from . import _lib
from .api import _OZ_DTYPE, _check_cuda
from .experts import _OnDevice, _stream_of

ORTHOGONALIZE_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def _coefficients(coefficients, steps: int):
    rows = [tuple(c) for c in coefficients] if hasattr(coefficients[0], "__len__") else \
        [tuple(coefficients)] * steps
    assert len(rows) == steps and all(len(r) == 3 for r in rows), \
        f"coefficients must be one (a, b, c) or one for each of the {steps} steps"
    return (ctypes.c_double * (3 * steps))(*[float(v) for r in rows for v in r])


def orthogonalize(g: torch.Tensor, steps: int = 5,
                  coefficients: Union[Sequence[float], Sequence[Sequence[float]]] = (
                      3.4445, -4.7750, 2.0315),
                  eps: float = 1e-7, *, num_splits: Optional[int] = None) -> torch.Tensor:
    """The (nearly) orthogonal matrix with the singular vectors of g.

    g (..., M, N) fp32, bf16 or fp16, any strides; batch members are
    independent.  X = g / (|g|_F + eps), then ``steps`` times with A = X X^T
    X <- a X + (b A + c A^2) X, which drives the singular values of X towards
    1 (``coefficients``: one (a, b, c) for all steps or one for each).  Returns
    a contiguous tensor of g's shape and dtype.

    ``num_splits`` is how many fp16 slices of each matrix the products use: 1
    (11 bits, the default for bf16 whose result has 8) or 2 (22 bits, the
    default for fp32 and fp16).  Sums are held in fp32.
    """
    assert g.dim() >= 2, f"g must be a matrix or a stack of them, got shape {tuple(g.shape)}"
    assert g.dtype in ORTHOGONALIZE_DTYPES, f"unsupported dtype: {g.dtype}"
    assert steps >= 1, f"at least one step is needed, got {steps}"
    assert eps >= 0, f"eps must not be negative, got {eps}"
    if num_splits is None:
        num_splits = 1 if g.dtype == torch.bfloat16 else 2
    assert num_splits in (1, 2), f"num_splits must be 1 or 2, got {num_splits}"
    coeffs = _coefficients(coefficients, steps)
    _check_cuda(g)
    out = torch.empty(g.shape, dtype=g.dtype, device=g.device)
    if g.numel() == 0:
        return out
    m, n = g.shape[-2:]
    g3 = g.reshape(-1, m, n)
    lib = _lib.load()
    code = _OZ_DTYPE[g.dtype]
    ws_bytes = lib.oz_orthogonalize_workspace_bytes(code, g3.shape[0], m, n, num_splits)
    ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=g.device)
    device = g.get_device()
    with _OnDevice(device):
        _lib.check(lib.oz_orthogonalize(
            g3.data_ptr(), code, g3.shape[0], m, n, *g3.stride(), steps, coeffs, float(eps),
            num_splits, out.data_ptr(), ws.data_ptr(), ws_bytes, _stream_of(device)))
    return out
