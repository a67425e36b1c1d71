"""Gradients of many tensors, clipped by their global norm."""

from __future__ import annotations

import ctypes
from typing import Iterable, Optional, Sequence

import torch

from . import _lib
from .api import _OZ_DTYPE
from .experts import _CURRENT_DEVICE, _LEVEL, _OnDevice, _check_places, _check_tangents, _stream_of

CLIP_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
_CODES = {t: _OZ_DTYPE[t] for t in CLIP_DTYPES}


def _dense(t: torch.Tensor) -> bool:
    """Whether t's elements fill their memory, in some order of its dimensions."""
    if t.is_contiguous():
        return True
    size = 1
    for stride, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != size:
            return False
        size *= n
    return True


def clip_gradients(grads: Iterable[torch.Tensor], max_norm: float, *, eps: float = 1e-6,
                   out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """Scales gradients so that their common norm is at most max_norm; returns the norm before.

    norm = sqrt(sum of the squares of all elements of all tensors), and every
    element is multiplied by min(1, max_norm / (norm + eps)).  grads: fp32, bf16
    or fp16 tensors on one device, mixed as they come, each dense (its elements
    fill their memory in some order of its dimensions).  In place, or into ``out``:
    as many tensors of the same shapes and strides, of any of these dtypes (the fp32
    gradients of bf16 weights, say); they must not share memory with each other or
    with gradients other than their own.  Returns the norm as a 0-dimensional fp32
    tensor; nothing waits for it.  A norm that is not finite scales by 0 (an infinite
    one) or makes every result NaN.  Forward-mode derivatives are refused, and no
    gradient is recorded.
    """
    grads = list(grads)
    assert grads, "at least one gradient is needed"
    assert max_norm >= 0, f"max_norm must not be negative, got {max_norm}"
    assert eps >= 0, f"eps must not be negative, got {eps}"
    outs = grads if out is None else list(out)
    assert len(outs) == len(grads), f"{len(grads)} gradients, but {len(outs)} results"
    if _LEVEL._current_level >= 0:
        _check_tangents(*grads, *outs)
    n = len(grads)
    device = grads[0].get_device()
    for t in grads if out is None else grads + outs:
        if t.dtype not in _CODES:
            raise AssertionError(f"unsupported dtype: {t.dtype}")
        if t.get_device() != device or device < 0:
            _check_places(grads[0], t)
        if not t.is_contiguous() and not _dense(t):
            raise AssertionError(f"a gradient of shape {tuple(t.shape)} and strides {t.stride()} is not dense")
    if out is not None:
        for g, o in zip(grads, outs):
            if g.shape != o.shape or (g.stride() != o.stride() and not (g.is_contiguous() and o.is_contiguous())):
                raise AssertionError(f"a result must be laid out like its gradient: {tuple(o.shape)}, strides "
                                     f"{o.stride()} for {tuple(g.shape)}, strides {g.stride()}")
    lib = _lib.load()
    norm = grads[0].new_empty((), dtype=torch.float32)
    size = lib.oz_clip_workspace_bytes(n)
    workspace = grads[0].new_empty((size,), dtype=torch.uint8)
    pointers = ctypes.c_void_p * n
    from_ = pointers(*[t.data_ptr() for t in grads])
    to = from_ if out is None else pointers(*[t.data_ptr() for t in outs])
    sizes = (ctypes.c_int64 * n)(*[t.numel() for t in grads])
    types = (ctypes.c_int32 * n)(*[_CODES[t.dtype] for t in grads])
    out_types = types if out is None else (ctypes.c_int32 * n)(*[_CODES[t.dtype] for t in outs])
    address = ctypes.addressof
    args = _lib.ClipArgs(address(from_), address(to), address(sizes), address(types), address(out_types),
                         norm.data_ptr(), workspace.data_ptr(), size, float(max_norm), float(eps), n, 0)
    if _CURRENT_DEVICE() == device:
        status = lib.oz_clip(ctypes.byref(args), _stream_of(device))
    else:
        with _OnDevice(device):
            status = lib.oz_clip(ctypes.byref(args), _stream_of(device))
    if status:
        _lib.check(status)
    torch.autograd.graph.increment_version(outs)      # the results' memory has changed behind torch's back
    return norm
