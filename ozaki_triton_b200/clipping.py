"""Gradients of many tensors, clipped by their global norm."""

from __future__ import annotations

import ctypes
from array import array
from operator import attrgetter
from typing import Iterable, Optional, Sequence

import torch

from . import _lib
from .api import _OZ_DTYPE
from .experts import _CURRENT_DEVICE, _LEVEL, _OnDevice, _check_places, _check_tangents, _stream_of

CLIP_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
_CODES = {t: _OZ_DTYPE[t] for t in CLIP_DTYPES}
_ALLOWED = frozenset(CLIP_DTYPES)
_WORKSPACES = {}             # bytes for so many tensors
# (a quarter less host time than by attribute, for each of a call's many tensors)
_Tensor, _DTYPE = torch.Tensor, attrgetter("dtype")


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
    tensor; nothing waits for it.  Squares may leave fp32's range as long as the norm does
    not (a factor below 1.2e-38 has fewer bits).  A norm that is not finite in fp32 scales
    by 0 (an infinite one) or makes every result NaN.  Forward-mode derivatives are refused,
    and no gradient is recorded.
    """
    grads = list(grads)
    assert grads, "at least one gradient is needed"
    assert max_norm >= 0, f"max_norm must not be negative, got {max_norm}"
    assert eps >= 0, f"eps must not be negative, got {eps}"
    outs = grads if out is None else list(out)
    assert len(outs) == len(grads), f"{len(grads)} gradients, but {len(outs)} results"
    if _LEVEL._current_level >= 0:
        _check_tangents(*grads, *outs)
    n, first = len(grads), grads[0]
    device = first.get_device()
    given = grads if out is None else grads + outs
    types = list(map(_DTYPE, given))
    if not _ALLOWED.issuperset(types):
        raise AssertionError(f"unsupported dtype: {next(t for t in types if t not in _ALLOWED)}")
    if device < 0 or set(map(_Tensor.get_device, given)) != {device}:
        _check_places(*given)
    if not all(map(_Tensor.is_contiguous, given)):
        for t in given:
            assert _dense(t), f"a gradient of shape {tuple(t.shape)} and strides {t.stride()} is not dense"
        for g, o in zip(grads, outs):
            assert g.stride() == o.stride() or (g.is_contiguous() and o.is_contiguous()), \
                f"a result must be laid out like its gradient: strides {o.stride()} for {g.stride()}"
    if out is not None and not all(map(_Tensor.is_same_size, grads, outs)):
        raise AssertionError("a result must have its gradient's shape")
    lib = _lib.load()
    norm = first.new_empty_strided((), (), dtype=torch.float32)
    size = _WORKSPACES.get(n) or _WORKSPACES.setdefault(n, lib.oz_clip_workspace_bytes(n))
    workspace = first.new_empty_strided((size,), (1,), dtype=torch.uint8)
    # addresses, sizes and types as the library takes them
    pointers = array("Q", map(_Tensor.data_ptr, given))
    sizes = array("q", map(_Tensor.numel, grads))
    codes = array("i", [_CODES[t] for t in types])
    at, at_codes = pointers.buffer_info()[0], codes.buffer_info()[0]
    second = 0 if out is None else n
    args = _lib.ClipArgs(at, at + 8 * second, sizes.buffer_info()[0], at_codes, at_codes + 4 * second, norm.data_ptr(),
                         workspace.data_ptr(), size, float(max_norm), float(eps), n, 0)
    if _CURRENT_DEVICE() == device:
        status = lib.oz_clip(ctypes.byref(args), _stream_of(device))
    else:
        with _OnDevice(device):
            status = lib.oz_clip(ctypes.byref(args), _stream_of(device))
    if status:
        _lib.check(status)
    torch.autograd.graph.increment_version(outs)      # the results' memory has changed behind torch's back
    return norm
