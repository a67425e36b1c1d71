"""Sizes past what the operators around an expert layer's products take are refused, by the library's
functions and by the calls, which reach them with views of little memory; no GPU needed."""

import ctypes

import pytest
import torch

import ozaki_triton_b200 as oz
from ozaki_triton_b200 import _lib, fused, routing

FAR = [2 ** 30 + 1, 2 ** 31, 2 ** 32 - 300, 2 ** 32, 2 ** 32 + 1, 2 ** 49, 2 ** 59, 2 ** 63 - 1]


@pytest.mark.parametrize("far", FAR)
def test_workspace_functions(far):
    lib = _lib.load()
    for act in (0, 2):
        for sums in (0, 1):
            assert lib.oz_linear_backward_workspace_bytes(1, far, act, sums) == _lib.OZ_ERR_INVALID
            assert lib.oz_linear_backward_workspace_bytes(far, 1, act, sums) == _lib.OZ_ERR_INVALID
            assert "range" in lib.oz_last_error().decode()
    for experts in (1, 64, 1024):
        assert lib.oz_route_workspace_bytes(far, experts) == _lib.OZ_ERR_INVALID
        assert "range" in lib.oz_last_error().decode()
    args = _lib.LinearArgs(rows=far, k=8, n=8, x_sr=8, w_sk=8, w_sn=1, dtype=_lib.OZ_F16, out_dtype=_lib.OZ_F16)
    assert lib.oz_linear_workspace_bytes(ctypes.byref(args)) == _lib.OZ_ERR_INVALID


@pytest.mark.parametrize("far", FAR)
def test_entries(far):
    lib, p = _lib.load(), 256
    for picks in (1, 2, 32):
        a = dict(logits=p, weights=p, chosen=p, counts=p, tokens=p, rows=far, row=64, col=1, experts=64, picks=picks,
                 dtype=_lib.OZ_F32)
        args = _lib.RouteArgs(loss=p, slots=p, offsets=p, workspace=p, workspace_bytes=2 ** 62, **a)
        assert lib.oz_route(ctypes.byref(args), None) == _lib.OZ_ERR_INVALID
        assert lib.oz_route_backward(ctypes.byref(_lib.RouteBackwardArgs(dlogits=p, **a)), None) == _lib.OZ_ERR_INVALID
        args = _lib.RowsArgs(x=p, rows=p, x_out=p, rows_out=p, slots=p, offsets=p, weights=p, dweights=p, tokens=far, d=8,
                             x_row=8, rows_row=8, experts=2, picks=picks, dtype=_lib.OZ_F32)
        for name in ("oz_dispatch", "oz_combine", "oz_combine_backward"):
            assert getattr(lib, name)(ctypes.byref(args), None) == _lib.OZ_ERR_INVALID
    if far > 2 ** 42:
        held = ((ctypes.c_void_p * 1)(p), (ctypes.c_int64 * 1)(far), (ctypes.c_int32 * 1)(_lib.OZ_F32))
        grads, sizes, types = map(ctypes.addressof, held)
        args = _lib.ClipArgs(grads=grads, outs=grads, sizes=sizes, dtypes=types, out_dtypes=types, norm=p, workspace=p,
                             workspace_bytes=2 ** 40, max_norm=1.0, tensors=1)
        assert lib.oz_clip(ctypes.byref(args), None) == _lib.OZ_ERR_INVALID


def test_calls(monkeypatch):
    for module in (fused, routing):
        monkeypatch.setattr(module, "_PLANS", type(module._PLANS)())
        monkeypatch.setattr(module, "_check_places", lambda *ts: 0)
        monkeypatch.setattr(module, "_launch", lambda plan: pytest.fail("launched"))
    for far in (2 ** 31, 2 ** 32, 2 ** 49):
        with pytest.raises(oz.OzakiError, match="range"):
            oz.route(torch.zeros(1, 1).expand(far, 1), 1)
    one = torch.zeros(1, 1, dtype=torch.float16)
    for rows, n in ((1, 2 ** 32), (2 ** 32, 1), (1, 2 ** 31), (2 ** 32, 2 ** 10)):
        with pytest.raises(oz.OzakiError, match="range"):
            oz.fused_matmul_backward(one.expand(rows, n), one.expand(rows, 1), one.expand(1, n), bias=True)
