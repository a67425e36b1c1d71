"""The library's entries refuse addresses that are not multiples of an element's size, which
the kernels cannot read; no GPU needed (nothing is launched)."""

import ctypes

import pytest

from ozaki_triton_b200 import _lib

P = 1024                          # never dereferenced: the checks fail first
F32, F16, BF16 = _lib.OZ_F32, _lib.OZ_F16, _lib.OZ_BF16

LINEAR = dict(x=P, w=P, y=P, bias=P, residual=P, pre=P, rows=4, k=8, n=8, x_sr=8, w_sk=8, w_sn=1, residual_sr=8, dtype=F16,
              out_dtype=F16, bias_dtype=F16)
LINEAR_BACKWARD = dict(dy=P, x=P, w=P, pre=P, dx=P, dw=P, db=P, workspace=P, workspace_bytes=1 << 20, rows=4, k=8, n=8,
                       dy_sr=8, x_sr=8, w_sk=8, w_sn=1, pre_sr=8, dtype=BF16, dw_dtype=BF16, act=1)
ROUTE = dict(logits=P, weights=P, loss=P, chosen=P, slots=P, offsets=P, counts=P, tokens=P, rows=4, row=8, col=1, experts=8,
             picks=2, dtype=F32)
ROUTE_BACKWARD = dict(logits=P, dweights=P, dloss=P, weights=P, chosen=P, counts=P, tokens=P, dlogits=P, rows=4, row=8, col=1,
                      experts=8, picks=2, dtype=F32)
ROWS = dict(x=P, rows=P, x_out=P, rows_out=P, slots=P, offsets=P, weights=P, dweights=P, tokens=4, d=8, x_row=8, rows_row=8,
            experts=2, picks=2, dtype=F32)

CASES = [("oz_linear", _lib.LinearArgs, LINEAR, dict.fromkeys(("x", "w", "y", "bias", "residual", "pre"), 1)),
         ("oz_linear", _lib.LinearArgs, {**LINEAR, "out_dtype": F32, "bias_dtype": F32}, dict(y=2, bias=2, residual=2, pre=1)),
         ("oz_linear_backward", _lib.LinearBackwardArgs, LINEAR_BACKWARD,
          dict(dy=1, x=1, w=1, pre=1, dx=1, dw=1, db=2)),
         ("oz_linear_backward", _lib.LinearBackwardArgs, {**LINEAR_BACKWARD, "dw_dtype": F32, "act": 0}, dict(dw=2, dy=1)),
         ("oz_route", _lib.RouteArgs, ROUTE,
          dict.fromkeys(("logits", "weights", "loss", "chosen", "slots", "offsets", "counts", "tokens"), 2)),
         ("oz_route", _lib.RouteArgs, {**ROUTE, "dtype": F16}, dict(logits=1)),
         ("oz_route_backward", _lib.RouteBackwardArgs, ROUTE_BACKWARD,
          dict.fromkeys(("logits", "dweights", "dloss", "weights", "chosen", "counts", "tokens", "dlogits"), 2)),
         ("oz_route_backward", _lib.RouteBackwardArgs, {**ROUTE_BACKWARD, "dtype": BF16}, dict(logits=1))]
CASES += [(name, _lib.RowsArgs, ROWS, dict.fromkeys(fields, 2)) for name, fields in (
    ("oz_dispatch", ("x", "rows_out", "slots", "offsets")), ("oz_combine", ("rows", "x_out", "slots", "weights")),
    ("oz_combine_backward", ("x", "rows", "rows_out", "slots", "offsets", "weights", "dweights")))]
CASES += [(name, _lib.RowsArgs, {**ROWS, "dtype": F16}, dict(x=1, rows=1)) for name in ("oz_combine_backward",)]


@pytest.mark.parametrize("name,struct,args,fields", CASES, ids=[f"{c[0]}{i}" for i, c in enumerate(CASES)])
def test_misaligned_addresses(name, struct, args, fields):
    lib = _lib.load()
    before = lib.oz_launch_count()
    for field, off in fields.items():
        held = struct(**{**args, field: P + off})
        assert getattr(lib, name)(ctypes.byref(held), None) == _lib.OZ_ERR_INVALID, field
        assert "aligned" in lib.oz_last_error().decode() or "boundary" in lib.oz_last_error().decode(), field
    assert lib.oz_launch_count() == before


def test_misaligned_norm():
    lib = _lib.load()
    held = ((ctypes.c_void_p * 1)(P), (ctypes.c_int64 * 1)(8), (ctypes.c_int32 * 1)(F32))
    grads, sizes, types = map(ctypes.addressof, held)
    args = _lib.ClipArgs(grads=grads, outs=grads, sizes=sizes, dtypes=types, out_dtypes=types, norm=P + 2, workspace=P,
                         workspace_bytes=1 << 20, max_norm=1.0, tensors=1)
    assert lib.oz_clip(ctypes.byref(args), None) == _lib.OZ_ERR_INVALID
    assert "aligned" in lib.oz_last_error().decode()
