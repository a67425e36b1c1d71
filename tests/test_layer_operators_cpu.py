"""Argument checks of the fused product, the router, the rows' operators and the
clipping; no GPU needed."""

import ctypes

import pytest
import torch
from torch.autograd import forward_ad

import ozaki_triton_b200 as oz
from ozaki_triton_b200 import _lib

F16, BF16, F32, I32 = torch.float16, torch.bfloat16, torch.float32, torch.int32


def zeros(*shape, dtype=F16):
    return torch.zeros(*shape, dtype=dtype)


def fused(**kw):
    a = dict(x=zeros(6, 64), w=zeros(64, 32), bias=zeros(32), activation="gelu", residual=zeros(6, 32), out_dtype=None)
    a.update(kw)
    return oz.fused_matmul(a["x"], a["w"], a["bias"], activation=a["activation"], residual=a["residual"],
                           out_dtype=a["out_dtype"])


@pytest.mark.parametrize("kw", [
    dict(x=zeros(6, 64, dtype=F32)), dict(x=zeros(6, 64, dtype=BF16)), dict(x=zeros(6, 63)), dict(x=zeros(1, 6, 64)),
    dict(x=zeros(64)), dict(w=zeros(1, 64, 32)), dict(w=zeros(64)), dict(bias=zeros(31)), dict(bias=zeros(1, 32)),
    dict(bias=zeros(32, dtype=BF16)), dict(activation="tanh"), dict(activation=""), dict(residual=zeros(6, 31)),
    dict(residual=zeros(32)), dict(residual=zeros(6, 32, dtype=F32)), dict(out_dtype=F32), dict(out_dtype=BF16),
    dict(out_dtype=torch.float64),
])
def test_fused_matmul_refuses(kw):
    with pytest.raises(AssertionError):
        fused(**kw)


def backward(**kw):
    a = dict(dy=zeros(6, 32), x=zeros(6, 64), w=zeros(64, 32), pre=zeros(6, 32), activation="silu", dw_dtype=None)
    a.update(kw)
    return oz.fused_matmul_backward(a["dy"], a["x"], a["w"], a["pre"], activation=a["activation"], bias=True,
                                    dw_dtype=a["dw_dtype"])


@pytest.mark.parametrize("kw", [
    dict(dy=zeros(6, 31)), dict(dy=zeros(5, 32)), dict(dy=zeros(6, 32, dtype=F32)), dict(dy=zeros(32)),
    dict(x=zeros(6, 63)), dict(x=zeros(6, 64, dtype=F32)), dict(w=zeros(64, 32, dtype=BF16)), dict(pre=None),
    dict(activation=None), dict(pre=zeros(6, 31)), dict(pre=zeros(6, 32, dtype=F32)), dict(dw_dtype=BF16),
    dict(activation="tanh"),
])
def test_fused_matmul_backward_refuses(kw):
    with pytest.raises(AssertionError):
        backward(**kw)


def routing(t=6, k=2, e=4, **kw):
    a = dict(weights=zeros(t, k, dtype=F32), experts=zeros(t, k, dtype=I32), slots=zeros(t, k, dtype=I32),
             offsets=zeros(e + 1, dtype=I32), counts=zeros(e, dtype=I32), tokens=zeros((), dtype=I32),
             balance_loss=zeros((), dtype=F32))
    a.update(kw)
    return oz.Routing(**a)


@pytest.mark.parametrize("logits,picks", [
    (zeros(6, 4, dtype=torch.float64), 2), (zeros(6, 4, dtype=I32), 2), (zeros(4), 2), (zeros(1, 6, 4), 2), (zeros(6, 4), 0),
    (zeros(6, 4), 5), (zeros(6, 64), 33), (zeros(6, 1025), 2), (zeros(6, 0), 1), (zeros(6, 4), -1),
])
def test_route_refuses(logits, picks):
    with pytest.raises(AssertionError):
        oz.route(logits, picks)


@pytest.mark.parametrize("kw", [
    dict(dweights=zeros(6, 3, dtype=F32)), dict(dweights=zeros(6, 2)), dict(dloss=zeros(1, dtype=F32)), dict(dloss=zeros(())),
    dict(logits=zeros(5, 4)), dict(logits=zeros(6, 5)), dict(logits=zeros(6, 1)), dict(routing=routing(weights=zeros(6, 2))),
    dict(routing=routing(experts=zeros(6, 2, dtype=torch.int64))), dict(routing=routing(counts=zeros(5, dtype=I32))),
    dict(routing=routing(tokens=zeros(1, dtype=I32))), dict(routing=routing(experts=zeros(6, dtype=I32))),
])
def test_route_backward_refuses(kw):
    a = dict(dweights=zeros(6, 2, dtype=F32), dloss=zeros((), dtype=F32), logits=zeros(6, 4), routing=routing())
    a.update(kw)
    with pytest.raises(AssertionError):
        oz.route_backward(**a)


BAD_ROUTINGS = [routing(slots=zeros(6, 2, dtype=torch.int64)), routing(slots=zeros(12, dtype=I32)),
                routing(slots=zeros(2, 6, dtype=I32).t()), routing(offsets=zeros(1, dtype=I32)),
                routing(offsets=zeros(5, dtype=torch.int64)), routing(offsets=zeros(10, dtype=I32)[::2]),
                routing(slots=zeros(6, 33, dtype=I32)), routing(slots=zeros(6, 0, dtype=I32))]


@pytest.mark.parametrize("r", BAD_ROUTINGS, ids=range(len(BAD_ROUTINGS)))
def test_rows_refuse_a_wrong_routing(r):
    t, n = (r.slots.shape[0], r.slots.numel()) if r.slots.dim() == 2 else (6, 12)
    for call in (lambda: oz.dispatch(zeros(t, 8), r), lambda: oz.combine(zeros(n, 8), r),
                 lambda: oz.dispatch_backward(zeros(n, 8), r), lambda: oz.combine_backward(zeros(t, 8), zeros(n, 8), r)):
        with pytest.raises(AssertionError):
            call()


def test_rows_refuse_wrong_tensors():
    r = routing()
    for call in (lambda: oz.dispatch(zeros(5, 8), r), lambda: oz.dispatch(zeros(6), r),
                 lambda: oz.dispatch(zeros(6, 8, dtype=I32), r), lambda: oz.combine(zeros(6, 8), r),
                 lambda: oz.combine(zeros(12, 8, dtype=torch.float64), r), lambda: oz.dispatch_backward(zeros(11, 8), r),
                 lambda: oz.combine(zeros(12, 8), routing(weights=zeros(6, 2))),
                 lambda: oz.combine(zeros(12, 8), routing(weights=zeros(6, 3, dtype=F32))),
                 lambda: oz.combine_backward(zeros(6, 8), zeros(12, 9), r),
                 lambda: oz.combine_backward(zeros(6, 8, dtype=BF16), zeros(12, 8), r),
                 lambda: oz.combine_backward(zeros(5, 8), zeros(12, 8), r)):
        with pytest.raises(AssertionError):
            call()


@pytest.mark.parametrize("grads,kw", [
    ([], {}), ([zeros(4)], dict(max_norm=-1.0)), ([zeros(4)], dict(eps=-1.0)), ([zeros(4)], dict(max_norm=float("nan"))),
    ([zeros(4, dtype=I32)], {}), ([zeros(4, dtype=torch.float64)], {}), ([zeros(4)], dict(out=[])),
])
def test_clip_refuses(grads, kw):
    with pytest.raises(AssertionError):
        oz.clip_gradients(grads, **{"max_norm": 1.0, **kw})


CALLS = {
    "product": lambda f: oz.fused_matmul(f(zeros(6, 64)), zeros(64, 32)),
    "product, w": lambda f: oz.fused_matmul(zeros(6, 64), f(zeros(64, 32))),
    "product, bias": lambda f: oz.fused_matmul(zeros(6, 64), zeros(64, 32), f(zeros(32))),
    "product, residual": lambda f: oz.fused_matmul(zeros(6, 64), zeros(64, 32), residual=f(zeros(6, 32))),
    "product's gradients": lambda f: oz.fused_matmul_backward(f(zeros(6, 32)), zeros(6, 64), zeros(64, 32)),
    "route": lambda f: oz.route(f(zeros(6, 4)), 2),
    "route's gradient": lambda f: oz.route_backward(f(zeros(6, 2, dtype=F32)), None, zeros(6, 4), routing()),
    "dispatch": lambda f: oz.dispatch(f(zeros(6, 8)), routing()),
    "dispatch's gradient": lambda f: oz.dispatch_backward(f(zeros(12, 8)), routing()),
    "combine": lambda f: oz.combine(f(zeros(12, 8)), routing()),
    "combine, weights": lambda f: oz.combine(zeros(12, 8), routing(weights=f(zeros(6, 2, dtype=F32)))),
    "combine's gradients": lambda f: oz.combine_backward(f(zeros(6, 8)), zeros(12, 8), routing()),
    "clip": lambda f: oz.clip_gradients([zeros(5), f(zeros(4))], 1.0),
}


@pytest.mark.parametrize("call", CALLS)
def test_hosts_and_tangents_are_refused(call):
    with pytest.raises(ValueError, match="CUDA tensors only"):
        CALLS[call](lambda t: t)
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="tangent"):
            CALLS[call](lambda t: forward_ad.make_dual(t, torch.ones_like(t)))


def test_library_entries_validate_without_a_launch():
    lib = _lib.load()
    n0 = lib.oz_launch_count()
    p = 256                       # never dereferenced: validation fails first
    bad, unsupported, ok = _lib.OZ_ERR_INVALID, _lib.OZ_ERR_UNSUPPORTED, _lib.OZ_OK

    def call(name, struct, **kw):
        args = struct(**kw)
        return getattr(lib, name)(ctypes.byref(args), None)

    def linear(**kw):
        a = dict(x=p, w=p, y=p, rows=4, k=8, n=8, x_sr=8, w_sk=8, w_sn=1, dtype=_lib.OZ_F16, out_dtype=_lib.OZ_F16,
                 bias_dtype=_lib.OZ_F16)
        a.update(kw)
        return call("oz_linear", _lib.LinearArgs, **a)
    assert lib.oz_linear(None, None) == bad
    assert linear(dtype=_lib.OZ_F32) == unsupported and linear(out_dtype=_lib.OZ_BF16) == unsupported
    assert linear(act=4) == unsupported and linear(act=-1) == unsupported
    assert linear(bias=p, bias_dtype=_lib.OZ_BF16) == unsupported
    assert linear(rows=-1) == bad and linear(k=2 ** 31) == bad and linear(y=None) == bad and linear(x=None) == bad
    assert linear(w_sk=8, w_sn=2) == bad
    # rows off the 16-byte boundaries, and sums in passes: copied first
    assert linear(k=12004, x_sr=12004, out_dtype=_lib.OZ_F32) == bad and "workspace" in lib.oz_last_error().decode()
    assert linear(x=p + 1) == bad and "aligned" in lib.oz_last_error().decode()
    assert linear(rows=0, y=None) == ok and linear(n=0, y=None) == ok

    def linear_backward(**kw):
        a = dict(dy=p, x=p, w=p, dx=p, dw=p, rows=4, k=8, n=8, dy_sr=8, x_sr=8, w_sk=8, w_sn=1, dtype=_lib.OZ_F16,
                 dw_dtype=_lib.OZ_F16)
        a.update(kw)
        return call("oz_linear_backward", _lib.LinearBackwardArgs, **a)
    assert lib.oz_linear_backward(None, None) == bad
    assert linear_backward(dtype=_lib.OZ_F32) == unsupported and linear_backward(dw_dtype=_lib.OZ_BF16) == unsupported
    assert linear_backward(dy=None) == bad and linear_backward(act=1) == bad and linear_backward(w=None) == bad
    assert linear_backward(act=1, pre=p) == bad and "workspace" in lib.oz_last_error().decode()
    assert lib.oz_linear_backward_workspace_bytes(-1, 4, 0, 0) == bad
    assert lib.oz_linear_backward_workspace_bytes(4, 9, 1, 0) == 256

    def route(**kw):
        a = dict(logits=p, weights=p, loss=p, chosen=p, slots=p, offsets=p, counts=p, tokens=p, rows=4, row=8, col=1,
                 experts=8, picks=2, dtype=_lib.OZ_F32)
        a.update(kw)
        return call("oz_route", _lib.RouteArgs, **a)
    assert lib.oz_route(None, None) == bad
    for kw in (dict(rows=-1), dict(experts=0), dict(experts=1025), dict(picks=0), dict(picks=9), dict(picks=33, experts=64),
               dict(rows=2 ** 30), dict(logits=None), dict(slots=None), dict(loss=None), dict(rows=10 ** 6)):
        assert route(**kw) == bad, kw
    assert route(dtype=_lib.OZ_I8) == unsupported
    assert lib.oz_route_workspace_bytes(4, 0) == bad and lib.oz_route_workspace_bytes(4, 8) == 0

    def route_backward(**kw):
        a = dict(logits=p, weights=p, chosen=p, counts=p, tokens=p, dlogits=p, rows=4, row=8, col=1, experts=8, picks=2,
                 dtype=_lib.OZ_F32)
        a.update(kw)
        return call("oz_route_backward", _lib.RouteBackwardArgs, **a)
    assert lib.oz_route_backward(None, None) == bad
    for kw in (dict(rows=-1), dict(experts=0), dict(picks=9), dict(dlogits=None), dict(tokens=None)):
        assert route_backward(**kw) == bad, kw
    assert route_backward(dtype=_lib.OZ_F64) == unsupported and route_backward(rows=0, dlogits=None) == ok

    for name in ("oz_dispatch", "oz_combine", "oz_combine_backward"):
        def rows(**kw):
            a = dict(x=p, rows=p, x_out=p, rows_out=p, slots=p, offsets=p, weights=p, dweights=p, tokens=4, d=8, x_row=8,
                     rows_row=8, experts=2, picks=2, dtype=_lib.OZ_F32)
            a.update(kw)
            return call(name, _lib.RowsArgs, **a)
        assert getattr(lib, name)(None, None) == bad
        for kw in (dict(tokens=-1), dict(d=-1), dict(picks=0), dict(picks=33), dict(experts=0), dict(tokens=2 ** 30),
                   dict(slots=None), dict(x=None, rows=None)):
            assert rows(**kw) == bad, (name, kw)
        assert rows(dtype=_lib.OZ_F64) == unsupported and rows(tokens=0, slots=None) == ok

    def clip(grads, outs, sizes, types=None, out_types=None, **kw):
        n = len(grads)
        types, out_types = types or [_lib.OZ_F32] * n, out_types or types or [_lib.OZ_F32] * n
        held = ((ctypes.c_void_p * n)(*grads), (ctypes.c_void_p * n)(*outs), (ctypes.c_int64 * n)(*sizes),
                (ctypes.c_int32 * n)(*types), (ctypes.c_int32 * n)(*out_types))
        a = dict(zip(("grads", "outs", "sizes", "dtypes", "out_dtypes"), map(ctypes.addressof, held)), norm=p, workspace=p,
                 workspace_bytes=1 << 30, max_norm=1.0, eps=0.0, tensors=n)
        a.update(kw)
        return call("oz_clip", _lib.ClipArgs, **a)
    assert lib.oz_clip(None, None) == bad
    assert clip([p], [p], [-1]) == bad and clip([p], [None], [4]) == bad and clip([p + 2], [p + 2], [4]) == bad
    assert clip([p], [p], [4], [_lib.OZ_F64]) == unsupported and clip([p], [p], [4], norm=None) == bad
    assert clip([p], [p], [4], workspace_bytes=8) == bad and clip([p], [p], [4], max_norm=-1.0) == bad
    assert clip([p], [p], [4], eps=float("nan")) == bad and clip([p], [p], [4], tensors=-1) == bad
    for grads, outs, sizes in (([512, 512], [512, 512], [4, 4]), ([512, 520], [512, 520], [4, 4]),
                               ([512, 1024], [1024, 512], [4, 4]), ([512], [516], [4]), ([512, 1024], [2048, 520], [4, 4])):
        assert clip(grads, outs, sizes) == bad
        assert "memory" in lib.oz_last_error().decode()
    assert clip([512], [512], [4], [_lib.OZ_F16], [_lib.OZ_F32]) == bad
    assert lib.oz_clip_workspace_bytes(-1) == bad and lib.oz_clip_workspace_bytes(3) > 0
    assert lib.oz_launch_count() == n0
