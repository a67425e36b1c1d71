"""Argument checks of the expert-layer operators, and the 4-bit layout; no GPU needed."""

import ctypes

import pytest
import torch

import ozaki_triton_b200 as oz
from ozaki_triton_b200 import _lib

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def args(**kw):
    a = dict(x=torch.zeros(6, 64, dtype=F16), w=torch.zeros(2, 64, 32, dtype=F16),
             offsets=torch.tensor([0, 2, 6], dtype=torch.int32))
    a.update(kw)
    return a["x"], a["w"], a["offsets"]


@pytest.mark.parametrize("kw", [
    dict(x=torch.zeros(6, 64, dtype=F32), w=torch.zeros(2, 64, 32, dtype=F32)),
    dict(x=torch.zeros(6, 64, dtype=BF16)),
    dict(x=torch.zeros(6, 63, dtype=F16)),
    dict(x=torch.zeros(1, 6, 64, dtype=F16)),
    dict(w=torch.zeros(64, 32, dtype=F16)),
    dict(w=torch.zeros(0, 64, 32, dtype=F16)),
    dict(offsets=torch.tensor([0, 6], dtype=torch.int32)),
    dict(offsets=torch.tensor([[0, 2, 6]], dtype=torch.int32)),
    dict(offsets=torch.tensor([0.0, 2.0, 6.0])),
    dict(offsets=torch.tensor([0, 9, 2, 9, 6, 9], dtype=torch.int32)[::2]),
])
def test_grouped_refuses(kw):
    with pytest.raises(AssertionError):
        oz.grouped_matmul(*args(**kw))


def test_grouped_refuses_other_results_and_hosts():
    with pytest.raises(ValueError):
        oz.grouped_matmul(*args())
    x, w, offsets = args()
    with pytest.raises(AssertionError):
        oz.grouped_matmul_backward(torch.zeros(5, 32, dtype=F16), x, w, offsets)
    with pytest.raises(ValueError):
        oz.grouped_matmul_backward(torch.zeros(6, 32, dtype=F16), x, w, offsets)


def w4(**kw):
    a = dict(x=torch.zeros(3, 128, dtype=F16), packed=torch.zeros(10, 64, dtype=torch.uint8),
             scales=torch.zeros(10, 4, dtype=F16), zeros=None, offsets=None)
    a.update(kw)
    return oz.matmul_w4(a["x"], a["packed"], a["scales"], a["zeros"], offsets=a["offsets"])


@pytest.mark.parametrize("kw", [
    dict(x=torch.zeros(3, 128)),
    dict(x=torch.zeros(3, 130, dtype=F16)),
    dict(x=torch.zeros(128, dtype=F16)),
    dict(packed=torch.zeros(10, 64, dtype=torch.int8)),
    dict(packed=torch.zeros(1, 10, 64, dtype=torch.uint8)),
    dict(scales=torch.zeros(10, 3, dtype=F16)),
    dict(scales=torch.zeros(10, 8, dtype=F16)),
    dict(scales=torch.zeros(10, 0, dtype=F16)),
    dict(scales=torch.zeros(9, 4, dtype=F16)),
    dict(scales=torch.zeros(10, 4, dtype=torch.float64)),
    dict(zeros=torch.zeros(10, 4, dtype=F16)),
    dict(zeros=torch.zeros(10, 2, dtype=torch.uint8)),
    dict(offsets=torch.tensor([0, 3])),
])
def test_w4_refuses(kw):
    with pytest.raises(AssertionError):
        w4(**kw)


def test_w4_refuses_host_tensors():
    with pytest.raises(ValueError):
        w4()


@pytest.mark.parametrize("kw", [
    dict(g=torch.zeros(4)), dict(g=torch.zeros(4, 4, dtype=torch.float64)), dict(steps=0), dict(eps=-1.0),
    dict(num_splits=3), dict(coefficients=(1.0, 2.0)), dict(coefficients=[(1.0, 2.0, 3.0)] * 4),
])
def test_orthogonalize_refuses(kw):
    a = dict(g=torch.zeros(4, 4))
    a.update(kw)
    with pytest.raises(AssertionError):
        oz.orthogonalize(**a)


def test_orthogonalize_refuses_host_tensors():
    with pytest.raises(ValueError):
        oz.orthogonalize(torch.zeros(4, 4))


def test_library_entries_validate_without_a_launch():
    lib = _lib.load()
    p = ctypes.c_void_p(256)      # never dereferenced: validation fails first
    n0 = lib.oz_launch_count()

    def grouped(dtype=_lib.OZ_F16, out=_lib.OZ_F16, groups=2, rows=4, k=8, n=8, x=p, y=p, ldy=8):
        return lib.oz_grouped_matmul(_lib.GroupedArgs(x, p, p, y, rows, k, n, k, k * n, n, 1, ldy, None, 0, groups,
                                                      0, dtype, out), None)
    assert lib.oz_grouped_matmul(None, None) == _lib.OZ_ERR_INVALID
    assert grouped(dtype=_lib.OZ_F32) == _lib.OZ_ERR_UNSUPPORTED
    assert grouped(out=_lib.OZ_BF16) == _lib.OZ_ERR_UNSUPPORTED
    assert grouped(groups=0) == _lib.OZ_ERR_INVALID
    assert grouped(rows=-1) == _lib.OZ_ERR_INVALID
    assert grouped(k=2 ** 31) == _lib.OZ_ERR_INVALID
    assert grouped(ldy=4) == _lib.OZ_ERR_INVALID
    assert grouped(x=None) == _lib.OZ_ERR_INVALID
    assert grouped(y=None) == _lib.OZ_ERR_INVALID
    assert grouped(rows=0, y=None) == _lib.OZ_OK
    assert grouped(x=ctypes.c_void_p(264)) == _lib.OZ_ERR_INVALID
    assert grouped(k=12) == _lib.OZ_ERR_INVALID          # rows 24 bytes apart, and no workspace
    assert "workspace" in lib.oz_last_error().decode()

    def wgrad(dtype=_lib.OZ_F16, groups=2, dw=p, k=8):
        return lib.oz_grouped_wgrad(_lib.GroupedWgradArgs(p, p, p, dw, 4, k, 8, 8, 8, None, 0, groups, 0, dtype,
                                                          dtype), None)
    assert lib.oz_grouped_wgrad(None, None) == _lib.OZ_ERR_INVALID
    assert wgrad(dtype=_lib.OZ_I8) == _lib.OZ_ERR_UNSUPPORTED
    assert wgrad(groups=-1) == _lib.OZ_ERR_INVALID
    assert wgrad(dw=None) == _lib.OZ_ERR_INVALID
    assert wgrad(k=0, dw=None) == _lib.OZ_OK

    def four(dtype=_lib.OZ_F16, scale=_lib.OZ_F16, experts=1, group=32, k=64, offsets=None, y=p, rows=1):
        return lib.oz_matmul_w4(_lib.W4Args(p, p, p, None, offsets, y, rows, k, 8, k, 4 * k, k // 2, 8 * 2, 2, 8,
                                            experts, group, 0, dtype, scale, dtype), None)
    assert lib.oz_matmul_w4(None, None) == _lib.OZ_ERR_INVALID
    assert four(dtype=_lib.OZ_F64) == _lib.OZ_ERR_UNSUPPORTED
    assert four(scale=_lib.OZ_I8) == _lib.OZ_ERR_UNSUPPORTED
    assert four(group=16) == _lib.OZ_ERR_INVALID
    assert four(group=48) == _lib.OZ_ERR_INVALID
    assert four(k=96, group=64) == _lib.OZ_ERR_INVALID
    assert four(experts=2) == _lib.OZ_ERR_INVALID
    assert four(y=None) == _lib.OZ_ERR_INVALID
    assert four(rows=0, y=None) == _lib.OZ_OK

    abc = (ctypes.c_double * 3)(1.5, -0.5, 0.0)

    def ortho(dtype=_lib.OZ_F32, batch=1, m=512, n=512, steps=1, c=abc, eps=0.0, splits=2, ws=p, ws_bytes=1 << 30):
        return lib.oz_orthogonalize(p, dtype, batch, m, n, 16, 4, 1, steps, c, eps, splits, p, ws, ws_bytes, None)
    assert ortho(dtype=_lib.OZ_F64) == _lib.OZ_ERR_UNSUPPORTED
    assert ortho(m=-1) == _lib.OZ_ERR_INVALID
    assert ortho(steps=0) == _lib.OZ_ERR_INVALID
    assert ortho(c=None) == _lib.OZ_ERR_INVALID
    assert ortho(c=(ctypes.c_double * 3)(1.5, float("inf"), 0.0)) == _lib.OZ_ERR_INVALID
    assert ortho(eps=-1.0) == _lib.OZ_ERR_INVALID
    assert ortho(eps=float("nan")) == _lib.OZ_ERR_INVALID
    assert ortho(splits=3) == _lib.OZ_ERR_INVALID
    assert ortho(ws=None) == _lib.OZ_ERR_INVALID
    assert ortho(ws=ctypes.c_void_p(128)) == _lib.OZ_ERR_INVALID
    assert ortho(ws_bytes=10) == _lib.OZ_ERR_INVALID
    assert ortho(n=0) == _lib.OZ_OK
    need = lib.oz_orthogonalize_workspace_bytes
    assert need(_lib.OZ_F32, 1, 4, 4, 1, 0) == _lib.OZ_ERR_INVALID
    assert need(_lib.OZ_F32, 1, 512, 512, 0, 1) == _lib.OZ_ERR_INVALID
    assert need(_lib.OZ_F32, 2, 640, 320, 5, 2) > need(_lib.OZ_F32, 2, 640, 320, 5, 1) > 0
    assert need(_lib.OZ_F32, 2, 64, 32, 5, 2) == 0       # small: kept on chip
    assert lib.oz_launch_count() == n0


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantized_weights_are_within_half_a_step(group, symmetric):
    g = torch.Generator().manual_seed(group)
    w = torch.randn(2, 128, 24, generator=g)
    w[0, :group, 3] = 0
    packed, scales, zeros = oz.quantize_w4(w, group, symmetric=symmetric)
    assert packed.shape == (2, 24, 64) and packed.dtype == torch.uint8
    assert scales.shape == (2, 24, 128 // group) and (zeros is None) == symmetric
    q = torch.stack([packed & 15, packed >> 4], -1).flatten(-2).float()
    z = 8.0 if symmetric else zeros.float().repeat_interleave(group, -1)
    s = scales.repeat_interleave(group, -1)
    back = ((q - z) * s).transpose(-1, -2)
    # half a step; a step more at the end that 0..15 cuts off (q - 8 <= 7), and for the rounded zero point
    assert bool(((back - w).abs() <= 1.001 * s.transpose(-1, -2)).all())
    assert bool(((back - w).abs() <= 0.501 * s.transpose(-1, -2)).float().mean() > 0.9)
    assert not back[0, :group, 3].any()
    with pytest.raises(AssertionError):
        oz.quantize_w4(w, 96)
