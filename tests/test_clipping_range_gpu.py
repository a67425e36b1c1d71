"""Clipping of gradients far from 1, against 64 bits.  Needs a B200.

Squares are summed in fp32 within 16 bytes (8 terms at most, each addition off by half a unit:
8 2^-24 of the sum, and what falls below fp32's smallest numbers, 2^-27 of it) and in fp64
beyond, so the norm is off by at most 4.5 2^-24 of itself with its own rounding, the factor
by two roundings more and a result by one more and its own.
"""

import math

import pytest
import torch

import ozaki_triton_b200 as oz

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
UNIT = {d: torch.finfo(d).eps / 2 for d in (F32, BF16, F16)}
SMALLEST = {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -24}      # rounded by half of it below the normal ones
NORM_UNITS, FACTOR_UNITS = 5.0, 8.5


def check(grads, max_norm, to=None, eps=0.0):
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    factor = min(1.0, max_norm / (norm + eps)) if norm + eps else 1.0
    want = [g.double() * factor for g in grads]
    outs = None if to is None else [torch.empty_like(g, dtype=to) for g in grads]
    got = oz.clip_gradients(grads, max_norm, eps=eps, out=outs)
    assert abs(got.item() - norm) <= NORM_UNITS * 2.0 ** -24 * norm + 2.0 ** -150
    for o, w in zip(outs or grads, want):
        bound = (UNIT[o.dtype] + FACTOR_UNITS * 2.0 ** -24) * w.abs() + SMALLEST[o.dtype] / 2
        assert bool(((o.double() - w).abs() <= bound * (1 + 1e-6)).all())
    assert oz.device_status() == 0
    return norm


def normal(g, n, scale, dtype):
    return (torch.randn(n, generator=g, device=DEV, dtype=torch.float64) * scale).to(dtype)


@pytest.mark.parametrize("to", [None, F32], ids=["in place", "fp32"])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
@pytest.mark.parametrize("scale", [1e20, 1e30, 1e37, 1e-12, 1e-16, 1e-20, 1e-25, 1e-32])
def test_large_and_small_gradients(scale, dtype, to):
    # whole 16 bytes, rests of them, and a tensor off the 16-byte boundaries
    g = torch.Generator(device=DEV).manual_seed(7)
    for sizes in ([1], [3, 8, 40000], [30011, 5]):
        grads = [normal(g, n, scale, dtype) for n in sizes]
        grads.append(normal(g, 1030, scale, dtype)[3:])
        for share in (0.25, 2.0):
            norm = math.sqrt(sum(float(v.double().square().sum()) for v in grads))
            if 2 * norm < 2 ** 127:
                check([v.clone() for v in grads], share * norm, to)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_magnitudes_side_by_side(dtype):
    g = torch.Generator(device=DEV).manual_seed(8)
    for scales in ([1e30, 1.0, 1e-30], [1e-25, 1e-3], [1e19, 1e18, 1e17], [0.0, 1e-30, 0.0], [1e25, 0.0]):
        grads = [normal(g, 5003, s, dtype) for s in scales]
        grads.append(torch.cat([normal(g, 1, s, dtype) for s in scales for _ in range(3)]))   # within 16 bytes
        check(grads, 1.0, F32)
        check(grads, 1e-3 * max(scales), F32)
        check([v.clone() for v in grads], 1.0)


def test_types_side_by_side():
    g = torch.Generator(device=DEV).manual_seed(9)
    grads = [normal(g, 4001, 1e22, F32), normal(g, 4001, 1e22, BF16), normal(g, 4001, 100.0, F16)]
    check(grads, 1.0, F32)
    check(grads, 1e10, F32)
    check(grads, 1.0, BF16)
    assert check([torch.full((4,), 1e20, device=DEV)], 1.0) == pytest.approx(2e20)


def test_norms_past_fp32():
    inf = float("inf")
    for most in (1.0, 1e30):
        grads = [torch.full((4,), 3e38, device=DEV), torch.ones(5, device=DEV)]          # norm 6e38
        assert oz.clip_gradients(grads, most) == inf and not grads[0].any() and not grads[1].any()
        grads = [torch.tensor([1.0, inf], device=DEV), torch.ones(5, device=DEV)]
        assert oz.clip_gradients(grads, most) == inf and grads[0][0] == 0 and grads[0][1].isnan() and not grads[1].any()
    for value in (float("nan"), -float("nan")):
        for others in (0.0, 1.0, 1e30, 1e-30):
            grads = [torch.full((100,), others, device=DEV), torch.full((16,), value, device=DEV).bfloat16()]
            assert oz.clip_gradients(grads, 1.0).isnan() and grads[0].isnan().all()
