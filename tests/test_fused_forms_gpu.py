"""Products with bias, activation and residual at sizes of many tiles and of middle ones: tiles of 256 x
256 and 128 x 128 with 16-bit and fp32 results, plain, by vectors and by elements, and contractions that
two and four pairs of CTAs share.  Needs a B200.

Whole numbers whose sums are exact in fp32, so the results have to equal the definition; normal
values for the smooth activations, held to half a unit of the result's type, 1.13 times (the
steepest slope) the sums' bound, (k + 3) 2^-23 of the sum of magnitudes, and 16 2^-24 of the value.
"""

import math

import pytest
import torch

import ozaki_triton_b200 as oz

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
UNIT = {d: torch.finfo(d).eps / 2 for d in (BF16, F16, F32)}
TINY = {BF16: 2.0 ** -134, F16: 2.0 ** -25, F32: 2.0 ** -126}

# four pairs a tile; two; many tiles of odd and of even width; few blocks of contraction
SIZES = [(700, 8192, 1000), (512, 8192, 1272), (580, 6504, 1024), (299, 4632, 3880), (536, 7504, 2688),
         (8687, 160, 2369), (5000, 136, 2003), (5000, 520, 2000), (2501, 264, 3001), (3000, 1000, 3000), (6000, 72, 1000),
         (4099, 72, 1001)]


def whole(g, *shape, most=2):
    return torch.randint(-most, most + 1, shape, generator=g, device=DEV).float()


def off_boundary(t):
    """t's values in rows that start 1 element past the 16-byte boundaries, NaN around them."""
    wide = torch.full((t.shape[0], (t.shape[1] + 15) // 8 * 8), float("nan"), dtype=t.dtype, device=DEV)
    return wide[:, 1:1 + t.shape[1]].copy_(t)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
@pytest.mark.parametrize("rows,k,n", SIZES)
def test_whole_numbers(rows, k, n, dtype):
    g = torch.Generator(device=DEV).manual_seed(rows + k + n)
    x, w = whole(g, rows, k).to(dtype), whole(g, k, n).to(dtype)
    bias, residual = whole(g, n, most=9).to(dtype), whole(g, rows, n, most=9)
    u = x.double() @ w.double()
    full = (u + bias.double()).clamp(min=0) + residual.double()
    for weight in (w, w.t().contiguous().t()):
        for out in (dtype, F32):
            r = residual.to(out)
            assert torch.equal(oz.fused_matmul(x, weight, out_dtype=out), u.to(out))
            assert torch.equal(oz.fused_matmul(x, weight, bias.float(), out_dtype=out), (u + bias.double()).to(out))
            assert torch.equal(oz.fused_matmul(x, weight, residual=off_boundary(r), out_dtype=out),
                               (u + residual.double()).to(out))
            y, pre = oz.fused_matmul(x, weight, bias, activation="relu", residual=r, out_dtype=out, return_pre=True)
            assert torch.equal(y, full.to(out)) and torch.equal(pre, (u + bias.double()).to(dtype))
            y, pre = oz.fused_matmul(x, weight, bias, activation="relu", residual=off_boundary(r), out_dtype=out,
                                     return_pre=True)
            assert torch.equal(y, full.to(out)) and torch.equal(pre, (u + bias.double()).to(dtype))
    assert oz.device_status() == 0


@pytest.mark.parametrize("rows,k,n", SIZES)
def test_smooth_activations(rows, k, n):
    g = torch.Generator(device=DEV).manual_seed(3 * rows + n)
    x = torch.randn(rows, k, generator=g, device=DEV).bfloat16()
    w = (torch.randn(k, n, generator=g, device=DEV) * 3 / math.sqrt(k)).bfloat16()
    bias, residual = torch.randn(n, generator=g, device=DEV).bfloat16(), torch.randn(rows, n, generator=g, device=DEV)
    u = x.double() @ w.double() + bias.double()
    sums = (k + 3) * 2.0 ** -23 * (x.double().abs() @ w.double().abs() + bias.double().abs())
    for name, want in (("gelu", u * 0.5 * torch.erfc(-u / math.sqrt(2))), ("silu", u * torch.sigmoid(u))):
        for out in (BF16, F32):
            r = residual.to(out)
            y, pre = oz.fused_matmul(x, w, bias, activation=name, residual=r, out_dtype=out, return_pre=True)
            added = want + r.double()
            bound = UNIT[out] * added.abs() + 1.13 * sums + 16 * 2.0 ** -24 * want.abs() + 2.0 ** -24 * added.abs() + TINY[out]
            assert bool(((y.double() - added).abs() <= bound).all())
            assert bool(((pre.double() - u).abs() <= UNIT[BF16] * u.abs() + sums + TINY[BF16]).all())
    assert oz.device_status() == 0


@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
@pytest.mark.parametrize("rows,k,n", [(8192, 700, 1000), (8192, 512, 1272), (1000, 3000, 3000), (264, 2501, 3001),
                                      (160, 2369, 8687), (72, 4000, 4001), (2000, 5000, 520)])
def test_gradients_of_whole_numbers(rows, k, n, dtype):
    # dw: both operands stored across the contraction, which is over the rows
    g = torch.Generator(device=DEV).manual_seed(rows + n)
    x, w, dy = (whole(g, *s).to(dtype) for s in ((rows, k), (k, n), (rows, n)))
    pre = whole(g, rows, n).to(dtype)
    for name, u in ((None, None), ("relu", pre)):
        du = dy.double() if u is None else dy.double() * (u.double() > 0)
        want_x, want_w = du @ w.double().t(), x.double().t() @ du
        for weight in (w, w.t().contiguous().t()):
            for to in (dtype, F32):
                dx, dw, db = oz.fused_matmul_backward(dy, x, weight, u, activation=name, bias=True, dw_dtype=to)
                assert torch.equal(dx, want_x.to(dtype)) and torch.equal(dw, want_w.to(to))
                assert torch.equal(db.double(), du.sum(0))
    assert oz.device_status() == 0
