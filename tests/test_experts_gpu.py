"""Ragged expert products, their gradients and 4-bit products against their
definitions in 64 bits.  Needs a B200.

Two kinds of inputs.  Small whole numbers, whose products and sums are exact
in fp32: the fp32 result then has to equal the definition exactly, so a wrong
index, a lost or doubled row or column cannot hide in a tolerance.  And normal
values, held to half a unit of the result's type (rounded once) plus the sum's
own bound: (terms + 2) * 2^-23 of the sum of the products' magnitudes (each
fp32 addition, rounded or cut, is off by at most 2^-23 of its result).
"""

import itertools

import pytest
import torch

import ozaki_triton_b200 as oz

pytestmark = pytest.mark.gpu

DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16]
UNIT = {d: torch.finfo(d).eps / 2 for d in (*DTYPES, torch.float32)}


def whole(g, *shape, most=3):
    return torch.randint(-most, most + 1, shape, generator=g, device=DEV).float()


def generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def offsets_of(sizes, first=0, dtype=torch.int32):
    return torch.tensor([first, *(first + s for s in itertools.accumulate(sizes))], dtype=dtype, device=DEV)


def define(x, w, bounds, rows=None):
    """(y, sum of magnitudes) of the product in 64 bits."""
    x, w = x.double(), w.double()
    y = torch.zeros(x.shape[0], w.shape[2], dtype=torch.float64, device=x.device)
    size = torch.zeros_like(y)
    for e in range(w.shape[0]):
        low, high = bounds[e], bounds[e + 1]
        y[low:high] = x[low:high] @ w[e]
        size[low:high] = x[low:high].abs() @ w[e].abs()
    return y, size


def define_dw(x, dy, bounds):
    x, dy = x.double(), dy.double()
    parts = [(x[a:b], dy[a:b]) for a, b in zip(bounds, bounds[1:])]
    return (torch.stack([u.t() @ v for u, v in parts]),
            torch.stack([u.abs().t() @ v.abs() for u, v in parts]))


def near(got, want, size, terms, dtype):
    assert got.dtype == dtype and got.shape == want.shape
    bound = UNIT[dtype] * want.abs() + (terms + 2) * 2.0 ** -23 * size
    if dtype == torch.float16:
        bound = bound + 2.0 ** -25        # half the smallest subnormal
    off = (got.double() - want).abs() - bound
    assert bool((off <= 0).all()), f"off by {off.max().item():.3g} more than the bound"


# sizes of the groups; rows before and after them; k; n
RAGGED = [
    ([1], 0, 0, 64, 64),
    ([1, 0, 2], 0, 0, 32, 96),
    ([5, 0, 0, 300, 1, 127, 128, 129], 0, 0, 192, 136),
    ([64, 256, 257, 511], 0, 0, 128, 512),
    ([3, 2, 40], 7, 9, 72, 200),
    ([0, 0, 0], 4, 4, 64, 64),
    ([17, 33], 0, 0, 1, 3),
    ([100, 29], 0, 0, 129, 77),
    ([600, 700], 0, 3, 1000, 1411),
    ([2] * 70, 0, 0, 64, 256),
    ([40] * 40, 0, 0, 256, 320),
    ([1100, 900], 0, 0, 520, 776),
    ([100] * 100, 0, 0, 200, 100),
    ([900, 1100, 700], 3, 5, 200, 1000),
    ([1300, 0, 901], 1, 0, 264, 1003),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("sizes,before,after,k,n", RAGGED)
def test_grouped_products_of_whole_numbers_are_exact(sizes, before, after, k, n, dtype):
    g = generator(k + n)
    rows = before + sum(sizes) + after
    x = whole(g, rows, k).to(dtype)
    w = whole(g, len(sizes), k, n).to(dtype)
    dy = whole(g, rows, n).to(dtype)
    offsets = offsets_of(sizes, before)
    bounds = offsets.tolist()
    y = oz.grouped_matmul(x, w, offsets, out_dtype=torch.float32)
    assert torch.equal(y.double(), define(x, w, bounds)[0])
    # the weights in the other order give the same
    wt = w.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(oz.grouped_matmul(x, wt, offsets, out_dtype=torch.float32), y)
    dx, dw = oz.grouped_matmul_backward(dy, x, w, offsets, dw_dtype=torch.float32)
    assert torch.equal(dw.double(), define_dw(x, dy, bounds)[0])
    want = define(dy, w.transpose(1, 2), bounds)[0]
    near(dx, want, torch.zeros_like(want), 0, dtype)
    assert oz.device_status() == 0


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("sizes,before,after,k,n", RAGGED[2:5] + RAGGED[7:9] + RAGGED[11:])
def test_grouped_products_of_normal_values(sizes, before, after, k, n, dtype):
    g = generator(k * n)
    rows = before + sum(sizes) + after
    x = torch.randn(rows, k, generator=g, device=DEV).to(dtype)
    w = (torch.randn(len(sizes), k, n, generator=g, device=DEV) / k ** 0.5).to(dtype)
    dy = torch.randn(rows, n, generator=g, device=DEV).to(dtype)
    offsets = offsets_of(sizes, before, torch.int64)
    bounds = offsets.tolist()
    for out in (dtype, torch.float32):
        near(oz.grouped_matmul(x, w, offsets, out_dtype=out), *define(x, w, bounds), k, out)
        dx, dw = oz.grouped_matmul_backward(dy, x, w, offsets, dw_dtype=out)
        near(dx, *define(dy, w.transpose(1, 2), bounds), n, dtype)
        near(dw, *define_dw(x, dy, bounds), max(sizes), out)


def test_values_outside_a_group_never_reach_it():
    # NaN and infinities in rows of no group, and in the next group's rows
    g = generator(3)
    x, w, dy = whole(g, 300, 96), whole(g, 3, 96, 160), whole(g, 300, 160)
    offsets = offsets_of([70, 37, 101], 50)
    bounds = offsets.tolist()
    for rows in (slice(0, 50), slice(258, 300), slice(120, 157)):
        x[rows], dy[rows] = float("nan"), float("inf")
    x, w, dy = x.bfloat16(), w.bfloat16(), dy.bfloat16()
    y = oz.grouped_matmul(x, w, offsets, out_dtype=torch.float32)
    dx, dw = oz.grouped_matmul_backward(dy, x, w, offsets, dw_dtype=torch.float32)
    assert not y[:50].any() and not y[258:].any() and not dx[:50].any() and not dx[258:].any()
    for low, high in ((50, 120), (157, 258)):
        e = bounds.index(low)
        assert torch.equal(y[low:high].double(), x[low:high].double() @ w[e].double())
        assert torch.equal(dw[e].double(), x[low:high].double().t() @ dy[low:high].double())
    assert bool(torch.isnan(y[120:157]).all()) and bool(torch.isnan(dw[1]).all())


@pytest.mark.parametrize("layout", ["columns of a wider tensor", "odd address", "transposed", "expanded",
                                    "every other row"])
def test_grouped_products_take_any_layout(layout):
    g = generator(11)
    sizes, k, n = [130, 0, 70], 88, 104
    offsets = offsets_of(sizes)

    def laid(*shape):
        if layout == "columns of a wider tensor":
            return whole(g, *shape[:-1], shape[-1] + 24).half()[..., 8:8 + shape[-1]]
        if layout == "odd address":
            v = whole(g, 1 + torch.Size(shape).numel()).half()
            return v[1:].view(shape)
        if layout == "transposed":
            return whole(g, *shape[:-2], shape[-1], shape[-2]).half().transpose(-1, -2)
        if layout == "expanded":
            return whole(g, *shape[:-2], 1, shape[-1]).half().expand(shape)
        return whole(g, *shape[:-2], 2 * shape[-2], shape[-1]).half()[..., ::2, :]

    x, w, dy = laid(200, k), laid(3, k, n), laid(200, n)
    y = oz.grouped_matmul(x, w, offsets, out_dtype=torch.float32)
    assert torch.equal(y.double(), define(x, w, offsets.tolist())[0])
    dx, dw = oz.grouped_matmul_backward(dy, x, w, offsets, dw_dtype=torch.float32)
    assert torch.equal(dw.double(), define_dw(x, dy, offsets.tolist())[0])
    want = define(dy, w.transpose(1, 2), offsets.tolist())[0]
    near(dx, want, torch.zeros_like(want), 0, torch.float16)


def test_grouped_product_without_rows_or_columns():
    w = torch.ones(2, 16, 24, dtype=torch.float16, device=DEV)
    none = torch.zeros(3, dtype=torch.int32, device=DEV)
    x = torch.ones(0, 16, dtype=torch.float16, device=DEV)
    assert oz.grouped_matmul(x, w, none).shape == (0, 24)
    dx, dw = oz.grouped_matmul_backward(torch.ones(0, 24, dtype=torch.float16, device=DEV), x, w, none)
    assert dx.shape == (0, 16) and dw.shape == (2, 16, 24) and not dw.any()
    x = torch.ones(5, 16, dtype=torch.float16, device=DEV)
    assert oz.grouped_matmul(x, w[..., :0], none).shape == (5, 0)
    y = oz.grouped_matmul(x[:, :0], w[:, :0], offsets_of([2, 3]))
    assert y.shape == (5, 24) and not y.any()


def test_wrong_offsets_stay_inside_the_tensors():
    # clamped to [0, rows]: values beyond are as if they were the ends
    g = generator(5)
    x, w = whole(g, 40, 64).half(), whole(g, 2, 64, 72).half()
    y = oz.grouped_matmul(x, w, torch.tensor([-5, 13, 4000], device=DEV), out_dtype=torch.float32)
    assert torch.equal(y.double(), define(x, w, [0, 13, 40])[0])
    dx, dw = oz.grouped_matmul_backward(y.half(), x, w, torch.tensor([-5, 13, 4000], device=DEV),
                                        dw_dtype=torch.float32)
    assert torch.equal(dw.double(), define_dw(x, y.half(), [0, 13, 40])[0])


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_autograd_gives_the_gradients_of_the_formula_and_of_differences(dtype):
    g = generator(7)
    sizes, k, n = [9, 0, 23], 40, 48
    offsets = offsets_of(sizes, 1)
    x = whole(g, 34, k, most=2).to(dtype).requires_grad_()
    w = whole(g, 3, k, n, most=2).to(dtype).requires_grad_()
    dy = whole(g, 34, n, most=2).to(dtype)
    y = oz.grouped_matmul(x, w, offsets, out_dtype=torch.float32)
    y.backward(dy.float())
    dx, dw = oz.grouped_matmul_backward(dy, x.detach(), w.detach(), offsets)
    assert torch.equal(x.grad, dx) and torch.equal(w.grad, dw)
    # y is linear in x and in w: a unit step's difference is the derivative, exactly
    with torch.no_grad():
        base = (y * dy.float()).sum()
        for i, j in ((0, 3), (1, 0), (20, 39), (33, 7)):
            x2 = x.detach().clone()
            x2[i, j] += 1
            diff = (oz.grouped_matmul(x2, w, offsets, out_dtype=torch.float32) * dy.float()).sum() - base
            assert diff.item() == dx[i, j].item()
        for e, i, j in ((0, 0, 0), (1, 5, 5), (2, 39, 47)):
            w2 = w.detach().clone()
            w2[e, i, j] += 1
            diff = (oz.grouped_matmul(x, w2, offsets, out_dtype=torch.float32) * dy.float()).sum() - base
            assert diff.item() == dw[e, i, j].item()


def test_grouped_products_follow_the_current_stream():
    g = generator(13)
    x, w, offsets = whole(g, 512, 256).half(), whole(g, 4, 256, 256).half(), offsets_of([100, 200, 12, 200])
    want = oz.grouped_matmul(x, w, offsets)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    late = torch.empty_like(x)
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        late.copy_(x)
        y = oz.grouped_matmul(late, w, offsets)
    side.synchronize()
    assert torch.equal(y, want)


# ------------------------------------------------------------------ 4 bits
def four_bits(g, lead, n, k, group, zeros, exact):
    packed = torch.randint(0, 256, (*lead, n, k // 2), generator=g, device=DEV, dtype=torch.uint8)
    if exact:
        scales = 2.0 ** torch.randint(-2, 3, (*lead, n, k // group), generator=g, device=DEV)
    else:
        scales = 0.5 + torch.rand(*lead, n, k // group, generator=g, device=DEV)
    z = torch.randint(0, 16, scales.shape, generator=g, device=DEV, dtype=torch.uint8) if zeros else None
    return packed, scales, z


def weights(packed, scales, zeros):
    """(K, N) weights in 64 bits, stacked."""
    q = torch.stack([packed % 16, packed // 16], -1).flatten(-2).double()
    group = q.shape[-1] // scales.shape[-1]
    z = 8.0 if zeros is None else zeros.double().repeat_interleave(group, -1)
    return ((q - z) * scales.double().repeat_interleave(group, -1)).transpose(-1, -2)


W4 = [(1, 32, 1, 32), (1, 256, 64, 32), (2, 64, 7, 64), (3, 4256, 517, 32), (8, 1024, 129, 128), (9, 2048, 256, 128),
      (1, 4096, 300, 256), (17, 96, 1000, 96), (40, 384, 33, 192), (5, 16384, 24, 128), (1, 8192, 2048, 64),
      (4, 1024, 20000, 64), (4, 1024, 20000, 128), (2, 1024, 20011, 32), (12, 320, 20000, 64), (20, 256, 9000, 128)]


@pytest.mark.parametrize("zeros", [False, True], ids=["symmetric", "zeros"])
@pytest.mark.parametrize("t,k,n,group", W4)
def test_w4_products(t, k, n, group, zeros):
    g = generator(t * k + n)
    for dtype, scale_dtype in itertools.product(DTYPES, (None, torch.float32)):
        scale_dtype = scale_dtype or dtype
        packed, scales, z = four_bits(g, (), n, k, group, zeros, True)
        x = whole(g, t, k, most=2).to(dtype)
        y = oz.matmul_w4(x, packed, scales.to(scale_dtype), z, out_dtype=torch.float32)
        w = weights(packed, scales, z)
        assert torch.equal(y.double(), x.double() @ w)
        packed, scales, z = four_bits(g, (), n, k, group, zeros, False)
        scales = scales.to(scale_dtype)
        w = weights(packed, scales, z)
        x = (torch.randn(t, k, generator=g, device=DEV) / k ** 0.5).to(dtype)
        near(oz.matmul_w4(x, packed, scales, z), x.double() @ w, x.double().abs() @ w.abs(), k, dtype)
    assert oz.device_status() == 0


@pytest.mark.parametrize("sizes,before,after", [([1], 0, 0), ([0, 1, 0, 2, 8, 9, 0], 0, 0), ([3, 0, 4], 2, 3),
                                                ([1] * 50, 0, 0), ([0, 0], 1, 1), ([70, 1, 25], 0, 0)])
@pytest.mark.parametrize("group", [32, 128])
def test_w4_products_of_experts(sizes, before, after, group):
    g = generator(len(sizes))
    k, n, e = 512, 200, len(sizes)
    packed, scales, z = four_bits(g, (e,), n, k, group, True, True)
    x = whole(g, before + sum(sizes) + after, k, most=2).bfloat16()
    for wide in (torch.int32, torch.int64):
        offsets = offsets_of(sizes, before, wide)
        y = oz.matmul_w4(x, packed, scales, z, offsets=offsets, out_dtype=torch.float32)
        assert torch.equal(y.double(), define(x, weights(packed, scales, z), offsets.tolist())[0])


def test_w4_layouts_and_wrong_offsets():
    g = generator(23)
    packed, scales, z = four_bits(g, (2,), 72, 256, 64, True, True)
    w = weights(packed, scales, z)
    x = whole(g, 2 * 11, 264, most=2).half()[::2, 8:]
    y = oz.matmul_w4(x, packed[0], scales[0], z[0], out_dtype=torch.float32)
    assert torch.equal(y.double(), x.double() @ w[0])
    odd = torch.empty(packed[0].numel() + 1, dtype=torch.uint8, device=DEV)[1:].view(packed[0].shape)
    odd.copy_(packed[0])
    assert torch.equal(oz.matmul_w4(x, odd, scales[0], z[0], out_dtype=torch.float32), y)
    x1 = whole(g, 1 + 3 * 256, most=2).half()[1:].view(3, 256)
    y = oz.matmul_w4(x1, packed[1].t().contiguous().t(), scales[1], z[1], out_dtype=torch.float32)
    assert torch.equal(y.double(), x1.double() @ w[1])
    y = oz.matmul_w4(x, packed, scales, z, offsets=torch.tensor([-3, 4, 99], device=DEV), out_dtype=torch.float32)
    assert torch.equal(y.double(), define(x, w, [0, 4, 11])[0])
    assert oz.matmul_w4(x[:0], packed[0], scales[0]).shape == (0, 72)


def test_w4_rows_do_not_touch_each_other():
    # an infinity or NaN of one row stays in that row
    g = generator(29)
    packed, scales, _ = four_bits(g, (), 40, 128, 32, False, True)
    x = whole(g, 6, 128, most=2).half()
    want = oz.matmul_w4(x, packed, scales, out_dtype=torch.float32)
    x[2, 5], x[4, 77] = float("nan"), float("inf")
    got = oz.matmul_w4(x, packed, scales, out_dtype=torch.float32)
    for r in (0, 1, 3, 5):
        assert torch.equal(got[r], want[r])
    assert bool(torch.isnan(got[2]).all()) and not bool(torch.isfinite(got[4]).any())
