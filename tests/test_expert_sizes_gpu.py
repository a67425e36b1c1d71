"""Expert-layer operators on tensors of more than 2^31 elements: what lies past
32-bit offsets is read and written where it is.  Needs a B200 (up to 40 GB).

Nearly all of each tensor is zero; small whole numbers stand at its start and end,
whose products are exact.
"""

import pytest
import torch

import ozaki_triton_b200 as oz

pytestmark = pytest.mark.gpu

DEV = "cuda"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def memory():
    yield
    torch.cuda.empty_cache()


def whole(seed, *shape, dtype=BF16):
    return torch.randint(-2, 3, shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def ends(seed, *shape, first=3, dtype=BF16):
    """Zeros but for the first and last `first` of the leading dimension."""
    t = torch.zeros(*shape, dtype=dtype, device=DEV)
    t[:first], t[-first:] = whole(seed, first, *shape[1:], dtype=dtype), whole(seed + 1, first, *shape[1:], dtype=dtype)
    return t


def offsets_of(*bounds):
    return torch.tensor(bounds, device=DEV)


ROWS = 2 ** 31 // 4096 + 300


def test_many_rows():
    x, w = ends(1, ROWS, 4096), whole(3, 2, 4096, 64)
    offsets = offsets_of(0, 2, ROWS - 1)                   # the last row belongs to no one
    y = oz.grouped_matmul(x, w, offsets, out_dtype=F32)
    assert torch.equal(y[:2].double(), x[:2].double() @ w[0].double())
    assert torch.equal(y[-3:-1].double(), x[-3:-1].double() @ w[1].double()) and not y[-1].any()
    dy = ends(5, ROWS, 64)
    dx, dw = oz.grouped_matmul_backward(dy, x, w, offsets, dw_dtype=F32)
    assert torch.equal(dx[-3:-1], (dy[-3:-1].double() @ w[1].double().t()).to(BF16)) and not dx[-1].any()
    want = x[2:3].double().t() @ dy[2:3].double() + x[-3:-1].double().t() @ dy[-3:-1].double()
    assert torch.equal(dw[1].double(), want)


def test_many_rows_off_the_16_byte_boundaries():
    rows = 2 ** 31 // 4095 + 300
    x, w = ends(7, rows, 4095), whole(9, 1, 4095, 40)
    y = oz.grouped_matmul(x, w, offsets_of(0, rows), out_dtype=F32)
    assert torch.equal(y[-3:].double(), x[-3:].double() @ w[0].double())
    assert torch.equal(y[:3].double(), x[:3].double() @ w[0].double())


def test_many_results():
    x, w = ends(11, ROWS, 72), whole(13, 1, 72, 4096)
    y = oz.grouped_matmul(x, w, offsets_of(0, ROWS))
    for rows in (slice(0, 3), slice(-3, None)):
        assert torch.equal(y[rows].double(), x[rows].double() @ w[0].double())
    assert not y[3:-3:5000].any()


def test_many_weights():
    e = 2 ** 31 // 4096 ** 2 + 4
    w, x, dy = ends(15, e, 4096, 4096, first=1), whole(17, 9, 4096), whole(19, 9, 4096)
    offsets = torch.full((e + 1,), 4, device=DEV)          # 4 rows of the first, 5 of the last
    offsets[0], offsets[-1] = 0, 9
    y = oz.grouped_matmul(x, w, offsets, out_dtype=F32)
    assert torch.equal(y[:4].double(), x[:4].double() @ w[0].double())
    assert torch.equal(y[4:].double(), x[4:].double() @ w[-1].double())
    dx, dw = oz.grouped_matmul_backward(dy, x, w, offsets, dw_dtype=F32)
    assert torch.equal(dx[4:], (dy[4:].double() @ w[-1].double().t()).to(BF16))
    assert torch.equal(dw[-1].double(), x[4:].double().t() @ dy[4:].double()) and not dw[1:-1:20].any()


@pytest.mark.parametrize("experts,n,k", [(260, 4096, 4096), (1, 2 ** 20 + 5, 4160)])
def test_many_4_bit_weights(experts, n, k):
    g = torch.Generator(device=DEV).manual_seed(n)
    assert experts * n * k // 2 > 2 ** 31
    packed = torch.full((experts, n, k // 2), 0x88, dtype=torch.uint8, device=DEV)
    packed[-1, -40:] = torch.randint(0, 256, (40, k // 2), generator=g, device=DEV, dtype=torch.uint8)
    scales = torch.ones(experts, n, k // 32, dtype=F16, device=DEV)
    scales[-1, -40:] = 2.0 ** torch.randint(-2, 3, (40, k // 32), generator=g, device=DEV).half()
    x = whole(21, 5, k, dtype=F16)
    if experts == 1:
        y = oz.matmul_w4(x, packed[0], scales[0], out_dtype=F32)
    else:
        offsets = torch.zeros(experts + 1, dtype=torch.int64, device=DEV)
        offsets[-1] = 5
        y = oz.matmul_w4(x, packed, scales, offsets=offsets, out_dtype=F32)
    p = packed[-1, -40:]
    w = (torch.stack([p % 16, p // 16], -1).flatten(-2).double() - 8) * scales[-1, -40:].double().repeat_interleave(32, -1)
    assert torch.equal(y[:, -40:].double(), x.double() @ w.t()) and not y[:, :-40].any()


@pytest.mark.parametrize("shape", [(2 ** 31 // 2048 ** 2 + 2, 2048, 2048), (2 ** 31 // (600 * 200) + 2, 600, 200)], ids=str)
def test_many_matrices(shape):
    g = torch.zeros(shape, dtype=BF16, device=DEV)
    g[-1] = torch.randn(shape[1:], generator=torch.Generator(device=DEV).manual_seed(23), device=DEV)
    got = oz.orthogonalize(g, steps=3, num_splits=1)
    x = g[-1].double()
    x = x / x.norm()
    for _ in range(3):
        s = x @ x.t() if shape[1] <= shape[2] else x.t() @ x
        p = -4.7750 * s + 2.0315 * s @ s
        x = 3.4445 * x + (p @ x if shape[1] <= shape[2] else x @ p)
    # one slice's 2^-12 in each of 9 products, as much as 3.4445^2 times in the first, and bf16's half unit
    assert ((got[-1].double() - x).norm() / x.norm()).item() <= 2.0 ** -9 + 9 * 12 * 2.0 ** -12
    assert not got[:-1:10].any() and not got[-2].any()


def test_a_stride_past_32_bits():
    store = torch.zeros(2, 2 ** 31 + 8, dtype=BF16, device=DEV)
    g = torch.randn(200, 300, generator=torch.Generator(device=DEV).manual_seed(25), device=DEV).bfloat16()
    view = store.as_strided((2, 200, 300), (2 ** 31 + 8, 300, 1))
    view[1] = g
    got = oz.orthogonalize(view)
    assert not got[0].any()
    want = oz.orthogonalize(g)
    # the same matrix alone: other tiles and so other fp32 sums, before one rounding to bf16
    assert ((got[1].double() - want.double()).norm() / want.double().norm()).item() <= 2.0 ** -9
