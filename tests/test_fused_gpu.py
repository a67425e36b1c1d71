"""Products with bias, activation and residual, and their gradients, against their
definitions in 64 bits.  Needs a B200.

Small whole numbers first: their products and sums are exact in fp32, so without
a smooth activation a fp32 result has to equal the definition, and a lost or
doubled element cannot hide in a tolerance.  Normal values are held to half a
unit of the result's type plus the sum's own bound, (terms + 2) 2^-23 of the
sum of the products' magnitudes (an fp32 addition, rounded or cut off, is off
by at most 2^-23 of its result); activations are off by a few fp32 units (16
2^-24 of their value) beside what their argument's error makes, at most 1.13
times it (the steepest slope, gelu's).
"""

import math

import pytest
import torch

import ozaki_triton_b200 as oz

pytestmark = pytest.mark.gpu

DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16]
UNIT = {d: torch.finfo(d).eps / 2 for d in (*DTYPES, torch.float32)}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -126}
ACTS = [None, "relu", "gelu", "silu"]


def generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def whole(g, *shape, most=3):
    return torch.randint(-most, most + 1, shape, generator=g, device=DEV).float()


def normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def phi(u):
    return 0.5 * torch.erfc(-u / math.sqrt(2))


def act(u, name):
    return {None: lambda: u, "relu": lambda: u.clamp(min=0), "gelu": lambda: u * phi(u),
            "silu": lambda: u * torch.sigmoid(u)}[name]()


def slope(u, name):
    if name == "relu":
        return (u > 0).double()
    if name == "gelu":
        return phi(u) + u * torch.exp(-u * u / 2) / math.sqrt(2 * math.pi)
    if name == "silu":
        return torch.sigmoid(u) * (1 + u * torch.sigmoid(-u))
    return torch.ones_like(u)


def within(got, want, bound, dtype):
    assert got.dtype == dtype and got.shape == want.shape
    off = (got.double() - want).abs() - (UNIT[dtype] * want.abs() + bound + TINY[dtype])
    assert bool((off <= 0).all()), f"off by {off.max().item():.3g} more than the bound"


# rows, k, n: one of each, few rows (one tile to many), odd sizes, both tile shapes
SIZES = [(1, 1, 1), (1, 64, 128), (3, 2048, 136), (5, 100, 77), (16, 512, 2816), (17, 129, 1407), (33, 1000, 64),
         (64, 264, 520), (67, 1000, 1407), (128, 72, 256), (129, 200, 129), (200, 2816, 264), (257, 64, 1000),
         (300, 1003, 515), (640, 320, 72), (1500, 136, 1032)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,k,n", SIZES)
def test_whole_numbers_are_exact(rows, k, n, dtype):
    g = generator(rows + k + n)
    x, w = whole(g, rows, k).to(dtype), whole(g, k, n).to(dtype)
    bias, residual = whole(g, n, most=9).to(dtype), whole(g, rows, n, most=9)
    u = x.double() @ w.double()
    wt = w.t().contiguous().t()
    for weight in (w, wt):
        assert torch.equal(oz.fused_matmul(x, weight, out_dtype=torch.float32).double(), u)
        y = oz.fused_matmul(x, weight, bias, residual=residual, out_dtype=torch.float32)
        assert torch.equal(y.double(), u + bias.double() + residual.double())
        y = oz.fused_matmul(x, weight, bias.float(), activation="relu", out_dtype=torch.float32)
        assert torch.equal(y.double(), (u + bias.double()).clamp(min=0))
        y, pre = oz.fused_matmul(x, weight, bias, activation="relu", residual=residual.to(dtype), return_pre=True)
        assert torch.equal(pre, (u + bias.double()).to(dtype))
        assert torch.equal(y, ((u + bias.double()).clamp(min=0) + residual.double()).to(dtype))
    assert oz.device_status() == 0


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,k,n", SIZES)
@pytest.mark.parametrize("name", ["gelu", "silu"])
def test_activations_of_normal_values(rows, k, n, dtype, name):
    g = generator(rows * 3 + n)
    x, w = normal(g, rows, k).to(dtype), (3 * normal(g, k, n) / math.sqrt(k)).to(dtype)
    bias, residual = normal(g, n).to(dtype), normal(g, rows, n)
    size = x.double().abs() @ w.double().abs() + bias.double().abs()
    u = x.double() @ w.double() + bias.double()
    sums = (k + 3) * 2.0 ** -23 * size
    for out in (torch.float32, dtype):
        r = residual.to(out)
        want = act(u, name)
        bound = 1.13 * sums + 16 * 2.0 ** -24 * want.abs()
        within(oz.fused_matmul(x, w, bias, activation=name, out_dtype=out), want, bound, out)
        added = want + r.double()
        y, pre = oz.fused_matmul(x, w, bias, activation=name, residual=r, out_dtype=out, return_pre=True)
        within(y, added, bound + 2.0 ** -24 * added.abs(), out)
        within(pre, u, sums, dtype)


@pytest.mark.parametrize("name", ACTS, ids=str)
def test_activations_over_their_range(name):
    # one product a result: u is x itself, exactly
    u = torch.cat([torch.linspace(-30, 30, 4001, device=DEV), torch.tensor([0.0, -0.0, 300.0, -300.0], device=DEV)])
    u = u.bfloat16()
    y = oz.fused_matmul(u[:, None], torch.ones(1, 8, device=DEV, dtype=torch.bfloat16), activation=name,
                        out_dtype=torch.float32)
    want = act(u.double(), name)[:, None].expand(-1, 8)
    # the tails are held to their own size: x phi(x) and x sigmoid(x) far below 0.  There
    # an exponent of up to 450 (gelu) is off by half a unit: 450 2^-24 of the value
    within(y, want, (16 + 450) * 2.0 ** -24 * want.abs(), torch.float32)
    odd = torch.tensor([float("nan"), float("inf"), float("-inf")], device=DEV).bfloat16()
    y = oz.fused_matmul(odd[:, None], torch.ones(1, 8, device=DEV, dtype=torch.bfloat16), activation=name)[:, 0]
    assert y[0].isnan() and y[1] == float("inf")
    if name is None:
        assert y[2] == float("-inf")
    elif name == "relu":
        assert y[2] == 0


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,k,n", SIZES)
def test_gradients_of_whole_numbers(rows, k, n, dtype):
    g = generator(rows + 2 * k + n)
    x, w, dy = (whole(g, *s, most=2).to(dtype) for s in ((rows, k), (k, n), (rows, n)))
    pre = whole(g, rows, n).to(dtype)
    for name, u in ((None, None), ("relu", pre)):
        du = dy.double() if u is None else dy.double() * (u.double() > 0)
        for weight in (w, w.t().contiguous().t()):
            dx, dw, db = oz.fused_matmul_backward(dy, x, weight, u, activation=name, bias=True, dw_dtype=torch.float32)
            assert torch.equal(dx, (du @ w.double().t()).to(dtype))
            assert torch.equal(dw.double(), x.double().t() @ du)
            assert torch.equal(db.double(), du.sum(0))
        dx, dw, db = oz.fused_matmul_backward(dy, x, w, u, activation=name)
        assert db is None and torch.equal(dw, (x.double().t() @ du).to(dtype))
    assert oz.device_status() == 0


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,k,n", SIZES[2:])
@pytest.mark.parametrize("name", ACTS, ids=str)
def test_gradients_through_autograd(rows, k, n, dtype, name):
    g = generator(rows + k + 5 * n)
    x, w = normal(g, rows, k).to(dtype), (normal(g, k, n) / math.sqrt(k)).to(dtype)
    bias, residual, dy = normal(g, n).to(dtype), normal(g, rows, n).to(dtype), normal(g, rows, n).to(dtype)
    _, pre = oz.fused_matmul(x, w, bias, activation=name, return_pre=True)
    leaves = [t.clone().requires_grad_() for t in (x, w, bias, residual)]
    y = oz.fused_matmul(*leaves[:3], activation=name, residual=leaves[3])
    dx, dw, db, dr = torch.autograd.grad(y, leaves, dy)
    du = dy.double() if name is None else dy.double() * slope(pre.double(), name)
    # du is rounded to the operands' type (not without an activation), after a few fp32 units
    off = 0 if name is None else UNIT[dtype] + 32 * 2.0 ** -24
    size = (dy.double() * 1.13).abs() if name else du.abs()
    xs, ws = x.double().abs(), w.double().abs()
    within(dx, du @ w.double().t(), ((n + 2) * 2.0 ** -23 + off) * (size @ ws.t()), dtype)
    within(dw, x.double().t() @ du, ((rows + 2) * 2.0 ** -23 + off) * (xs.t() @ size), dtype)
    within(db, du.sum(0), (rows + 40) * 2.0 ** -23 * size.sum(0), dtype)
    assert torch.equal(dr, dy)


@pytest.mark.parametrize("name", ACTS, ids=str)
def test_gradients_against_differences(name):
    g = generator(11)
    rows, k, n = 24, 40, 32
    x, w, b = normal(g, rows, k).half(), (normal(g, k, n) / 6).half(), normal(g, n).half()
    dy = normal(g, rows, n).half()
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    got = torch.autograd.grad(oz.fused_matmul(*leaves, activation=name), leaves, dy)
    base = [t.double() for t in (x, w, b)]

    def value(x, w, b):
        return (act(x @ w + b, name) * dy.double()).sum()

    for i in range(3):
        direction = normal(g, *base[i].shape).double()
        step = 1e-6
        moved = [[t + s * direction if j == i else t for j, t in enumerate(base)] for s in (step, -step)]
        slope_of = (value(*moved[0]) - value(*moved[1])) / (2 * step)
        # each gradient element is off by at most (half a unit for itself, for du and for the rounded
        # u, whose slope moves by less than u's error) of the sum of its terms' magnitudes
        sizes = [dy.double().abs() @ base[1].abs().t(), base[0].abs().t() @ dy.double().abs(), dy.double().abs().sum(0)]
        u_size = (base[0].abs() @ base[1].abs() + base[2].abs()).max()
        bound = (sizes[i] * direction.abs()).sum() * UNIT[torch.float16] * (2.5 + u_size)
        if name == "relu":          # a step that passes the corner: none does unless |u| < step |d u|
            bound = bound + 1e-4
        assert (slope_of - (got[i].double() * direction).sum()).abs() <= bound + 1e-6


def test_only_what_is_needed():
    g = generator(3)
    x, w, b = normal(g, 40, 64).bfloat16(), normal(g, 64, 72).bfloat16(), normal(g, 72).bfloat16()
    r = normal(g, 40, 72).bfloat16()
    dy = normal(g, 40, 72).bfloat16()
    whole_set = [t.clone().requires_grad_() for t in (x, w, b, r)]
    want = torch.autograd.grad(oz.fused_matmul(*whole_set[:3], activation="silu", residual=whole_set[3]), whole_set, dy)
    for i in range(4):
        args = [t.clone() for t in (x, w, b, r)]
        args[i].requires_grad_()
        (got,) = torch.autograd.grad(oz.fused_matmul(*args[:3], activation="silu", residual=args[3]), args[i], dy)
        assert torch.equal(got, want[i])
    with pytest.raises(RuntimeError, match="once_differentiable"):
        leaf = x.clone().requires_grad_()
        (dx,) = torch.autograd.grad(oz.fused_matmul(leaf, w), leaf, dy.clone().requires_grad_(), create_graph=True)
        dx.sum().backward()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_layouts(dtype):
    g = generator(5)
    rows, k, n = 70, 136, 200
    x, w, r, b = (whole(g, *s).to(dtype) for s in ((rows, k), (k, n), (rows, n), (n,)))
    want = oz.fused_matmul(x, w, b, residual=r)

    def spread(t, by):
        held = torch.full((*t.shape[:-1], t.shape[-1] * by + 3), float("nan"), dtype=t.dtype, device=DEV)
        view = held[..., 1:1 + t.shape[-1] * by:by]
        return view.copy_(t)

    views = [lambda t: spread(t, 1), lambda t: spread(t, 2), lambda t: t.t().contiguous().t()]
    for change in views:
        assert torch.equal(oz.fused_matmul(change(x), w, b, residual=r), want)
        assert torch.equal(oz.fused_matmul(x, change(w), b, residual=r), want)
        assert torch.equal(oz.fused_matmul(x, w, b, residual=change(r)), want)
    assert torch.equal(oz.fused_matmul(x, w, spread(b, 2), residual=r), want)
    one = x[:1].expand(rows, k)
    assert torch.equal(oz.fused_matmul(one, w, b, residual=r[:1].expand(rows, n)),
                       oz.fused_matmul(one.contiguous(), w, b, residual=r[:1].expand(rows, n).contiguous()))
    pre, dy = whole(g, rows, n).to(dtype), whole(g, rows, n).to(dtype)
    grads = oz.fused_matmul_backward(dy, x, w, pre, activation="silu", bias=True)
    for change in views:
        for i in range(4):
            args = [change(t) if i == j else t for j, t in enumerate((dy, x, w, pre))]
            got = oz.fused_matmul_backward(*args, activation="silu", bias=True)
            assert all(torch.equal(a, b) for a, b in zip(got, grads))
    assert oz.device_status() == 0


@pytest.mark.parametrize("rows,k,n", [(1, 8191, 129), (3, 777, 2049), (15, 4097, 33), (16, 65, 1001), (40, 1001, 515),
                                      (64, 2050, 1407), (100, 999, 130), (128, 514, 2001), (250, 1500, 63), (9, 63, 7)])
def test_operands_off_the_16_byte_boundaries(rows, k, n):
    # every parity and offset of x's and w's rows; NaN around them
    g = generator(rows + k)
    for dx, dw in ((0, 0), (1, 3), (5, 0), (2, 7), (7, 6)):
        wide = torch.full((rows, k + 9), float("nan"), dtype=torch.bfloat16, device=DEV)
        x = wide[:, dx:dx + k].copy_(whole(g, rows, k))
        big = torch.full((k, n + 9), float("nan"), dtype=torch.bfloat16, device=DEV)
        w = big[:, dw:dw + n].copy_(whole(g, k, n))
        tall = torch.full((n, k + 9), float("nan"), dtype=torch.bfloat16, device=DEV)
        wt = tall[:, dw:dw + k].copy_(w.t()).t()
        u = x.double() @ w.double()
        for weight in (w, wt):
            assert torch.equal(oz.fused_matmul(x, weight), u.bfloat16())
            assert torch.equal(oz.fused_matmul(x, weight, out_dtype=torch.float32).double(), u)
    assert oz.device_status() == 0


@pytest.mark.parametrize("rows,k,n", [(1, 8192, 64), (5, 16384, 200), (40, 12000, 72), (100, 20001, 136), (200, 9000, 260)])
def test_long_contractions(rows, k, n):
    # few tiles: the contraction over as many as 16 CTAs.  Sums of up to 20001 terms of magnitude
    # 4 at most are exact in fp32
    g = generator(k)
    x, w, dy = (whole(g, *s, most=2).bfloat16() for s in ((rows, k), (k, n), (k, n)))
    bias, residual = whole(g, n).bfloat16(), whole(g, rows, n).bfloat16()
    u = x.double() @ w.double()
    assert torch.equal(oz.fused_matmul(x, w), u.bfloat16())
    assert torch.equal(oz.fused_matmul(x, w, out_dtype=torch.float32).double(), u)
    y, pre = oz.fused_matmul(x, w, bias, activation="relu", residual=residual, return_pre=True)
    assert torch.equal(pre, (u + bias.double()).bfloat16())
    assert torch.equal(y, ((u + bias.double()).clamp(min=0) + residual.double()).bfloat16())
    # k rows now: dw (rows, n) sums over them
    tall = x.t().contiguous()
    dx, dw, db = oz.fused_matmul_backward(dy, tall, torch.ones(rows, n, device=DEV).bfloat16(), bias=True,
                                          dw_dtype=torch.float32)
    assert torch.equal(dw.double(), x.double() @ dy.double()) and torch.equal(db.double(), dy.double().sum(0))
    assert torch.equal(dx, dy.double().sum(1, keepdim=True).expand(k, rows).bfloat16())
    assert oz.device_status() == 0


@pytest.mark.parametrize("rows,k,n", [(580, 6504, 1056), (299, 4632, 3880), (536, 7504, 2688), (3384, 4608, 384),
                                      (257, 8192, 519)])
def test_middle_sizes(rows, k, n):
    # a few tiles of 256 x 256, whose contraction pairs of CTAs share
    g = generator(n)
    x, w = whole(g, rows, k, most=2).bfloat16(), whole(g, k, n, most=2).bfloat16()
    bias, residual = whole(g, n).bfloat16(), whole(g, rows, n).bfloat16()
    u = x.double() @ w.double()
    for weight in (w, w.t().contiguous().t()):
        y, pre = oz.fused_matmul(x, weight, bias, activation="relu", residual=residual, return_pre=True)
        assert torch.equal(pre, (u + bias.double()).bfloat16())
        assert torch.equal(y, ((u + bias.double()).clamp(min=0) + residual.double()).bfloat16())
        assert torch.equal(oz.fused_matmul(x, weight), u.bfloat16())
    tall = x.t().contiguous()                         # dw (rows, n) sums over k rows
    dy = w
    dx, dw, _ = oz.fused_matmul_backward(dy, tall, torch.ones(rows, n, device=DEV).bfloat16())
    assert torch.equal(dw, u.bfloat16())
    assert torch.equal(dx, dy.double().sum(1, keepdim=True).expand(k, rows).bfloat16())
    assert oz.device_status() == 0


def test_empty_sizes():
    z = dict(device=DEV, dtype=torch.bfloat16)
    b, r = torch.randn(6, device=DEV).bfloat16(), torch.randn(4, 6, device=DEV).bfloat16()
    assert oz.fused_matmul(torch.zeros(0, 8, **z), torch.zeros(8, 6, **z), b).shape == (0, 6)
    assert oz.fused_matmul(torch.zeros(4, 8, **z), torch.zeros(8, 0, **z)).shape == (4, 0)
    x0, w0 = torch.zeros(4, 0, **z), torch.zeros(0, 6, **z)
    y, pre = oz.fused_matmul(x0, w0, b, activation="relu", residual=r, return_pre=True)
    assert torch.equal(y, (b.float().clamp(min=0) + r.float()).bfloat16()) and torch.equal(pre, b.expand(4, 6))
    y = oz.fused_matmul(x0, w0, out_dtype=torch.float32)
    assert y.dtype == torch.float32 and not y.any()
    for rows, k, n in ((0, 8, 6), (4, 0, 6), (4, 8, 0)):
        dx, dw, db = oz.fused_matmul_backward(torch.ones(rows, n, **z), torch.ones(rows, k, **z), torch.ones(k, n, **z),
                                              bias=True)
        assert dx.shape == (rows, k) and dw.shape == (k, n) and torch.equal(db, torch.full((n,), float(rows), device=DEV))
        assert not dx.any() and not dw.any()


def test_nothing_outside_the_operands_is_read_into_a_result():
    # NaN all around the operands, in the padding of their rows too
    g = generator(9)
    for rows, k, n in ((5, 72, 136), (70, 72, 136), (300, 72, 136), (300, 1000, 520)):
        big = torch.full((rows + 2, k + 16), float("nan"), dtype=torch.bfloat16, device=DEV)
        x = big[1:rows + 1, 8:8 + k].copy_(whole(g, rows, k))
        wide = torch.full((k + 2, n + 16), float("nan"), dtype=torch.bfloat16, device=DEV)
        w = wide[1:k + 1, 8:8 + n].copy_(whole(g, k, n))
        dy = whole(g, rows, n).bfloat16()
        assert torch.equal(oz.fused_matmul(x, w, out_dtype=torch.float32).double(), x.double() @ w.double())
        dx, dw, _ = oz.fused_matmul_backward(dy, x, w, dw_dtype=torch.float32)
        assert torch.equal(dw.double(), x.double().t() @ dy.double())
        assert torch.equal(dx, (dy.double() @ w.double().t()).bfloat16())
