"""Newton-Schulz orthogonalisation against its definition in 64 bits.  Needs a B200.

The bound of a result is that of a model of the roundings that the operator
documents: each matrix that enters a product is rounded to one or two fp16
slices at its power-of-two scale, everything else is 64 bits.  A result may
be twice as far from the definition as the model is, plus half a unit of its
own type, plus 2^-23 (terms of a sum)^(1/2) a step for the fp32 sums,
each step's error growing by at most the largest factor a step has for any
singular value (the linear coefficient, for small ones).
"""

import pytest
import torch

import ozaki_triton_b200 as oz

pytestmark = pytest.mark.gpu

DEV = "cuda"
ABC = (3.4445, -4.7750, 2.0315)
CUBIC = [(1.5, -0.5, 0.0)] * 8
UNIT = {torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def sliced(x, splits):
    """x as the sum of `splits` fp16 slices at a scale that puts a norm of 1 at 2^12."""
    if splits is None:
        return x, x
    high = (x * 2.0 ** 12).half().double()
    low = (x * 2.0 ** 12 - high).half().double()
    return high * 2.0 ** -12, (high + low) * 2.0 ** -12


def steps_of(g, coefficients, eps, splits=None):
    """The definition (splits None), or the model of its roundings."""
    x = g.double()
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    for a, b, c in coefficients:
        high, wide = sliced(x, splits)
        u = high if splits == 1 else wide
        s = sliced(u @ u.mT, splits)[0 if splits == 1 else 1]
        p = sliced(b * s + c * (s @ s), splits)[0 if splits == 1 else 1]
        x = a * wide + p @ u
    return x.mT if tall else x


def rel(x, y):
    return ((x.double() - y).norm() / y.norm()).item()


def gradient(seed, *shape, kind="normal"):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(*shape, generator=g, device=DEV)
    if kind == "low rank":
        r = max(1, min(shape[-2:]) // 16)
        u = torch.randn(*shape[:-1], r, generator=g, device=DEV)
        v = torch.randn(*shape[:-2], r, shape[-1], generator=g, device=DEV)
        x = 1e-3 * (u @ v + 0.2 * x)
    return x


SHAPES = [(1, 1), (1, 40), (33, 1), (3, 5, 7), (16, 64), (2, 64, 16), (130, 257), (2, 3, 129, 100), (256, 256),
          (511, 300), (300, 1000), (5, 128, 384), (1030, 520), (640, 1288), (1900, 2100),
          (2, 70, 2600), (4200, 130), (1, 33, 9000), (3, 300, 2050), (1400, 3500)]


@pytest.mark.parametrize("kind", ["normal", "low rank"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_orthogonalize(shape, dtype, kind):
    g = gradient(sum(shape), *shape, kind=kind).to(dtype)
    got = oz.orthogonalize(g)
    assert got.shape == g.shape and got.dtype == dtype and got.is_contiguous()
    splits = 1 if dtype == torch.bfloat16 else 2
    want = steps_of(g, [ABC] * 5, 1e-7)
    model = rel(steps_of(g, [ABC] * 5, 1e-7, splits), want)
    sums = sum(ABC[0] ** i for i in range(5)) * 2.0 ** -23 * max(shape[-2:]) ** 0.5
    assert rel(got, want) <= 2 * model + UNIT[dtype] + sums
    assert oz.device_status() == 0


@pytest.mark.parametrize("steps,coefficients", [(1, ABC), (3, ABC), (8, CUBIC), (2, [(3.0, -3.2, 1.2), (1.5, -0.5, 0.0)])])
def test_steps_and_coefficients(steps, coefficients):
    g = gradient(steps, 2, 96, 160)
    rows = coefficients if isinstance(coefficients, list) else [coefficients] * steps
    for splits in (1, 2):
        want = steps_of(g, rows, 1e-3)
        model = rel(steps_of(g, rows, 1e-3, splits), want)
        sums = sum(max(abs(r[0]) for r in rows) ** i for i in range(steps)) * 2.0 ** -23 * 160 ** 0.5
        got = oz.orthogonalize(g, steps, coefficients, 1e-3, num_splits=splits)
        assert rel(got, want) <= 2 * model + 2.0 ** -24 + sums


def test_singular_values_come_near_one():
    u, _, v = torch.linalg.svd(gradient(1, 256, 512), full_matrices=False)
    s = torch.logspace(0, -2, 256, device=DEV)
    for dtype in (torch.float32, torch.bfloat16):
        q = oz.orthogonalize(((u * s) @ v).to(dtype), 6).float()
        found = torch.linalg.svdvals(q)
        assert 0.6 < found.min().item() and found.max().item() < 1.3


@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1.0, 1e18])
def test_the_scale_of_the_gradient_does_not_matter(scale):
    g = gradient(2, 64, 96)
    x = g.double() * scale
    got = oz.orthogonalize(x.float(), eps=0.0)
    want = steps_of(x.float(), [ABC] * 5, 0.0)
    model = rel(steps_of(x.float(), [ABC] * 5, 0.0, 2), want)
    assert rel(got, want) <= 2 * model + 2.0 ** -24 + 177 * 2.0 ** -23 * 96 ** 0.5


def test_members_of_a_batch_are_independent():
    g = gradient(4, 4, 48, 80)
    g[1] = 0
    g[2, 0, 0] = float("nan")
    got = oz.orthogonalize(g)
    for i in (0, 3):
        assert torch.equal(got[i], oz.orthogonalize(g[i]))
    assert not got[1].any() and bool(torch.isnan(got[2]).all())


def test_layouts_and_empty_stacks():
    g = gradient(6, 96, 200)
    want = oz.orthogonalize(g)
    wide = torch.zeros(96, 2, 400, device=DEV)
    wide[:, 1, 3::2][:, :198] = g[:, :198]
    for view, of in ((g.t().contiguous().t(), g), (wide[:, 1, 3::2][:, :198], g[:, :198].contiguous()),
                     (torch.empty(96 * 200 + 1, device=DEV)[1:].view(96, 200).copy_(g), g)):
        assert torch.equal(oz.orthogonalize(view), oz.orthogonalize(of))
    same = oz.orthogonalize(g.expand(3, 96, 200))
    assert all(torch.equal(m, want) for m in same)
    assert oz.orthogonalize(g[:0]).shape == (0, 200)
    assert oz.orthogonalize(g.expand(0, 96, 200)).shape == (0, 96, 200)


def test_same_input_same_bits():
    g = gradient(8, 3, 520, 700, kind="low rank").bfloat16()
    first = oz.orthogonalize(g)
    for _ in range(3):
        assert torch.equal(oz.orthogonalize(g), first)
