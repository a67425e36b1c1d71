"""Newton-Schulz orthogonalisation of matrices too large for one launch (products on
the tensor cores in fp16 slices) against its definition in 64 bits.  Needs a B200.

Every shape here takes that path: its calls need a workspace, which is asserted.

A result's error has three parts, each of which is computed for the very input
and then allowed twice: the slices (a model of the documented roundings: each
matrix that enters a product is rounded to one or two fp16 slices at a power-of-two
scale, everything else in 64 bits), the fp32 sums (what the definition is off
by when it is evaluated in fp32 throughout), and half a unit of the
result's type, once.
"""

import math

import pytest
import torch

import ozaki_triton_b200 as oz
from ozaki_triton_b200 import _lib

pytestmark = pytest.mark.gpu

DEV = "cuda"
ABC = (3.4445, -4.7750, 2.0315)
CUBIC = [(1.5, -0.5, 0.0)] * 8
# a published minimax schedule: steep outside the interval that each step expects
STEEP = [(8.28721201814563, -23.595886519098837, 17.300387312530933),
         (4.107059111542203, -2.9478499167379106, 0.5448431082926601),
         (3.9486908534822946, -2.908902115962949, 0.5518191394370137),
         (3.3184196573706015, -2.488488024314874, 0.51004894012372),
         (2.300652019954817, -1.6689039845747493, 0.4188073119525673),
         (1.891301407787398, -1.2679958271945868, 0.37680408948524835),
         (1.8750014808534479, -1.2500016453999487, 0.3750001645474248),
         (1.875, -1.25, 0.375)]
# the same with its interval widened by a hundredth, as it is used with rounded products
SAFE = [(a / 1.01, b / 1.01 ** 3, c / 1.01 ** 5) for a, b, c in STEEP[:-1]] + STEEP[-1:]
UNIT = {torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
CODE = {torch.float32: _lib.OZ_F32, torch.float16: _lib.OZ_F16, torch.bfloat16: _lib.OZ_BF16}


def sliced(x, splits):
    """x as the products see it, and as the linear term does: one or two fp16 slices at a
    scale that puts a norm of 1 at 2^12."""
    high = (x * 2.0 ** 12).half().double()
    low = (x * 2.0 ** 12 - high).half().double()
    wide = (high + low) * 2.0 ** -12
    return (high * 2.0 ** -12 if splits == 1 else wide), wide


def steps_of(g, coefficients, eps=1e-7, splits=None, dtype=torch.float64, cut=0.0):
    """The definition in dtype's arithmetic, or (splits) the model of the slices; cut: what every
    product loses of its size."""
    x = g.to(dtype)
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    for a, b, c in coefficients:
        if splits:
            u, wide = sliced(x, splits)
            s = sliced(u @ u.mT, splits)[0]
            x = a * wide + sliced(b * s + c * (s @ s), splits)[0] @ u
        else:
            s = (x @ x.mT) * (1 - cut)
            x = a * x + ((b * s + c * (s @ s) * (1 - cut)) @ x) * (1 - cut)
    return x.mT if tall else x


def rel(x, y):
    return ((x.double() - y).norm() / y.norm()).item()


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV)


def general(g, steps, splits):
    """The tensor-core path is the one that g takes."""
    m, n = g.shape[-2:]
    return _lib.load().oz_orthogonalize_workspace_bytes(CODE[g.dtype], g.numel() // (m * n), m, n, steps, splits) > 0


def bound(g, coefficients, splits, eps=1e-7):
    """(definition, allowed relative error)."""
    want = steps_of(g, coefficients, eps)
    slices = rel(steps_of(g, coefficients, eps, splits), want)
    sums = rel(steps_of(g, coefficients, eps, dtype=torch.float32), want)
    return want, 2 * slices + 2 * sums + UNIT[g.dtype]


@pytest.mark.parametrize("splits", [1, 2])
@pytest.mark.parametrize("schedule", [STEEP[:5], STEEP, SAFE], ids=["5 steps", "8 steps", "widened"])
@pytest.mark.parametrize("shape", [(300, 1000), (1000, 300), (2, 520, 700)], ids=str)
def test_steep_schedules(shape, schedule, splits):
    g = normal(sum(shape), *shape)
    assert general(g, len(schedule), splits)
    want, allowed = bound(g, schedule, splits)
    assert rel(oz.orthogonalize(g, len(schedule), schedule, num_splits=splits), want) <= allowed
    assert oz.device_status() == 0


def test_schedules_that_diverge_are_refused():
    # (4, -6, 3) maps 0.54 to 1.35, 1.35 to 4.2 and 4.2 to 3300: good for the last step only
    g = normal(5, 300, 300)
    for steps in (1, 3):
        want, allowed = bound(g, [(4.0, -6.0, 3.0)] * steps, 2)
        assert rel(oz.orthogonalize(g, steps, (4.0, -6.0, 3.0)), want) <= allowed
    with pytest.raises(oz.OzakiError, match="before step 4 of 5"):
        oz.orthogonalize(g, 5, (4.0, -6.0, 3.0))


def normal_or_low_rank(seed, shape, kind):
    x = normal(seed, *shape)
    if kind == "low rank":
        r = max(1, min(shape[-2:]) // 16)
        x = 1e-3 * (normal(seed + 1, *shape[:-1], r) @ normal(seed + 2, *shape[:-2], r, shape[-1]) + 0.2 * x)
    return x


def with_cuts(g, coefficients, splits, eps=1e-7):
    """bound(), and for the tensor core's sums, which are cut off and not rounded: an
    instruction of 16 terms loses up to 2^-23 of the running sum, which grows evenly, and half of
    that on average, so m instructions 2^-25 m.  m: 12 for each block of 64 terms that an
    accumulator takes with two slices (1, 2 or 4 blocks by the work), 4 for each of all with one."""
    want, allowed = bound(g, coefficients, splits, eps)
    rows, cols = sorted(g.shape[-2:])
    if splits == 2:
        work = g.numel() // cols * rows * (3 * cols + rows)
        m = 12 * (1 if work < 2e10 else 2 if rows < 1536 else 4)
    else:
        m = 4 * math.ceil(cols / 64)
    return want, allowed + 2 * rel(steps_of(g, coefficients, eps, cut=m * 2.0 ** -25), want)


@pytest.mark.parametrize("kind", ["normal", "low rank"])
@pytest.mark.parametrize("shape", [(130, 130), (256, 256), (511, 300), (300, 1000), (1030, 520), (640, 1288), (1900, 2100),
                                   (4200, 130), (2, 70, 2600), (3, 300, 2050), (148, 3737), (1400, 3500),
                                   (5, 128, 384), (4096, 4096)], ids=str)
def test_fp32_is_held_to_two_slices_and_fp32_sums(shape, kind):
    g = normal_or_low_rank(sum(shape), shape, kind)
    assert general(g, 5, 2)
    want, allowed = with_cuts(g, [ABC] * 5, 2)
    # the bound tells one slice from two
    assert rel(steps_of(g, [ABC] * 5, splits=1), want) > 4 * allowed
    assert rel(oz.orthogonalize(g), want) <= allowed
    assert oz.device_status() == 0


@pytest.mark.parametrize("kind", ["normal", "low rank"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("shape", [(256, 256), (300, 1000), (1030, 520), (2, 200, 144)], ids=str)
def test_16_bit_results_are_the_rounded_definition(shape, dtype, kind):
    """Below 5e9 of work both 16-bit types take two slices.  A result off by d before it is
    rounded is rounded the other way with a chance of |d| over the spacing of its type, s, and
    differs by s then: |d| s in the mean square, sqrt(rel(d) rel(s)) of the whole (half of it
    again allowed for chance).  s is at most 2^-7 (bf16) or 2^-10 (fp16; and 2^-24 for
    subnormal results) of the value."""
    g = normal_or_low_rank(sum(shape), shape, kind).to(dtype)
    assert general(g, 5, 2)
    want, allowed = with_cuts(g, [ABC] * 5, 2)
    allowed -= UNIT[dtype]
    spacing = 2.0 ** -7 if dtype == torch.bfloat16 else \
        (want.abs() * 2.0 ** -10).clamp(min=2.0 ** -24).norm().item() / want.norm().item()
    rounded = want.to(dtype).double()
    off = rel(oz.orthogonalize(g), rounded)
    assert off <= 1.5 * (spacing * allowed) ** 0.5
    one = rel(steps_of(g, [ABC] * 5, splits=1).to(dtype), rounded)
    assert one > 1.5 * (spacing * allowed) ** 0.5          # the bound tells one slice from two


SCHEDULES = {"1 step": [ABC], "3 steps": [ABC] * 3, "7 steps": [ABC] * 7, "cubic": CUBIC,
             "two kinds": [(3.0, -3.2, 1.2), (1.5, -0.5, 0.0)], "linear": [(0.5, 0.0, 0.0)] * 2}


@pytest.mark.parametrize("eps", [1e-7, 3.0])
@pytest.mark.parametrize("schedule", SCHEDULES)
@pytest.mark.parametrize("shape", [(300, 1000), (1000, 300), (2, 520, 700)], ids=str)
def test_schedules_and_slices(shape, schedule, eps):
    coefficients = SCHEDULES[schedule]
    g = normal(sum(shape), *shape)
    off = {}
    for splits in (1, 2):
        assert general(g, len(coefficients), splits)
        want, allowed = with_cuts(g, coefficients, splits, eps)
        got = oz.orthogonalize(g, len(coefficients), coefficients, eps, num_splits=splits)
        off[splits] = rel(got, want)
        assert off[splits] <= allowed
    if schedule != "linear":                               # its products vanish
        assert off[1] > 10 * off[2]


@pytest.mark.parametrize("dtype,scale", [(torch.float32, s) for s in (1e-36, 1e-30, 1e-12, 1e18, 1e34)]
                         + [(torch.bfloat16, 1e-36), (torch.bfloat16, 1e30), (torch.float16, 1e-6), (torch.float16, 1e4)],
                         ids=str)
@pytest.mark.parametrize("shape", [(300, 400), (400, 300)], ids=str)
def test_the_scale_of_the_gradient_does_not_matter(shape, dtype, scale):
    g = (normal(2, *shape).double() * scale).to(dtype)
    assert general(g, 5, 2)
    want, allowed = with_cuts(g.double().div(scale).float(), [ABC] * 5, 2, 0.0)
    assert rel(oz.orthogonalize(g, eps=0.0), want) <= allowed + UNIT[dtype]


@pytest.mark.parametrize("bad", [0.0, float("nan"), float("inf")], ids=str)
@pytest.mark.parametrize("splits", [1, 2])
@pytest.mark.parametrize("shape", [(4, 300, 400), (4, 400, 300), (4, 70, 2600)], ids=str)
def test_members_of_a_batch_are_independent(shape, splits, bad):
    g = normal(4, *shape)
    assert general(g, 5, splits)
    before = oz.orthogonalize(g, num_splits=splits)
    if bad == 0:
        g[1] = 0
    else:
        g[1, 5, 7] = bad
    got = oz.orthogonalize(g, num_splits=splits)
    for i in (0, 2, 3):
        assert torch.equal(got[i], before[i])
    assert not got[1].any() if bad == 0 else bool(torch.isnan(got[1]).all())


@pytest.mark.parametrize("shape", [(40, 60), (300, 400)], ids=str)
def test_a_zero_matrix_stays_zero_without_eps(shape):
    assert not oz.orthogonalize(torch.zeros(shape, device=DEV), eps=0.0).any()


LAYOUTS = {
    "columns first": lambda g: g.mT.contiguous().mT,
    "every other element": lambda g: torch.zeros(*g.shape[:-1], 2 * g.shape[-1], device=DEV, dtype=g.dtype)[..., ::2].copy_(g),
    "every third row": lambda g: torch.zeros(*g.shape[:-2], 3 * g.shape[-2], g.shape[-1], device=DEV,
                                             dtype=g.dtype)[..., ::3, :].copy_(g),
    "odd address": lambda g: torch.zeros(g.numel() + 1, device=DEV, dtype=g.dtype)[1:].view(g.shape).copy_(g),
    "odd pitch": lambda g: torch.zeros(*g.shape[:-1], g.shape[-1] + 1, device=DEV, dtype=g.dtype)[..., 1:].copy_(g),
    "wide pitch": lambda g: torch.zeros(*g.shape[:-1], g.shape[-1] + 8, device=DEV, dtype=g.dtype)[..., 8:].copy_(g),
    "odd pitch, columns first": lambda g: torch.zeros(*g.shape[:-2], g.shape[-1], g.shape[-2] + 3, device=DEV,
                                                      dtype=g.dtype)[..., 3:].mT.copy_(g),
}


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("shape", [(300, 400), (400, 300), (2, 301, 203)], ids=str)
def test_layouts(shape, dtype, layout):
    g = normal(sum(shape), *shape).to(dtype)
    view = LAYOUTS[layout](g)
    assert general(view, 5, 2) and torch.equal(view, g)
    want, allowed = with_cuts(g, [ABC] * 5, 2)
    got = oz.orthogonalize(view)
    assert got.is_contiguous() and rel(got, want) <= allowed


def test_expanded_and_strided_stacks():
    g = normal(6, 300, 400)
    want, allowed = with_cuts(g, [ABC] * 5, 2)
    for m in oz.orthogonalize(g.expand(3, 300, 400)):
        assert rel(m, want) <= allowed
    row = normal(7, 1, 400).expand(300, 400)               # rank one, rows repeated
    want, allowed = with_cuts(row, [ABC] * 5, 2)
    assert rel(oz.orthogonalize(row), want) <= allowed
    stack = torch.zeros(300, 3, 400, device=DEV)
    stack[:, 1] = g
    stack[:, 2] = 2 * g
    got = oz.orthogonalize(stack.transpose(0, 1)[1:])
    want, allowed = with_cuts(g, [ABC] * 5, 2)
    assert rel(got[0], want) <= allowed and rel(got[1], want) <= allowed
    four = oz.orthogonalize(g.expand(2, 2, 300, 400))
    assert four.shape == (2, 2, 300, 400) and all(rel(m, want) <= allowed for m in four.flatten(0, 1))
