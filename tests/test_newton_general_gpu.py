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

import pytest
import torch

import ozaki_triton_b200 as oz
from ozaki_triton_b200 import _lib

pytestmark = pytest.mark.gpu

DEV = "cuda"
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


def steps_of(g, coefficients, eps=1e-7, splits=None, dtype=torch.float64):
    """The definition in dtype's arithmetic, or (splits) the model of the slices."""
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
            s = x @ x.mT
            x = a * x + (b * s + c * (s @ s)) @ x
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
