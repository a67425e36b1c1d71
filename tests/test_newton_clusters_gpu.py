"""Small matrices whose cluster has CTAs without any columns: such a CTA has no
loads to wait for and reaches the exchange of the norms first, so the exchange
has to wait until every CTA of the cluster has started.  Needs a B200.
"""

import pytest
import torch

import ozaki_triton_b200 as oz

pytestmark = pytest.mark.gpu

ABC = (3.4445, -4.7750, 2.0315)


def define(g, steps=5, eps=1e-7):
    a, b, c = ABC
    x = g.double()
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    for _ in range(steps):
        s = x @ x.mT
        x = a * x + (b * s + c * (s @ s)) @ x
    return x


# 8 CTAs a matrix: of 12 columns for 65 (two have none) and for 81 (one), of 16 for
# 101 and of 20 for 130 (one)
@pytest.mark.parametrize("shape", [(8, 64, 65), (8, 64, 81), (8, 100, 101), (1, 128, 130)], ids=str)
def test_clusters_with_empty_panels(shape):
    g = torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(shape[-1]), device="cuda")
    want = define(g)
    first = oz.orthogonalize(g)
    # fp32 throughout: each step's sums are off by 2^-24 a term at most in the worst
    # case and by its square root as a rule, and 5 steps multiply an error by 3.4445 each
    # where the singular value is small: 3.4445^4 2^-24 (terms)^(1/2) and as much again
    # for each of the 3 products of a step
    bound = 3 * 141 * 2.0 ** -24 * shape[-1] ** 0.5
    assert (first.double() - want).flatten(1).norm(dim=1).div(want.flatten(1).norm(dim=1)).max().item() <= bound
    for _ in range(50):
        assert torch.equal(oz.orthogonalize(g), first)
