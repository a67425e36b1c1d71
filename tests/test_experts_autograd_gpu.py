"""Second derivatives of the grouped product on the GPU.  Needs a B200.

Small whole numbers: every product and sum is exact in fp32, so a result in the
operands' type is the definition rounded once.
"""

import pytest
import torch

import ozaki_triton_b200 as oz

pytestmark = pytest.mark.gpu

DEV = "cuda"


def plain(x, w, bounds):
    parts = [x[:bounds[0]] @ torch.zeros_like(w[0])]
    parts += [x[a:b] @ w[e] for e, (a, b) in enumerate(zip(bounds, bounds[1:]))]
    return torch.cat([*parts, x[bounds[-1]:] @ torch.zeros_like(w[0])])


@pytest.mark.parametrize("sizes,k,n", [([3, 0, 6], 16, 24), ([150, 0, 41], 72, 40)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_gradients_of_gradients(dtype, sizes, k, n):
    g = torch.Generator(device=DEV).manual_seed(k)
    ends = torch.tensor([1] + sizes, device=DEV).cumsum(0)
    bounds, rows = ends.tolist(), 2 + sum(sizes)

    def whole(*shape):
        return torch.randint(-1, 2, shape, generator=g, device=DEV).to(dtype)

    x, w = whole(rows, k).requires_grad_(), whole(len(sizes), k, n).requires_grad_()
    v, p, q = whole(rows, n).requires_grad_(), whole(rows, k), whole(len(sizes), k, n)
    dx, dw = torch.autograd.grad(oz.grouped_matmul(x, w, ends), (x, w), v, create_graph=True)
    got = torch.autograd.grad((dx, dw), (x, w, v), (p, q))
    x6, w6, v6 = (t.detach().double().requires_grad_() for t in (x, w, v))
    dx6, dw6 = torch.autograd.grad(plain(x6, w6, bounds), (x6, w6), v6, create_graph=True)
    want = torch.autograd.grad((dx6, dw6), (x6, w6, v6), (p.double(), q.double()))
    assert torch.equal(dx, dx6.to(dtype)) and torch.equal(dw, dw6.to(dtype))
    for a, b in zip(got[:2], want[:2]):
        assert torch.equal(a, b.to(dtype))
    # v's is the sum of two products, each rounded to the type and then added in it
    half = torch.finfo(dtype).eps / 2
    a6, b6 = plain(p.double(), w6.detach(), bounds), plain(x6.detach(), q.double(), bounds)
    assert bool(((got[2].double() - want[2]).abs() <= half * (a6.abs() + b6.abs() + 1.01 * want[2].abs()) + 1e-12).all())
