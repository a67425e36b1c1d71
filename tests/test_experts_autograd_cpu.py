"""Derivatives of the grouped product through autograd, with the library's two
products replaced by their definitions; no GPU needed."""

import pytest
import torch

import ozaki_triton_b200 as oz
from ozaki_triton_b200 import experts

F64 = torch.float64


def product(x, w, offsets, out_dtype):
    bounds = offsets.tolist()
    y = x.new_zeros(x.shape[0], w.shape[2])
    for e, (a, b) in enumerate(zip(bounds, bounds[1:])):
        y[a:b] = (x.detach()[a:b, :, None] * w.detach()[e]).sum(1)
    return y


def weight_gradient(x, dy, offsets, groups, out_dtype):
    bounds = offsets.tolist()
    return torch.stack([(x.detach()[a:b, :, None] * dy.detach()[a:b, None, :]).sum(0)
                        for a, b in zip(bounds, bounds[1:])])


@pytest.fixture
def plain(monkeypatch):
    monkeypatch.setattr(experts, "_product", product)
    monkeypatch.setattr(experts, "_weight_gradient", weight_gradient)


def operands():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(9, 5, generator=g, dtype=F64, requires_grad=True)
    w = torch.randn(3, 5, 4, generator=g, dtype=F64, requires_grad=True)
    return x, w, torch.tensor([1, 4, 4, 8])               # a row before, an empty group, a row after


def test_first_and_second_derivatives_against_differences(plain):
    x, w, offsets = operands()
    f = lambda x, w: oz.grouped_matmul(x, w, offsets)      # noqa: E731
    assert torch.autograd.gradcheck(f, (x, w))
    assert torch.autograd.gradgradcheck(f, (x, w))


@pytest.mark.parametrize("of", ["x", "w"])
def test_second_derivative_of_one_operand(plain, of):
    x, w, offsets = operands()
    f = (lambda x: oz.grouped_matmul(x, w.detach(), offsets)) if of == "x" else \
        (lambda w: oz.grouped_matmul(x.detach(), w, offsets))
    # nonlinear in the result, so that the gradient depends on the operand
    h = lambda v: f(v).square()                            # noqa: E731
    assert torch.autograd.gradgradcheck(h, (x if of == "x" else w,))


def test_a_gradient_penalty_beside_another_path_is_whole(plain):
    x, w, offsets = operands()
    y = oz.grouped_matmul(x, w, offsets)
    dx, = torch.autograd.grad((y.square().sum() + x.pow(4).sum()), x, create_graph=True)
    got, = torch.autograd.grad(dx.square().sum(), w)
    bounds = offsets.tolist()
    x2, w2 = x.detach().requires_grad_(), w.detach().requires_grad_()
    y2 = torch.cat([x2[:1] @ w2[0] * 0, *(x2[a:b] @ w2[e] for e, (a, b) in enumerate(zip(bounds, bounds[1:]))),
                    x2[8:] @ w2[0] * 0])
    dx2, = torch.autograd.grad((y2.square().sum() + x2.pow(4).sum()), x2, create_graph=True)
    want, = torch.autograd.grad(dx2.square().sum(), w2)
    assert torch.allclose(got, want, rtol=1e-12, atol=1e-12)
