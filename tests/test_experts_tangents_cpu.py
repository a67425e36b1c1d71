"""Forward-mode derivatives are refused, not lost; no GPU needed."""

import pytest
import torch
from torch.autograd import forward_ad

import ozaki_triton_b200 as oz

F16 = torch.float16


def dual(t):
    return forward_ad.make_dual(t, torch.ones_like(t))


X, W, DY = torch.zeros(6, 64, dtype=F16), torch.zeros(2, 64, 32, dtype=F16), torch.zeros(6, 32, dtype=F16)
OFFSETS = torch.tensor([0, 2, 6])
PACKED, SCALES = torch.zeros(10, 32, dtype=torch.uint8), torch.zeros(10, 2, dtype=F16)
CALLS = {
    "product, x": lambda f: oz.grouped_matmul(f(X), W, OFFSETS),
    "product, w": lambda f: oz.grouped_matmul(X, f(W), OFFSETS),
    "gradients, dy": lambda f: oz.grouped_matmul_backward(f(DY), X, W, OFFSETS),
    "gradients, x": lambda f: oz.grouped_matmul_backward(DY, f(X), W, OFFSETS),
    "gradients, w": lambda f: oz.grouped_matmul_backward(DY, X, f(W), OFFSETS),
    "4 bits, x": lambda f: oz.matmul_w4(f(X), PACKED, SCALES),
    "4 bits, scales": lambda f: oz.matmul_w4(X, PACKED, f(SCALES)),
    "orthogonalize": lambda f: oz.orthogonalize(f(torch.zeros(4, 4))),
}


@pytest.mark.parametrize("call", CALLS)
def test_a_tangent_is_refused(call):
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="tangent"):
            CALLS[call](dual)
        # without a tangent the call goes on to its own checks, inside a level as outside
        with pytest.raises(ValueError, match="CUDA tensors only"):
            CALLS[call](lambda t: t)
    with pytest.raises(ValueError, match="CUDA tensors only"):
        CALLS[call](lambda t: t)


def test_a_tangent_beside_a_recorded_gradient_is_refused():
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError):
            oz.grouped_matmul(dual(X), W.clone().requires_grad_(), OFFSETS)


def test_a_tangent_that_reaches_the_backward_pass_is_refused(monkeypatch):
    from ozaki_triton_b200 import experts
    monkeypatch.setattr(experts, "_product", lambda x, w, o, d: x.new_zeros(x.shape[0], w.shape[2]))
    monkeypatch.setattr(experts, "_weight_gradient", lambda x, dy, o, n, d: x.new_zeros(n, x.shape[1], dy.shape[1]))
    for x, w in ((X.clone().requires_grad_(), W), (X, W.clone().requires_grad_())):
        y = oz.grouped_matmul(x, w, OFFSETS)
        with forward_ad.dual_level():
            with pytest.raises(NotImplementedError, match="tangent"):
                torch.autograd.grad(y, x if x.requires_grad else w, dual(DY))
