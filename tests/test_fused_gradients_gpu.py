"""Gradients of the fused product, element by element, against 64-bit differentiation of
act(x w + b) by the autograd engine and against central differences: neither shares the
formulas of the slopes.  Needs a B200.

What the call rounds on the way, per element: u to fp16 (the slope then moves by at most its own
largest slope, 0.8 for gelu and 0.5 for silu, times 2^-11 |u|; relu's by nothing, since rounding keeps
the sign), the sums of u (k + 3 terms at 2^-23 of their magnitudes), du to fp16 (2^-11 of it) and
the activations' arithmetic (32 2^-24).  A gradient sums those over its terms, n or rows of them
(2^-23 of their magnitudes each), and is rounded to fp16.  The bounds are held below a tenth of the
gradients they check, so that one which is zero, halved or doubled, or lacks a term of the slope, fails.
"""

import math

import pytest
import torch

import ozaki_triton_b200 as oz

pytestmark = pytest.mark.gpu

DEV = "cuda"
HALF = 2.0 ** -11
STEEPEST, BEND = {None: 1.0, "relu": 1.0, "gelu": 1.13, "silu": 1.1}, {None: 0.0, "relu": 0.0, "gelu": 0.8, "silu": 0.5}
ACTS = [None, "relu", "gelu", "silu"]


def act(u, name):
    return {None: lambda: u, "relu": lambda: u.clamp(min=0), "gelu": lambda: u * 0.5 * torch.erfc(-u / math.sqrt(2)),
            "silu": lambda: u * torch.sigmoid(u)}[name]()


def inputs(rows, k, n, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    return [normal(rows, k).half(), (normal(k, n) * 1.5 / math.sqrt(k)).half(), normal(n).half()], normal(rows, n).half()


def bounds(name, x, w, b, dy, want):
    """Of dx, dw and db; x, w, b, dy in 64 bits."""
    rows, k = x.shape
    n = w.shape[1]
    u = x @ w + b
    sums = (k + 3) * 2.0 ** -23 * (x.abs() @ w.abs() + b.abs())
    # of du: the slope at a rounded u, and what is rounded itself where there is an activation
    du = dy.abs() * (BEND[name] * (HALF * u.abs() + sums) + (STEEPEST[name] * (32 * 2.0 ** -24 + (HALF if name else 0))))
    if name == "relu":                          # a sum next to 0 may fall on its other side
        du = du + dy.abs() * (u.abs() <= sums)
    size = STEEPEST[name] * dy.abs()
    terms = [(n + 2) * 2.0 ** -23 * (size @ w.abs().t()) + du @ w.abs().t(),
             (rows + 2) * 2.0 ** -23 * (x.abs().t() @ size) + x.abs().t() @ du, (rows + 40) * 2.0 ** -23 * size.sum(0) + du.sum(0)]
    return [t + HALF * g.abs() + 2.0 ** -25 for t, g in zip(terms, want)]


def hold(got, want, limits):
    for a, b, limit in zip(got, want, limits):
        assert limit.norm() <= 0.1 * b.norm()               # or the check would say little
        assert bool(((a.double() - b).abs() <= limit).all()), ((a.double() - b).abs() / limit).max().item()


@pytest.mark.parametrize("name", ACTS, ids=str)
@pytest.mark.parametrize("rows,k,n", [(24, 40, 32), (1, 64, 8), (33, 129, 77), (200, 264, 520), (130, 1000, 257)])
def test_gradients_by_64_bit_autograd(rows, k, n, name):
    for seed in (11, 12, 13):
        given, dy = inputs(rows, k, n, seed)
        leaves = [t.clone().requires_grad_() for t in given]
        got = torch.autograd.grad(oz.fused_matmul(*leaves, activation=name), leaves, dy)
        exact = [t.double().requires_grad_() for t in given]
        want = torch.autograd.grad(act(exact[0] @ exact[1] + exact[2], name), exact, dy.double())
        hold(got, want, bounds(name, *(t.detach() for t in exact), dy.double(), want))


@pytest.mark.parametrize("name", ACTS, ids=str)
def test_gradients_by_differences(name):
    # every element of x, w and b moved by itself
    given, dy = inputs(12, 20, 16, 21)
    leaves = [t.clone().requires_grad_() for t in given]
    got = torch.autograd.grad(oz.fused_matmul(*leaves, activation=name), leaves, dy)
    x, w, b = (t.double() for t in given)
    step = 2.0 ** -20

    def value(x, w, b):
        return (act(x @ w + b, name) * dy.double()).sum((-2, -1))

    def moved(t):
        eye = torch.eye(t.numel(), dtype=torch.float64, device=DEV).view(t.numel(), *t.shape) * step
        return t + eye, t - eye

    want = []
    for i, t in enumerate((x, w, b)):
        up, down = moved(t)
        if i == 2:
            up, down = up[:, None], down[:, None]
        args = [[x, w, b], [x, w, b]]
        args[0][i], args[1][i] = up, down
        want.append(((value(*args[0]) - value(*args[1])) / (2 * step)).view(t.shape))
    # a difference is off by its value's rounding, 2^-52 of a sum of some 200 terms of magnitude up to 10 over
    # the step, and by step^2 / 6 of the third derivative: 1e-6 holds both; relu's corner lies within a step of none
    limits = bounds(name, x, w, b, dy.double(), want)
    if name == "relu":
        assert bool(((x @ w + b).abs() > 16 * step).all())
    hold(got, want, [t + 1e-6 for t in limits])
