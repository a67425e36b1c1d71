"""Calls at the edges of what the operators around an expert layer's products take: tensors
without elements in any layout.  Needs a B200."""

import pytest
import torch

import ozaki_triton_b200 as oz

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_no_tokens_in_any_layout(dtype):
    r = oz.route(torch.zeros(0, 6, device=DEV), 2)
    wide = torch.zeros(4, 40, device=DEV, dtype=dtype)
    for x in (wide[:0, ::2], wide.t()[:20, :0].t(), wide.t()[:0, :4].t()[:, :0].t(), wide[:1, :20].expand(4, 20)[:0]):
        x = x.requires_grad_()
        rows = oz.dispatch(x, r)
        y = oz.combine(rows, r)
        (dx,) = torch.autograd.grad(y, x, torch.zeros_like(y))
        assert rows.shape == y.shape == dx.shape == x.shape
        drows, dweights = oz.combine_backward(x.detach(), wide[:0, :2 * x.shape[1]:2], r)
        assert drows.shape == x.shape and dweights.shape == (0, 2)
        assert oz.dispatch_backward(wide[:0, :2 * x.shape[1]:2], r).shape == x.shape
    few = oz.route(torch.randn(3, 6, device=DEV), 2)
    none = wide[:3, :0:2]
    assert oz.combine(oz.dispatch(none, few), few).shape == (3, 0)
    assert not oz.combine_backward(none, wide.t()[:6, :0], few)[1].any()
    assert oz.device_status() == 0
