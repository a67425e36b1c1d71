"""Rows operators on tensors without elements in any layout; no GPU needed.

The device check and the launch are replaced, so that a call runs as far as its plan
and its result's allocation.
"""

import pytest
import torch

import ozaki_triton_b200 as oz
from ozaki_triton_b200 import routing as module

I32, F32 = torch.int32, torch.float32


@pytest.fixture
def launches(monkeypatch):
    found = []
    monkeypatch.setattr(module, "_PLANS", type(module._PLANS)())
    monkeypatch.setattr(module, "_check_places", lambda *ts: 0)
    monkeypatch.setattr(module, "_launch", found.append)
    return found


def routing(t, k, e=4):
    return oz.Routing(torch.zeros(t, k), torch.zeros(t, k, dtype=I32), torch.zeros(t, k, dtype=I32),
                      torch.zeros(e + 1, dtype=I32), torch.zeros(e, dtype=I32), torch.zeros((), dtype=I32), torch.zeros(()))


def layouts(rows, columns, dtype):
    """(rows, columns) tensors without elements: contiguous, across, and with a step along the columns."""
    z = torch.zeros(max(rows, columns) + 8, 2 * max(rows, columns) + 16, dtype=dtype)
    return [torch.zeros(rows, columns, dtype=dtype), torch.zeros(columns, rows, dtype=dtype).t(), z[:rows, :2 * columns:2],
            z.t()[:rows, :columns], torch.zeros(rows, 1, dtype=dtype).expand(rows, columns) if rows == 0 else z[:rows, :0]]


@pytest.mark.parametrize("dtype", [F32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("tokens,d", [(0, 0), (0, 1), (0, 8), (0, 33), (1, 0), (6, 0)])
def test_every_layout_without_elements(launches, tokens, d, dtype):
    k, r = 2, routing(tokens, 2)
    for x in layouts(tokens, d, dtype):
        assert oz.dispatch(x, r).shape == (tokens * k, d)
        for rows in layouts(tokens * k, d, dtype):
            drows, dweights = oz.combine_backward(x, rows, r)
            assert drows.shape == rows.shape and dweights.shape == (tokens, k)
    for rows in layouts(tokens * k, d, dtype):
        assert oz.combine(rows, r).shape == (tokens, d)
        assert oz.dispatch_backward(rows, r).shape == (tokens, d)
    assert not launches or tokens > 0


def test_layouts_with_elements_are_still_copied(launches):
    x = torch.zeros(6, 16)[:, ::2]
    assert oz.dispatch(x, routing(6, 2)).shape == (12, 8)
    assert launches[-1].args.x != x.data_ptr() and launches[-1].args.x_row == 8
