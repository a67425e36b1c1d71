"""Clipping of many gradients by their global norm, against 64 bits.  Needs a B200.

The sum of squares is held in fp32 over at most 64 terms and in fp64 beyond, so
the norm is off by at most 34 2^-24 of itself, and so is the factor, with two
more roundings.
"""

import math

import pytest
import torch

import ozaki_triton_b200 as oz

pytestmark = pytest.mark.gpu

DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
UNIT = {d: torch.finfo(d).eps / 2 for d in DTYPES}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -126}


def generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def define(grads, max_norm, eps=1e-6):
    norm = math.sqrt(sum(float((g.double() ** 2).sum()) for g in grads))
    return norm, min(1.0, max_norm / (norm + eps))


def check(grads, max_norm, to=None, eps=1e-6):
    norm, factor = define(grads, max_norm, eps)
    want = [g.double() * factor for g in grads]
    outs = None if to is None else [torch.empty_like(g, dtype=to) for g in grads]
    before = [g.clone() for g in grads]
    got = oz.clip_gradients(grads, max_norm, eps=eps, out=outs)
    assert got.dtype == torch.float32 and got.shape == ()
    assert abs(got.item() - norm) <= 36 * 2.0 ** -24 * norm
    for g, o, w, b in zip(grads, outs or grads, want, before):
        if outs is not None:
            assert torch.equal(g, b)
        bound = UNIT[o.dtype] * w.abs() + 40 * 2.0 ** -24 * w.abs() + TINY[o.dtype]
        assert bool(((o.double() - w).abs() <= bound).all())
    return got


SIZES = [[1], [7, 1, 33], [8192], [8191, 8193, 16384], [100000, 3, 0, 77777], [1] * 70, [5000] * 700, [3000001]]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{s[0]}")
def test_clip(sizes, dtype):
    g = generator(len(sizes) + sizes[0])
    grads = [torch.randn(n, generator=g, device=DEV).to(dtype) for n in sizes]
    norm, _ = define(grads, 1.0)
    for to in (torch.float32, dtype, torch.bfloat16):
        check(grads, 0.3 * norm, to)
    check([v.clone() for v in grads], 2 * norm)         # nothing to clip: unchanged
    check(grads, 0.3 * norm)
    assert oz.device_status() == 0


def test_types_shapes_and_layouts_together():
    g = generator(5)
    base = torch.randn(4000, generator=g, device=DEV)
    grads = [torch.randn(30, 50, generator=g, device=DEV).bfloat16(), torch.randn(3, 4, 5, generator=g, device=DEV).half(),
             torch.randn(40, 60, generator=g, device=DEV).t(), torch.randn((), generator=g, device=DEV),
             base[1:1000], base[1003:3001].half()[1:], torch.randn(6, 8, 10, generator=g, device=DEV).permute(1, 2, 0),
             torch.randn(1, 5, generator=g, device=DEV).expand(1, 5), torch.empty(0, 4, device=DEV)]
    check(grads, 1.5, torch.float32)
    check(grads, 1.5)


def test_special_values():
    zero = [torch.zeros(100, device=DEV), torch.zeros(3, device=DEV).bfloat16()]
    assert check(zero, 1.0).item() == 0
    assert oz.clip_gradients(zero, 1.0, eps=0.0).item() == 0 and not zero[0].any()
    assert oz.clip_gradients([torch.empty(0, device=DEV)], 1.0).item() == 0
    for value in (float("inf"), float("nan")):
        grads = [torch.ones(1000, device=DEV), torch.ones(10, device=DEV)]
        grads[0][77] = value
        norm = oz.clip_gradients(grads, 1.0)
        if value == float("inf"):
            assert norm == float("inf") and not grads[1].any()
            assert grads[0][77].isnan() and not torch.cat([grads[0][:77], grads[0][78:]]).any()
        else:
            assert norm.isnan() and grads[0].isnan().all() and grads[1].isnan().all()
    grads = [torch.ones(10, device=DEV)]
    oz.clip_gradients(grads, 0.0)
    assert not grads[0].any()
    oz.clip_gradients([torch.ones(10, device=DEV)], float("inf"))


def test_no_element_outside_is_touched():
    held = torch.ones(5000, device=DEV).bfloat16()
    grads = [held[1:1000], held[1001:1002], held[1003:4000]]
    oz.clip_gradients(grads, 1e-3)
    edge = torch.ones(5000, dtype=torch.bool, device=DEV)
    for a, b in ((1, 1000), (1001, 1002), (1003, 4000)):
        edge[a:b] = False
    assert bool((held[edge] == 1).all()) and bool((held[~edge] < 0.01).all())


def test_shared_memory_is_refused():
    a, b = torch.ones(100, device=DEV), torch.ones(100, device=DEV)
    for grads, outs in (([a, a], None), ([a[:60], a[40:]], None), ([a, b], [b, a]), ([a, b], [a, a]),
                        ([a[:50], b[:50]], [a[25:75], b[50:]]), ([a.view(10, 10), a.view(10, 10).t()], None)):
        with pytest.raises(oz.OzakiError, match="memory"):
            oz.clip_gradients(grads, 1.0, out=outs)
    assert bool((a == 1).all()) and bool((b == 1).all())
    oz.clip_gradients([a[:50], a[50:]], 1.0)
    oz.clip_gradients([a, b], 1.0, out=[a, b])
    oz.clip_gradients([a, a], 1.0, out=[b, torch.empty_like(b)])      # read twice: counted twice


def test_a_gradient_that_a_graph_needs_is_seen_to_have_changed():
    x = torch.ones(4, device=DEV, requires_grad=True)
    v = x * 2
    y = v.square()
    oz.clip_gradients([v.detach()], 0.1)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()
