"""The router, its gradient and the rows' way to the experts and back, against their
definitions in 64 bits.  Needs a B200.

Picks, slots and counts are whole numbers and have to be equal.  A weight is
off by the rounding of exp's argument (d 2^-24 of it, d the distance to the
row's largest logit), of exp itself, of a sum of E terms and of a quotient:
(d + E + 8) 2^-24 of its value.
"""

import pytest
import torch

import ozaki_triton_b200 as oz

pytestmark = pytest.mark.gpu

DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
UNIT = {d: torch.finfo(d).eps / 2 for d in DTYPES}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -126}
INF = float("inf")


def generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def define(logits, picks, normalize):
    """(p, weights, experts, slots, offsets, counts, tokens, loss)."""
    t, e = logits.shape
    v = logits.double()
    held = (v > -INF).any(1)
    p = torch.zeros_like(v)
    p[held] = torch.softmax(v[held], 1)
    order = torch.sort(v, dim=1, descending=True, stable=True).indices[:, :picks]
    real = v.gather(1, order) > -INF
    weights = p.gather(1, order) * real
    if normalize:
        weights = weights / weights.sum(1, keepdim=True).clamp(min=1e-300)
    experts = torch.where(real, order, -1)
    taken = torch.zeros(t, e + 1, dtype=torch.long, device=DEV)
    taken.scatter_(1, torch.where(real, order, e), 1)
    taken = taken[:, :e]
    counts = taken.sum(0)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    rows = offsets[:-1] + taken.cumsum(0) - taken
    slots = torch.where(real, rows.gather(1, order), -1)
    tokens = int(held.sum())
    loss = e * (counts.double() / max(1, int(counts.sum())) * p.sum(0) / max(1, tokens)).sum()
    return p, weights, experts, slots, offsets, counts, tokens, loss


def check(logits, picks, normalize):
    got = oz.route(logits, picks, normalize=normalize)
    p, weights, experts, slots, offsets, counts, tokens, loss = define(logits, picks, normalize)
    for name, t in (("experts", experts), ("slots", slots), ("offsets", offsets), ("counts", counts)):
        v = getattr(got, name)
        assert v.dtype == torch.int32 and torch.equal(v.long(), t), name
    assert got.tokens.item() == tokens
    finite = logits.double().clamp(min=-1e30)
    spread = (finite.max(1, keepdim=True).values - torch.where(logits > -INF, finite, finite.max(1, keepdim=True).values))
    d = spread.max().clamp(max=110).item() if logits.numel() else 0.0
    e = logits.shape[1]
    assert got.weights.dtype == torch.float32
    assert bool(((got.weights.double() - weights).abs() <= (d + e + 8) * 2.0 ** -24 * weights + 2.0 ** -126).all())
    # the loss adds positive terms: those of a thread and of a block in fp32, at most 300 in a row
    assert abs(got.balance_loss.double() - loss) <= (d + e + 308) * 2.0 ** -24 * loss
    return got


CASES = [(1, 1, 1), (1, 64, 6), (7, 8, 8), (8, 64, 6), (33, 5, 3), (100, 9, 2), (129, 16, 4), (250, 20, 1), (256, 64, 8),
         (257, 64, 8), (300, 33, 7), (511, 100, 5), (1000, 128, 8), (1500, 130, 3), (2048, 256, 8), (700, 257, 32),
         (900, 512, 9), (300, 1000, 17), (4100, 8, 2), (40000, 3, 2), (20000, 61, 6)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,e,picks", CASES)
def test_route(rows, e, picks, dtype):
    g = generator(rows + e)
    logits = (2 * torch.randn(rows, e, generator=g, device=DEV) + torch.randn(e, generator=g, device=DEV)).to(dtype)
    for normalize in (False, True):
        check(logits, picks, normalize)
    # padding, in the middle and at the end, and experts that some tokens may not use
    masked = logits.clone()
    masked[torch.rand(rows, e, generator=g, device=DEV) < 0.4] = -INF
    masked[torch.rand(rows, generator=g, device=DEV) < 0.2] = -INF
    masked[rows - rows // 5:] = -INF
    for normalize in (False, True):
        check(masked, picks, normalize)


def test_many_tokens():
    g = generator(1)
    check(torch.randn(200000, 16, generator=g, device=DEV), 2, True)


@pytest.mark.parametrize("e,picks", [(8, 3), (64, 8), (300, 4)])
def test_ties_and_special_values(e, picks):
    g = generator(e)
    few = torch.randint(-1, 2, (300, e), generator=g, device=DEV).float()
    few[few == 0] = torch.where(torch.rand(int((few == 0).sum()), generator=g, device=DEV) < 0.5, 0.0, -0.0)
    for dtype in DTYPES:
        check(few.to(dtype), picks, False)                           # the lowest index first, also among zeros
    check(torch.zeros(300, e, device=DEV), picks, True)
    check(torch.full((70, e), -INF, device=DEV), picks, True)        # nothing but padding
    low = torch.full((70, e), torch.finfo(torch.float32).min, device=DEV)
    check(low, picks, False)                                         # the lowest value is no mask
    low[:, 1] = 3e38
    got = oz.route(low, picks)
    assert bool((got.experts[:, 0] == 1).all()) and bool((got.weights[:, 0] == 1).all())
    odd = torch.randn(300, e, generator=g, device=DEV)
    odd[5, 2], odd[9, 1], odd[200, 0] = float("nan"), INF, -float("nan")
    got = oz.route(odd, picks)
    clean = torch.ones(300, dtype=torch.bool, device=DEV)
    clean[[5, 9, 200]] = False
    p, weights, experts = define(odd, picks, False)[:3]
    assert torch.equal(got.experts[clean].long(), experts[clean])
    assert got.experts[5, 0] == 2 and got.experts[9, 0] == 1 and got.experts[200, 0] == 0
    assert got.weights[5].isnan().all() and got.balance_loss.isnan() and not got.weights[clean].isnan().any()
    assert int(got.offsets[-1]) == 300 * picks
    assert torch.equal(got.slots.flatten().sort().values.long(), torch.arange(300 * picks, device=DEV))


def test_no_tokens():
    for dtype in DTYPES:
        got = oz.route(torch.zeros(0, 6, device=DEV, dtype=dtype), 2)
        assert got.weights.shape == (0, 2) and not got.offsets.any() and not got.counts.any()
        assert got.tokens.item() == 0 and got.balance_loss.item() == 0
        assert oz.dispatch(torch.zeros(0, 16, device=DEV), got).shape == (0, 16)
        assert oz.combine(torch.zeros(0, 16, device=DEV), got).shape == (0, 16)
        assert oz.route_backward(got.weights, got.balance_loss, torch.zeros(0, 6, device=DEV), got).shape == (0, 6)


def test_strides():
    g = generator(4)
    logits = torch.randn(300, 64, generator=g, device=DEV)
    want = oz.route(logits, 4)
    wide = torch.randn(300, 200, generator=g, device=DEV)
    for view in (wide[:, 3:131:2], wide.new_empty(64, 300).t(), wide[:, 1:65]):
        view.copy_(logits)
        got = oz.route(view, 4)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert torch.equal(oz.route_backward(want.weights, want.balance_loss, view, got),
                           oz.route_backward(want.weights, want.balance_loss, logits, want))


def exact_gradient(logits, routing, dweights, dloss, normalize):
    """(dlogits, bound's size) by the formula."""
    v = logits.double()
    t, e = v.shape
    held = (v > -INF).any(1)
    p = torch.zeros_like(v)
    p[held] = torch.softmax(v[held], 1)
    experts = routing.experts.long()
    real = experts >= 0
    at = experts.clamp(min=0)
    share = routing.counts.double() / max(1, int(routing.counts.sum()))
    g = (dloss.double() * e / max(1, int(routing.tokens)) * share).expand(t, e).clone()
    dw = dweights.double() * real
    w = p.gather(1, at) * real
    if normalize:
        w = w / w.sum(1, keepdim=True).clamp(min=1e-300)
        extra = torch.zeros_like(p).scatter_add_(1, at, w * (dw - (w * dw).sum(1, keepdim=True)))
        size = torch.zeros_like(p).scatter_add_(1, at, w * (dw.abs() + (w * dw.abs()).sum(1, keepdim=True)))
    else:
        g.scatter_add_(1, at, dw)
        extra, size = 0, 0
    found = p * (g - (p * g).sum(1, keepdim=True)) + extra
    return found, p * (g.abs() + (p * g.abs()).sum(1, keepdim=True)) + size


@pytest.mark.parametrize("normalize", [False, True])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,e,picks", CASES)
def test_route_gradient(rows, e, picks, dtype, normalize):
    g = generator(rows * 7 + e)
    logits = (2 * torch.randn(rows, e, generator=g, device=DEV)).to(dtype)
    logits[torch.rand(rows, e, generator=g, device=DEV) < 0.2] = -INF
    logits[torch.rand(rows, generator=g, device=DEV) < 0.2] = -INF
    dweights, dloss = torch.randn(rows, picks, generator=g, device=DEV), torch.tensor(1.7, device=DEV)
    leaf = logits.clone().requires_grad_()
    r = oz.route(leaf, picks, normalize=normalize)
    d = 16.0 + e
    for wanted in ((dweights, dloss), (dweights, None), (None, dloss)):
        outs = [(o, v) for o, v in zip((r.weights, r.balance_loss), wanted) if v is not None]
        (got,) = torch.autograd.grad([o for o, _ in outs], leaf, [v for _, v in outs], retain_graph=True)
        zero = [torch.zeros_like(dweights) if wanted[0] is None else dweights,
                torch.zeros_like(dloss) if wanted[1] is None else dloss]
        want, size = exact_gradient(logits, r, *zero, normalize)
        assert got.dtype == dtype and got.shape == logits.shape
        # p's own bound twice (it stands in the sum too), and a few roundings
        bound = UNIT[dtype] * want.abs() + 3 * (d + 24) * 2.0 ** -24 * size + TINY[dtype]
        assert bool(((got.double() - want).abs() <= bound).all())
        plain = oz.Routing(*(v.detach() for v in r))
        assert torch.equal(oz.route_backward(*wanted, logits, plain, normalize=normalize), got)


@pytest.mark.parametrize("normalize", [False, True])
def test_route_gradient_against_differences(normalize):
    g = generator(2)
    logits = torch.randn(50, 12, generator=g, device=DEV)
    dweights, dloss = torch.randn(50, 3, generator=g, device=DEV), torch.tensor(5.0, device=DEV)
    leaf = logits.clone().requires_grad_()
    r = oz.route(leaf, 3, normalize=normalize)
    (got,) = torch.autograd.grad((r.weights, r.balance_loss), leaf, (dweights, dloss))
    share = r.counts.double() / r.counts.sum()

    def value(v):
        p = torch.softmax(v, 1)
        w = p.gather(1, r.experts.long())
        w = w / w.sum(1, keepdim=True) if normalize else w
        return (w * dweights.double()).sum() + dloss.double() * 12 * (share * p.mean(0)).sum()

    direction = torch.randn(50, 12, generator=g, device=DEV).double()
    step = 1e-6
    want = (value(logits.double() + step * direction) - value(logits.double() - step * direction)) / (2 * step)
    size = exact_gradient(logits, r, dweights, dloss, normalize)[1]
    bound = (size * direction.abs()).sum() * 3 * (16 + 12 + 24) * 2.0 ** -24
    assert (want - (got.double() * direction).sum()).abs() <= bound + 1e-7


# tokens, experts, picks, columns
ROWS = [(1, 4, 1, 1), (3, 4, 2, 8), (50, 6, 3, 33), (100, 8, 2, 64), (129, 64, 8, 130), (300, 16, 4, 256), (70, 12, 9, 1001),
        (33, 40, 17, 2048), (500, 8, 2, 2056), (20, 8, 4, 8200), (1000, 4, 1, 24)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("tokens,e,picks,d", ROWS)
def test_rows_there_and_back(tokens, e, picks, d, dtype):
    g = generator(tokens + d)
    logits = torch.randn(tokens, e, generator=g, device=DEV)
    logits[torch.rand(tokens, e, generator=g, device=DEV) < 0.3] = -INF
    logits[torch.rand(tokens, generator=g, device=DEV) < 0.2] = -INF
    r = oz.route(logits, picks)
    x = torch.randn(tokens, d, generator=g, device=DEV).to(dtype)
    real, n = r.slots >= 0, int(r.offsets[-1])
    rows = oz.dispatch(x, r)
    want = torch.zeros(tokens * picks, d, dtype=dtype, device=DEV)
    want[r.slots[real].long()] = x[:, None].expand(-1, picks, -1)[real]
    assert torch.equal(rows, want) and not rows[n:].any()
    assert torch.equal(oz.dispatch(x.t().contiguous().t(), r), rows)

    results = torch.randn(tokens * picks, d, generator=g, device=DEV).to(dtype)
    results[n:] = float("nan")                                       # no pick's: never read
    at = r.slots.clamp(min=0).long()
    terms = results.double()[at].masked_fill(~real[..., None], 0) * r.weights.double()[..., None]

    def near(got, want, size, count, to=dtype):
        bound = UNIT[to] * want.abs() + (count + 2) * 2.0 ** -24 * size + TINY[to]
        assert got.dtype == to and got.shape == want.shape and bool(((got.double() - want).abs() <= bound).all())

    near(oz.combine(results, r), terms.sum(1), terms.abs().sum(1), picks)
    dy = torch.randn(tokens, d, generator=g, device=DEV).to(dtype)
    drows, dweights = oz.combine_backward(dy, results, r)
    want = torch.zeros(tokens * picks, d, dtype=torch.float64, device=DEV)
    want[r.slots[real].long()] = (dy.double()[:, None] * r.weights.double()[..., None])[real]
    near(drows, want, want.abs(), 1)
    assert not drows[n:].any()
    products = results.double()[at].masked_fill(~real[..., None], 0) * dy.double()[:, None]
    near(dweights, products.sum(-1), products.abs().sum(-1), d, torch.float32)
    back = results.double()[at].masked_fill(~real[..., None], 0)
    near(oz.dispatch_backward(results, r), back.sum(1), back.abs().sum(1), picks)
    # through autograd: the same numbers
    a, b, w = x.clone().requires_grad_(), results.clone().requires_grad_(), r.weights.clone().requires_grad_()
    (dx,) = torch.autograd.grad(oz.dispatch(a, r), a, results)
    assert torch.equal(dx, oz.dispatch_backward(results, r))
    found = torch.autograd.grad(oz.combine(b, r._replace(weights=w)), (b, w), dy)
    assert torch.equal(found[0], drows) and torch.equal(found[1], dweights)


def test_rows_of_other_layouts():
    g = generator(8)
    r = oz.route(torch.randn(90, 8, generator=g, device=DEV), 3)
    x = torch.randn(90, 136, generator=g, device=DEV).bfloat16()
    rows = torch.randn(270, 136, generator=g, device=DEV).bfloat16()

    def changed(t):
        yield t.t().contiguous().t()
        held = torch.full((t.shape[0], t.shape[1] + 9), float("nan"), dtype=t.dtype, device=DEV)
        yield held[:, 1:1 + t.shape[1]].copy_(t)                     # off the 16-byte boundaries
        held = torch.full((t.shape[0], t.shape[1] + 8), float("nan"), dtype=t.dtype, device=DEV)
        yield held[:, 8:].copy_(t)

    for a, b in zip(changed(x), changed(rows)):
        assert torch.equal(oz.dispatch(a, r), oz.dispatch(x, r))
        assert torch.equal(oz.combine(b, r), oz.combine(rows, r))
        assert torch.equal(oz.dispatch_backward(b, r), oz.dispatch_backward(rows, r))
        (drows, dweights), (want, near) = oz.combine_backward(a, b, r), oz.combine_backward(x, rows, r)
        assert torch.equal(drows, want)
        # a thread's share of a row's columns is another one off the 16-byte boundaries: two sums of
        # 136 terms, each off by at most 138 2^-24 of their magnitudes
        size = (rows.double()[r.slots.long()] * x.double()[:, None]).abs().sum(-1)
        assert bool(((dweights.double() - near.double()).abs() <= 2 * 138 * 2.0 ** -24 * size).all())
    one = x[:1].expand(90, 136)
    assert torch.equal(oz.dispatch(one, r), oz.dispatch(one.contiguous(), r))
    turned = r._replace(weights=r.weights.t().contiguous().t())
    assert torch.equal(oz.combine(rows, turned), oz.combine(rows, r))


def test_rows_without_columns():
    r = oz.route(torch.randn(20, 8, device=DEV), 2)
    x, rows = torch.empty(20, 0, device=DEV), torch.empty(40, 0, device=DEV)
    assert oz.dispatch(x, r).shape == (40, 0) and oz.combine(rows, r).shape == (20, 0)
    assert oz.dispatch_backward(rows, r).shape == (20, 0)
    drows, dweights = oz.combine_backward(x, rows, r)
    assert drows.shape == (40, 0) and dweights.shape == (20, 2) and not dweights.any()


def test_a_routing_made_by_hand_stays_in_bounds():
    g = generator(6)
    x = torch.randn(40, 64, generator=g, device=DEV)
    rows = torch.randn(80, 64, generator=g, device=DEV)
    r = oz.route(torch.randn(40, 8, generator=g, device=DEV), 2)
    for bad in (-5, 80, 2 ** 31 - 1, -2 ** 31):
        slots = r.slots.clone()
        slots[3, 1] = bad
        wrong = r._replace(slots=slots)
        y = oz.combine(rows, wrong)
        want = r.weights[3, 0].double() * rows[r.slots[3, 0].long()].double()
        assert bool(((y[3].double() - want).abs() <= 2.0 ** -23 * want.abs()).all())
        assert oz.combine_backward(x, rows, wrong)[1][3, 1] == 0
        assert oz.dispatch(x, wrong).shape == (80, 64)
        for end in (-3, 10 ** 9):
            offsets = r.offsets.clone()
            offsets[-1] = end
            assert oz.dispatch(x, r._replace(offsets=offsets)).shape == (80, 64)
        experts = r.experts.clone()
        experts[3, 1] = bad
        assert oz.route_backward(r.weights, None, torch.randn(40, 8, generator=g, device=DEV),
                                 r._replace(experts=experts)).shape == (40, 8)
