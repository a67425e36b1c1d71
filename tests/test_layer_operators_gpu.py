"""The operators around an expert layer's products together: a whole layer forward and
backward, in CUDA graphs, on streams and threads side by side, past 32-bit
offsets.  Needs a B200."""

import math
import threading

import pytest
import torch

import ozaki_triton_b200 as oz

pytestmark = pytest.mark.gpu

DEV = "cuda"


def generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


# ---------------------------------------------------------------------------
# a layer
# ---------------------------------------------------------------------------
def weights_of(g, width=96, hidden=160, experts=6, dtype=torch.bfloat16):
    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV) / math.sqrt(shape[-2])

    return dict(router=normal(width, experts).to(dtype), up=normal(experts, width, hidden).to(dtype),
                down=normal(experts, hidden, width).to(dtype), dense=normal(width, width).to(dtype),
                bias=(0.3 * torch.randn(width, generator=g, device=DEV)).to(dtype))


def layer(x, w, picks=2):
    """x + combine(experts(dispatch(x))) and a dense layer beside it, and the balance loss."""
    scores = oz.fused_matmul(x, w["router"], out_dtype=torch.float32)
    routing = oz.route(scores, picks, normalize=True)
    rows = oz.dispatch(x, routing)
    rows = oz.grouped_matmul(torch.nn.functional.silu(oz.grouped_matmul(rows, w["up"], routing.offsets)), w["down"],
                             routing.offsets)
    y = oz.fused_matmul(x, w["dense"], w["bias"], activation="gelu", residual=oz.combine(rows, routing))
    return y, routing


def layer64(x, w, experts, picks=2):
    """The same in 64 bits, with the picks given."""
    p = torch.softmax(x @ w["router"], 1)
    at = experts.long()
    gate = p.gather(1, at)
    gate = gate / gate.sum(1, keepdim=True)
    u = torch.einsum("td,tkdh->tkh", x, w["up"][at])
    rows = torch.einsum("tkh,tkhd->tkd", u * torch.sigmoid(u), w["down"][at])
    v = x @ w["dense"] + w["bias"]
    y = v * 0.5 * torch.erfc(-v / math.sqrt(2)) + (gate[..., None] * rows).sum(1)
    n = w["router"].shape[1]
    share = torch.bincount(at.flatten(), minlength=n).double() / at.numel()
    return y, n * (share * p.mean(0)).sum()


def test_a_layer_and_its_gradients():
    g = generator(1)
    w = weights_of(g)
    x = torch.randn(300, 96, generator=g, device=DEV).bfloat16()
    leaves = [t.clone().requires_grad_() for t in (x, *w.values())]
    y, routing = layer(leaves[0], dict(zip(w, leaves[1:])))
    dy = torch.randn(300, 96, generator=g, device=DEV).bfloat16()
    got = torch.autograd.grad((y, routing.balance_loss), leaves, (dy, torch.tensor(0.5, device=DEV)))
    exact = [t.double().requires_grad_() for t in (x, *w.values())]
    y64, loss64 = layer64(exact[0], dict(zip(w, exact[1:])), routing.experts)
    want = torch.autograd.grad((y64, loss64), exact, (dy.double(), torch.tensor(0.5, dtype=torch.float64, device=DEV)))
    # Roundings to bf16 on the way of y: hidden rows, their silu, the rows, the combination
    # and y, 5 of them; of a gradient the same ones in what was kept and as many again on the way
    # back (du, rows, hidden rows and their slopes, dispatched rows, the result).  Each is off by
    # at most 2^-8 of an element, 2^-8 / sqrt(3) of a norm, and they add up at most linearly;
    # matrices of independent elements keep a relative error of a norm within a factor of 2.
    def near(a, b, roundings):
        assert (a.double() - b).norm() <= 2 * roundings * 2.0 ** -8 / math.sqrt(3) * b.norm()

    near(y, y64.detach(), 5)
    assert abs(routing.balance_loss.double() - loss64) <= 1e-5
    for a, b in zip(got, want):
        near(a, b, 11)
    assert oz.device_status() == 0


def test_padded_tokens_change_nothing():
    g = generator(2)
    w = weights_of(g)
    x = torch.randn(200, 96, generator=g, device=DEV).bfloat16()
    scores = oz.fused_matmul(x, w["router"], out_dtype=torch.float32)
    padded = torch.cat([scores, scores.new_full((56, 6), -float("inf"))])
    wide = torch.cat([x, x.new_full((56, 96), float("nan"))])
    found = []
    for s, v in ((scores, x), (padded, wide)):
        r = oz.route(s, 2)
        rows = oz.grouped_matmul(oz.dispatch(v, r), w["up"], r.offsets)
        found.append((r, oz.combine(rows, r)))
    (a, y), (b, z) = found
    assert torch.equal(a.experts, b.experts[:200]) and torch.equal(a.slots, b.slots[:200])
    assert torch.equal(a.weights, b.weights[:200]) and torch.equal(a.offsets, b.offsets)
    assert torch.equal(y, z[:200]) and not z[200:].any()
    assert bool((a.balance_loss - b.balance_loss).abs() <= 1e-6 * a.balance_loss)


def test_a_training_step():
    g = generator(3)
    w = weights_of(g)
    x = torch.randn(256, 96, generator=g, device=DEV).bfloat16()
    leaves = {k: t.clone().requires_grad_() for k, t in w.items()}
    y, routing = layer(x, leaves)
    (y.float().square().mean() + 0.01 * routing.balance_loss).backward()
    grads = [t.grad for t in leaves.values()]
    held = [torch.empty_like(t, dtype=torch.float32) for t in grads]
    before = [t.clone() for t in grads]
    norm = oz.clip_gradients(grads, 0.01, out=held)
    want = math.sqrt(sum(float(t.double().square().sum()) for t in before))
    assert abs(norm.item() - want) <= 1e-5 * want and want > 0.01
    for t, b in zip(held, before):
        assert bool(((t.double() - b.double() * 0.01 / (want + 1e-6)).abs() <= 1e-5 * b.double().abs()).all())
    update = oz.orthogonalize(held[1])
    assert update.shape == w["up"].shape and bool(update.isfinite().all())


# ---------------------------------------------------------------------------
# graphs, streams, threads
# ---------------------------------------------------------------------------
def inputs(seed):
    g = generator(seed)

    def normal(*shape, dtype=torch.bfloat16):
        return torch.randn(shape, generator=g, device=DEV).to(dtype)

    return {"x": normal(900, 264), "w": normal(264, 320), "odd": normal(264, 321), "b": normal(320), "r": normal(900, 320),
            "dy": normal(900, 320), "pre": normal(900, 320), "few": normal(3, 264),
            "scores": normal(900, 40, dtype=torch.float32), "dweights": normal(900, 3, dtype=torch.float32),
            "dloss": normal(dtype=torch.float32), "rows": normal(2700, 264), "thin": normal(2700, 33),
            "g0": normal(100000), "g1": normal(33, 7, dtype=torch.float32)}


def everything(v):
    out = [oz.fused_matmul(v["x"], v["w"], v["b"], activation="gelu", residual=v["r"]),
           oz.fused_matmul(v["few"], v["w"], v["b"], activation="silu"), oz.fused_matmul(v["x"], v["odd"]),
           *oz.fused_matmul_backward(v["dy"], v["x"], v["w"], v["pre"], activation="silu", bias=True)]
    r = oz.route(v["scores"], 3, normalize=True)
    few = oz.route(v["scores"][:8], 3)
    out += [*r, *few, oz.route_backward(v["dweights"], v["dloss"], v["scores"], r, normalize=True), oz.dispatch(v["x"], r),
            oz.combine(v["rows"], r), oz.combine(v["thin"], r), oz.dispatch_backward(v["rows"], r),
            *oz.combine_backward(v["x"], v["rows"], r)]
    clipped = [torch.empty_like(v["g0"], dtype=torch.float32), torch.empty_like(v["g1"])]
    out += [oz.clip_gradients([v["g0"], v["g1"]], 1.0, out=clipped), *clipped]
    return out


def through_autograd(v):
    x, w, b, scores = (v[k].detach().requires_grad_() for k in ("x", "w", "b", "scores"))
    r = oz.route(scores, 3, normalize=True)
    rows = oz.dispatch(oz.fused_matmul(x, w, b, activation="gelu"), r)
    y = oz.combine(rows, r)
    return torch.autograd.grad((y, r.balance_loss), (x, w, b, scores), (v["dy"], v["dloss"]))


@pytest.mark.parametrize("work", [everything, through_autograd])
def test_graphs_follow_their_inputs(work):
    held = inputs(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(held)
    torch.cuda.current_stream().wait_stream(side)
    graphs, found = [], []
    for _ in range(2):                    # two graphs: neither writes into the other's results
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            found.append(work(held))
        graphs.append(graph)
    for seed in (1, 2, 3):
        fresh = inputs(seed)
        want = work(fresh)
        for name, t in held.items():
            t.copy_(fresh[name])
        graphs[seed % 2].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(found[seed % 2], want))
    assert oz.device_status() == 0


def test_streams_side_by_side():
    sets = [inputs(seed) for seed in range(4)]
    want = [everything(v) for v in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    found = [[] for _ in sets]
    for _ in range(8):
        for v, stream, out in zip(sets, streams, found):
            with torch.cuda.stream(stream):
                out.append(everything(v))
    torch.cuda.synchronize()
    for runs, expected in zip(found, want):
        for run in runs:
            assert all(torch.equal(a, b) for a, b in zip(run, expected))
    assert oz.device_status() == 0


def test_threads_side_by_side():
    sets = [inputs(seed) for seed in range(4)]
    want = [everything(v) for v in sets]
    torch.cuda.synchronize()
    wrong = []

    def run(v, expected):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(6):
                    got = everything(v)
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, expected)):
                        wrong.append("other results")
        except Exception as e:            # noqa: BLE001
            wrong.append(repr(e))

    threads = [threading.Thread(target=run, args=pair) for pair in zip(sets, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_results_repeat():
    v = inputs(5)
    first = everything(v)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(everything(v), first))


# ---------------------------------------------------------------------------
# sizes past 32 bits
# ---------------------------------------------------------------------------
def test_products_past_32_bit_offsets():
    rows, k, n = 280000, 24, 8192                     # 2.3e9 results
    g = generator(1)
    x = torch.randint(-2, 3, (rows, k), generator=g, device=DEV).bfloat16()
    w = torch.randint(-2, 3, (k, n), generator=g, device=DEV).bfloat16()
    r = torch.zeros(1, n, device=DEV).bfloat16().expand(rows, n)
    y, pre = oz.fused_matmul(x, w, activation="relu", residual=r, return_pre=True)
    dx, dw, db = oz.fused_matmul_backward(y, x, w, pre, activation="relu", bias=True, dw_dtype=torch.float32)
    for a, b in ((0, 300), (262100, 262500), (rows - 300, rows)):
        u = x[a:b].double() @ w.double()
        assert torch.equal(y[a:b].double(), u.clamp(min=0)) and torch.equal(pre[a:b].double(), u)
        assert torch.equal(dx[a:b], (u.clamp(min=0) @ w.double().t()).bfloat16())
    assert oz.device_status() == 0


def test_rows_past_32_bit_offsets():
    tokens, picks, d = 300000, 2, 4096                # 2.5e9 elements of rows
    g = generator(2)
    r = oz.route(torch.randn(tokens, 8, generator=g, device=DEV), picks)
    x = torch.randn(tokens, d, generator=g, device=DEV).bfloat16()
    rows = oz.dispatch(x, r)
    y = oz.combine(rows, r)
    drows, dweights = oz.combine_backward(x, rows, r)
    for a, b in ((0, 200), (149900, 150100), (tokens - 200, tokens)):
        at = r.slots[a:b].long()
        assert torch.equal(rows[at], x[a:b, None].expand(-1, picks, -1))
        want = x[a:b].double() * r.weights[a:b].double().sum(1, keepdim=True)
        assert bool(((y[a:b].double() - want).abs() <= (2.0 ** -8 + 2.0 ** -20) * want.abs()).all())
        want = x[a:b, None].double() * r.weights[a:b, :, None].double()
        assert bool(((drows[at].double() - want).abs() <= (2.0 ** -8 + 2.0 ** -20) * want.abs()).all())
        size = x[a:b].double().square().sum(1, keepdim=True)
        assert bool(((dweights[a:b].double() - size).abs() <= (d + 2) * 2.0 ** -24 * size).all())
    del rows, drows
    odd = x.flatten()[:tokens * 4095].view(tokens, 4095)
    rows = oz.dispatch(odd, r)
    back = oz.combine(rows, r)
    for a, b in ((0, 200), (tokens - 200, tokens)):
        assert torch.equal(rows[r.slots[a:b].long()], odd[a:b, None].expand(-1, picks, -1))
        want = odd[a:b].double() * r.weights[a:b].double().sum(1, keepdim=True)
        assert bool(((back[a:b].double() - want).abs() <= (2.0 ** -8 + 2.0 ** -20) * want.abs()).all())


def test_logits_past_32_bit_offsets():
    tokens, e = 2400000, 1000                         # 2.4e9 logits
    g = generator(3)
    logits = torch.randn(tokens, e, generator=g, device=DEV, dtype=torch.float16)
    r = oz.route(logits, 2)
    d = oz.route_backward(r.weights, None, logits, r)
    for a, b in ((0, 300), (tokens - 300, tokens)):
        v, i = logits[a:b].sort(dim=1, descending=True, stable=True)
        assert torch.equal(r.experts[a:b].long(), i[:, :2])
        p = torch.softmax(logits[a:b].double(), 1)
        assert bool((r.weights[a:b].double() - p.gather(1, i[:, :2])).abs().max() <= 1e-4)
        w = r.weights[a:b].double()
        slope = torch.zeros_like(p).scatter_(1, i[:, :2], w)
        want = p * (slope - (p * slope).sum(1, keepdim=True))
        assert bool((d[a:b].double() - want).abs().max() <= 2.0 ** -11 * want.abs().max() + 2.0 ** -24)
    assert int(r.offsets[-1]) == 2 * tokens
    places = torch.zeros(2 * tokens, dtype=torch.bool, device=DEV)
    places[r.slots.flatten().long()] = True
    assert bool(places.all())


def test_gradients_past_32_bit_offsets():
    big = torch.ones(2 ** 31 + 5, device=DEV, dtype=torch.bfloat16)
    small = torch.ones(3, device=DEV)
    norm = oz.clip_gradients([small, big], 1.0)
    want = math.sqrt(2 ** 31 + 8)
    assert abs(norm.item() - want) <= 1e-6 * want
    one = torch.tensor(1 / want).bfloat16().item()
    assert bool((big[:1000] == one).all()) and bool((big[-1000:] == one).all()) and big.float().amax() == one


def test_calls_that_reuse_memory_follow_one_another():
    # a kernel may start while those before it run: the routing, the sums and the rows of each turn
    # stand where those of the turn before stood, and no other kernel comes between
    torch.manual_seed(3)
    scores = [torch.randn(96, 16, device="cuda") for _ in range(8)]
    x = torch.randn(96, 64, device="cuda", dtype=torch.bfloat16)
    w = torch.randn(64, 64, device="cuda", dtype=torch.bfloat16)
    grads = [torch.randn(5000, device="cuda") * (i + 1) for i in range(8)]
    spare = torch.empty(5000, device="cuda")

    def turn(i):
        r = oz.route(scores[i], 2)
        rows = oz.dispatch(x, r)
        y = oz.combine(rows, r)
        u = oz.fused_matmul(y, w, residual=y)
        return y, u, oz.clip_gradients([grads[i]], 1.0, out=[spare])

    want = []
    for i in range(8):
        want.append(turn(i))
        torch.cuda.synchronize()
    for _ in range(20):
        found = [turn(i) for i in range(8)]
        for a, b in zip(found, want):
            assert all(torch.equal(s, t) for s, t in zip(a, b))
