"""What stands around an expert layer's products when it is trained and served, as measured cases.

Four operators: the product with bias, activation and residual in its epilogue
and its backward pass (``linear``, ``linear_grad``); the router with its picks,
per-expert counts, row order and balance loss and its backward pass (``route``,
``route_grad``); the way of the tokens' rows to their experts and back, with
its backward pass (``rows``); and the clipping of many gradients by their
global norm (``clip``).  With ``own`` false ``run`` computes each from
elementary torch operations in 32 bits; with ``own`` true it calls the package.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
CLIP_EPS = 1e-6


def listed():
    return [
        # one token's projection while serving: latency, and the weights' bytes
        {"name": "linear token", "op": "linear", "dtype": "bf16", "t": 1, "k": 2048, "n": 2816, "act": "silu",
         "bias": True, "residual": False},
        # a short chunk through a layer of odd sizes, added to the residual stream
        {"name": "linear odd", "op": "linear", "dtype": "fp16", "t": 67, "k": 1000, "n": 1407, "act": "none",
         "bias": True, "residual": True},
        # a long prompt through the dense layer beside the experts
        {"name": "linear prompt", "op": "linear", "dtype": "bf16", "t": 8192, "k": 4096, "n": 8192, "act": "gelu",
         "bias": True, "residual": False},
        # the backward pass of a training micro-batch
        {"name": "linear grad", "op": "linear_grad", "dtype": "bf16", "t": 8192, "k": 2048, "n": 8192, "act": "silu",
         "bias": True},
        # one decoding step of a small batch: latency
        {"name": "route token", "op": "route", "dtype": "fp32", "t": 8, "e": 64, "picks": 6, "normalize": True,
         "padded": 0},
        # a long prompt through fine-grained experts, its end padding
        {"name": "route prompt", "op": "route", "dtype": "bf16", "t": 32768, "e": 64, "picks": 8, "normalize": False,
         "padded": 1000},
        # the backward pass of a training batch, many experts
        {"name": "route grad", "op": "route_grad", "dtype": "fp32", "t": 16384, "e": 256, "picks": 8,
         "normalize": True, "padded": 0},
        # rows of an odd width on their way to the experts
        {"name": "dispatch odd", "op": "rows", "step": "dispatch", "dtype": "fp16", "t": 5003, "e": 12, "picks": 2,
         "d": 1001, "padded": 3},
        # a long prompt's rows back from the experts
        {"name": "combine prompt", "op": "rows", "step": "combine", "dtype": "bf16", "t": 32768, "e": 64, "picks": 6,
         "d": 2048, "padded": 0},
        # the backward pass of that in a training micro-batch
        {"name": "combine grad", "op": "rows", "step": "combine_grad", "dtype": "bf16", "t": 8192, "e": 16, "picks": 4,
         "d": 2816, "padded": 0},
        # the gradients of one small layer, some of odd sizes
        {"name": "clip small", "op": "clip", "dtype": "bf16", "to": "bf16", "tensors": 9, "total": 300000,
         "max_norm": 0.25},
        # the gradients of a stack of layers, to 32 bits for the update
        {"name": "clip large", "op": "clip", "dtype": "bf16", "to": "fp32", "tensors": 48, "total": 400000000,
         "max_norm": 1.0},
    ]


def _spread(rng, low, high, multiple=1):
    """A whole number between low and high, even over its logarithm."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return max(multiple, v // multiple * multiple)


def _drawn(rng):
    op = rng.choice(["linear", "linear", "linear_grad", "route", "route_grad", "rows", "rows", "clip"])
    dtype = rng.choice(["bf16", "fp16"])
    if op in ("linear", "linear_grad"):
        case = {"op": op, "dtype": dtype, "t": _spread(rng, 1, 16384), "k": _spread(rng, 64, 8192, rng.choice([1, 8, 64])),
                "n": _spread(rng, 64, 8192, rng.choice([1, 8, 64])), "act": rng.choice(["none", "relu", "gelu", "silu"]),
                "bias": rng.choice([True, False])}
        if op == "linear":
            case["residual"] = rng.choice([True, False])
        return case
    if op == "clip":
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        return {"op": op, "dtype": dtype, "to": rng.choice([dtype, "fp32"]), "tensors": _spread(rng, 1, 60),
                "total": _spread(rng, 1000, 400000000), "max_norm": rng.choice([0.1, 1.0, 1000.0])}
    e = _spread(rng, 2, 512)
    case = {"op": op, "dtype": rng.choice(["bf16", "fp16", "fp32"]), "t": _spread(rng, 1, 32768), "e": e,
            "picks": min(e, rng.randint(1, 8))}
    case["padded"] = rng.choice([0, rng.randint(0, case["t"]) // 3])
    if op == "rows":
        case["step"] = rng.choice(["dispatch", "dispatch_grad", "combine", "combine_grad"])
        case["d"] = _spread(rng, 32, 8192, rng.choice([1, 8, 64]))
    else:
        case["normalize"] = rng.choice([True, False])
    return case


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        m = most.setdefault(c["op"], {"bytes": 0.0, "flops": 0.0})
        m["bytes"], m["flops"] = max(m["bytes"], w["bytes"]), max(m["flops"], w["flops"])
    while True:
        case = _drawn(rng)
        w, m = work(case), most[case["op"]]
        if w["bytes"] <= m["bytes"] and w["flops"] <= m["flops"]:
            return case


def _sizes(case):
    """Elements of each gradient: a few large ones, many small, odd ones among them."""
    rng = random.Random(case["tensors"] * 1000003 + case["total"])
    parts = [math.exp(rng.uniform(0.0, 5.0)) for _ in range(case["tensors"])]
    whole = sum(parts)
    return [max(1, int(case["total"] * p / whole)) for p in parts]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    state = {"case": case}
    if case["op"] == "clip":
        to = DTYPES[case["to"]]
        state["grads"] = [normal(n, scale=1e-3) for n in _sizes(case)]
        state["out"] = [torch.empty_like(v, dtype=to) for v in state["grads"]]
        return state
    t = case["t"]
    if case["op"] in ("linear", "linear_grad"):
        k, n = case["k"], case["n"]
        state["x"], state["w"] = normal(t, k), normal(k, n, scale=1.0 / math.sqrt(k))
        state["bias"] = normal(n, scale=0.5) if case["bias"] else None
        if case["op"] == "linear":
            state["residual"] = normal(t, n) if case["residual"] else None
        else:
            # what the forward pass kept, and the gradient that arrives
            state["pre"] = normal(t, n, scale=1.1) if case["act"] != "none" else None
            state["dy"] = normal(t, n, scale=0.1)
        return state
    e, picks = case["e"], case["picks"]
    # a router's scores: some experts are more popular than others
    state["logits"] = (normal(t, e, scale=1.2).float() + 0.5 * torch.randn(e, generator=g, device="cuda")).to(dtype)
    if case["padded"]:
        state["logits"][t - case["padded"]:] = float("-inf")
    if case["op"] == "route":
        return state
    # what the forward pass returned
    state["routing"] = _plain_route(state["logits"], picks, case.get("normalize", False))
    if case["op"] == "route_grad":
        state["dweights"] = torch.randn(t, picks, generator=g, device="cuda")
        state["dloss"] = torch.rand((), generator=g, device="cuda") + 0.5
        return state
    d = case["d"]
    if case["step"] in ("dispatch", "combine_grad"):
        state["x"] = normal(t, d)                       # tokens, or the gradient of their results
    if case["step"] != "dispatch":
        state["rows"] = normal(t * picks, d)            # the experts' results, or the gradient of their inputs
    del state["logits"]
    return state


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _act(v, name):
    if name == "relu":
        return v * (v > 0)
    if name == "gelu":
        return v * 0.5 * torch.erfc(v * -math.sqrt(0.5))
    if name == "silu":
        return v / (1 + torch.exp(-v))
    return v


def _act_slope(v, name):
    if name == "relu":
        return (v > 0).to(v.dtype)
    if name == "gelu":
        return 0.5 * torch.erfc(v * -math.sqrt(0.5)) + v * torch.exp(-0.5 * v * v) * (1 / math.sqrt(2 * math.pi))
    if name == "silu":
        s = 1 / (1 + torch.exp(-v))
        return s * (1 + v * (1 - s))
    return torch.ones_like(v)


def _plain_linear(state):
    x, act = state["x"], state["case"]["act"]
    v = x.float() @ state["w"].float()
    if state["bias"] is not None:
        v = v + state["bias"].float()
    v = _act(v, act)
    if state["residual"] is not None:
        v = v + state["residual"].float()
    return v.to(x.dtype)


def _plain_linear_grad(state):
    x, w, act = state["x"], state["w"], state["case"]["act"]
    v = state["dy"].float()
    if act != "none":
        v = v * _act_slope(state["pre"].float(), act)
    out = [(v @ w.float().t()).to(x.dtype), (x.float().t() @ v).to(x.dtype)]
    if state["bias"] is not None:
        out.append(v.sum(0))
    return out


def _probabilities(logits):
    """Softmax rows, zeros in rows that hold nothing, and which rows hold something."""
    v = logits.float()
    top = v.max(1, keepdim=True).values
    held = top > float("-inf")
    p = torch.exp(v - torch.where(held, top, torch.zeros_like(top)))
    return torch.where(held, p / p.sum(1, keepdim=True), torch.zeros_like(p)), held[:, 0]


def _plain_route(logits, picks, normalize):
    t, e = logits.shape
    p, held = _probabilities(logits)
    score, chosen = torch.sort(logits.float(), dim=1, descending=True, stable=True)
    real = score[:, :picks] > float("-inf")
    experts = torch.where(real, chosen[:, :picks], torch.full_like(chosen[:, :picks], -1))
    weights = torch.where(real, torch.gather(p, 1, chosen[:, :picks]), torch.zeros_like(p[:, :1]))
    if normalize:
        total = weights.sum(1, keepdim=True)
        weights = weights / torch.where(total > 0, total, torch.ones_like(total))
    # rows in the order of their experts, of their tokens within one
    flat = torch.where(real, experts, torch.full_like(experts, e)).flatten()
    order = torch.argsort(flat, stable=True)
    place = torch.empty_like(order)
    place[order] = torch.arange(len(order), device=order.device)
    slots = torch.where(real, place.view(t, picks), torch.full_like(experts, -1))
    counts = (flat[:, None] == torch.arange(e, device=flat.device)).sum(0) if flat.numel() * e < 1 << 22 else \
        torch.bincount(flat, minlength=e + 1)[:e]
    offsets = torch.cat([counts.new_zeros(1), torch.cumsum(counts, 0)])
    mean = p.sum(0) / held.sum().clamp(min=1)
    share = counts.float() / counts.sum().clamp(min=1)
    whole = (v.int() for v in (experts, slots, offsets, counts, held.sum()))
    return weights, *whole, e * (share * mean).sum()


def _plain_route_grad(state):
    logits, normalize = state["logits"], state["case"]["normalize"]
    weights, experts, _, _, counts, tokens, _ = state["routing"]
    p, _ = _probabilities(logits)
    real = experts >= 0
    at = torch.where(real, experts, torch.zeros_like(experts)).long()
    dw = torch.where(real, state["dweights"], torch.zeros_like(state["dweights"]))
    share = counts.float() / counts.sum().clamp(min=1)
    slope = (state["dloss"] * logits.shape[1] / tokens.clamp(min=1)) * share
    slope = slope.expand_as(p)
    if normalize:
        # the picks' weights are a softmax over themselves
        own_part = weights * (dw - (weights * dw).sum(1, keepdim=True))
        rest = torch.zeros_like(p).scatter_add_(1, at, torch.where(real, own_part, torch.zeros_like(own_part)))
    else:
        slope = slope.scatter_add(1, at, dw)
        rest = 0
    return (p * (slope - (p * slope).sum(1, keepdim=True)) + rest).to(logits.dtype)


def _plain_rows(state):
    case = state["case"]
    weights, _, slots = state["routing"][:3]
    rows = case["t"] * case["picks"]
    at = torch.where(slots < 0, torch.full_like(slots, rows), slots).long()     # one more row for what has none

    def gathered():
        v = state["rows"]
        return torch.cat([v, v.new_zeros(1, v.shape[1])])[at].float()

    if case["step"] == "dispatch":
        x = state["x"]
        out = x.new_zeros(rows + 1, x.shape[1])
        out[at.flatten()] = x[:, None].expand(-1, case["picks"], -1).flatten(0, 1)
        out[rows] = 0
        return out[:rows]
    if case["step"] == "dispatch_grad":
        return gathered().sum(1).to(state["rows"].dtype)
    if case["step"] == "combine":
        return (gathered() * weights.unsqueeze(-1)).sum(1).to(state["rows"].dtype)
    dy = state["x"].float()[:, None]
    out = dy.new_zeros(rows + 1, dy.shape[-1])
    out[at.flatten()] = (dy * weights.unsqueeze(-1)).flatten(0, 1)
    return out[:rows].to(state["rows"].dtype), (gathered() * dy).sum(-1)


def _plain_clip(state):
    grads, case = state["grads"], state["case"]
    norm = torch.stack([v.float().square().sum(dtype=torch.float64) for v in grads]).sum().sqrt().float()
    scale = (case["max_norm"] / (norm + CLIP_EPS)).clamp(max=1.0)
    to = DTYPES[case["to"]]
    return [norm] + [(v.float() * scale).to(to) for v in grads]


# ---------------------------------------------------------------------------
# the package's calls
# ---------------------------------------------------------------------------
def _own(state):
    import ozaki_triton_b200 as oz

    case = state["case"]
    act = case.get("act", "none")
    act = None if act == "none" else act
    if case["op"] == "linear":
        return oz.fused_matmul(state["x"], state["w"], state["bias"], activation=act, residual=state["residual"])
    if case["op"] == "linear_grad":
        out = oz.fused_matmul_backward(state["dy"], state["x"], state["w"], state["pre"], activation=act,
                                       bias=state["bias"] is not None)
        return [v for v in out if v is not None]
    if case["op"] == "clip":
        norm = oz.clip_gradients(state["grads"], case["max_norm"], eps=CLIP_EPS, out=state["out"])
        return [norm] + state["out"]
    if case["op"] == "route":
        return tuple(oz.route(state["logits"], case["picks"], normalize=case["normalize"]))
    routing = oz.Routing(*state["routing"])
    if case["op"] == "route_grad":
        return oz.route_backward(state["dweights"], state["dloss"], state["logits"], routing,
                                 normalize=case["normalize"])
    if case["step"] == "dispatch":
        return oz.dispatch(state["x"], routing)
    if case["step"] == "dispatch_grad":
        return oz.dispatch_backward(state["rows"], routing)
    if case["step"] == "combine":
        return oz.combine(state["rows"], routing)
    return oz.combine_backward(state["x"], state["rows"], routing)


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "route":
        return _plain_route(state["logits"], state["case"]["picks"], state["case"]["normalize"])
    return {"linear": _plain_linear, "linear_grad": _plain_linear_grad, "route_grad": _plain_route_grad,
            "rows": _plain_rows, "clip": _plain_clip}[op](state)


def work(case):
    es = BYTES[case["dtype"]]
    if case["op"] == "clip":
        total = float(sum(_sizes(case)))
        return {"bytes": total * (es + BYTES[case["to"]]), "flops": 3.0 * total}
    t = case["t"]
    if case["op"] == "linear":
        k, n = case["k"], case["n"]
        return {"bytes": float(es * (t * k + k * n + t * n * (2 if case["residual"] else 1) + (n if case["bias"] else 0))),
                "flops": 2.0 * t * k * n}
    if case["op"] == "linear_grad":
        k, n = case["k"], case["n"]
        return {"bytes": float(es * (2 * t * k + 2 * k * n + t * n * (2 if case["act"] != "none" else 1))
                               + (4 * n if case["bias"] else 0)), "flops": 4.0 * t * k * n}
    e, picks, held = case["e"], case["picks"], case["t"] - case["padded"]
    if case["op"] == "route":
        return {"bytes": float(t * e * es + 12 * t * picks + 8 * e + 12), "flops": float(t * e * (4 + picks))}
    if case["op"] == "route_grad":
        return {"bytes": float(2 * t * e * es + 12 * t * picks + 4 * e), "flops": 10.0 * t * e}
    d = case["d"]
    if case["step"] == "dispatch":
        return {"bytes": float(es * d * (held + t * picks) + 4 * t * picks), "flops": 0.0}
    if case["step"] == "dispatch_grad":
        return {"bytes": float(es * d * (t + held * picks) + 4 * t * picks), "flops": float(held * picks * d)}
    if case["step"] == "combine":
        return {"bytes": float(es * d * (t + held * picks) + 8 * t * picks), "flops": 2.0 * held * picks * d}
    return {"bytes": float(es * d * (held + held * picks + t * picks) + 12 * t * picks), "flops": 3.0 * held * picks * d}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _phi(v):
    """The normal distribution's function."""
    return 0.5 * (1 + torch.erf(v / math.sqrt(2)))


def _exact_linear(state):
    v = state["x"].double() @ state["w"].double()
    if state["bias"] is not None:
        v += state["bias"].double()
    act = state["case"]["act"]
    if act == "relu":
        v = v.clamp(min=0)
    elif act == "gelu":
        v = v * _phi(v)
    elif act == "silu":
        v = v * torch.sigmoid(v)
    return v if state["residual"] is None else v + state["residual"].double()


def _exact_linear_grad(state):
    act, v = state["case"]["act"], state["dy"].double()
    if act != "none":
        u = state["pre"].double()
        if act == "relu":
            v[u <= 0] = 0
        elif act == "gelu":
            v = v * (_phi(u) + u * torch.exp(-u * u / 2) / math.sqrt(2 * math.pi))
        else:
            v = v * (torch.sigmoid(u) + u * torch.sigmoid(u) * torch.sigmoid(-u))
    out = [v @ state["w"].double().t(), state["x"].double().t() @ v]
    return out + [v.sum(0)] if state["bias"] is not None else out


def _exact_route(case, logits):
    """Picks by repeated maxima, rows by a count of what comes before."""
    t, e = logits.shape
    picks = case["picks"]
    v = logits.double()
    held = (v > float("-inf")).any(1)
    p = torch.zeros_like(v)
    p[held] = torch.softmax(v[held], 1)
    left, index = v.clone(), torch.arange(e, device=v.device)
    experts = torch.full((t, picks), -1, dtype=torch.int64, device=v.device)
    weights = torch.zeros(t, picks, dtype=torch.float64, device=v.device)
    taken = torch.zeros(t, e, dtype=torch.bool, device=v.device)
    for j in range(picks):
        top = left.max(1, keepdim=True).values
        first = torch.where(left == top, index, e).min(1).values.clamp(max=e - 1)
        real = top[:, 0] > float("-inf")
        experts[real, j] = first[real]
        weights[real, j] = p[real, first[real]]
        left[real, first[real]] = float("-inf")
        taken[real, first[real]] = True
    if case["normalize"]:
        weights /= weights.sum(1, keepdim=True).clamp(min=1e-300)
    counts = taken.sum(0)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    before = taken.cumsum(0) - taken.long()             # earlier tokens of the expert
    row = offsets[:-1] + before
    slots = torch.where(experts >= 0, row.gather(1, experts.clamp(min=0)), -1)
    loss = e * (counts.double() / max(1, int(counts.sum())) * p.sum(0) / max(1, int(held.sum()))).sum()
    return weights, experts, slots, offsets, counts, held.sum(), loss


def _exact_route_grad(state):
    """By differentiation of the weights and the loss."""
    case = state["case"]
    _, experts, _, _, counts, _, _ = state["routing"]
    v = state["logits"].double()
    held = (v > float("-inf")).any(1)
    v = v[held].requires_grad_()
    p = torch.softmax(v, 1)
    real = experts[held] >= 0
    w = p.gather(1, experts[held].long().clamp(min=0)) * real
    if case["normalize"]:
        w = w / w.sum(1, keepdim=True)
    loss = v.shape[1] * (counts.double() / max(1, int(counts.sum())) * p.sum(0) / max(1, v.shape[0])).sum()
    (found,) = torch.autograd.grad((w * state["dweights"][held].double()).sum() + loss * state["dloss"].double(), v)
    out = torch.zeros(state["logits"].shape, dtype=torch.float64, device=v.device)
    out[held] = found
    return out


def _exact_rows(state):
    case = state["case"]
    weights, _, slots = state["routing"][:3]
    t, picks, d = case["t"], case["picks"], case["d"]
    if case["step"] == "combine_grad":
        drows = torch.zeros(t * picks, d, dtype=torch.float64, device=weights.device)
        dweights = torch.zeros(t, picks, dtype=torch.float64, device=weights.device)
    else:
        out = torch.zeros(t * picks if case["step"] == "dispatch" else t, d, dtype=torch.float64, device=weights.device)
    for j in range(picks):
        tokens = (slots[:, j] >= 0).nonzero()[:, 0]
        rows = slots[tokens, j].long()
        w = weights[tokens, j].double()[:, None]
        if case["step"] == "dispatch":
            out[rows] = state["x"][tokens].double()
        elif case["step"] == "dispatch_grad":
            out[tokens] += state["rows"][rows].double()
        elif case["step"] == "combine":
            out[tokens] += w * state["rows"][rows].double()
        else:
            dy = state["x"][tokens].double()
            drows[rows] = w * dy
            dweights[tokens, j] = (dy * state["rows"][rows].double()).sum(1)
    return (drows, dweights) if case["step"] == "combine_grad" else out


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "linear":
        return _exact_linear(state)
    if op == "linear_grad":
        return _exact_linear_grad(state)
    if op == "route":
        return _exact_route(case, state["logits"])
    if op == "route_grad":
        return _exact_route_grad(state)
    if op == "rows":
        return _exact_rows(state)
    norm = math.sqrt(sum(float((v.double() ** 2).sum()) for v in state["grads"]))
    scale = min(1.0, case["max_norm"] / (norm + CLIP_EPS))
    return [torch.tensor(norm, dtype=torch.float64)] + [v.double() * scale for v in state["grads"]]
