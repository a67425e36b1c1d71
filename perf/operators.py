"""The operators of a mixture-of-experts layer that is trained and served, as measured cases.

Four operators: the ragged products of an expert layer (``experts``), their
gradients (``experts_grad``), the products of a few rows with 4-bit expert
weights (``w4``), and the Newton-Schulz orthogonalisation of a weight update
(``orthogonalize``).  With ``own`` false ``run`` computes each from elementary
torch operations in 32 bits; with ``own`` true it calls the package.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}

# quintic Newton-Schulz coefficients (a, b, c) of X <- aX + (bA + cA^2)X, A = XX^T
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
EPS = 1e-7


def listed():
    return [
        # one decoding step of a small batch: a few rows per expert, some experts without any
        {"name": "experts decode", "op": "experts", "dtype": "bf16", "t": 16, "e": 8, "k": 1024, "n": 2048},
        # a short chunk with sizes that fit no tile, and rows that start at odd addresses
        {"name": "experts odd", "op": "experts", "dtype": "fp16", "t": 1003, "e": 12, "k": 1000, "n": 1407},
        # a long prompt through fine-grained experts
        {"name": "experts prompt", "op": "experts", "dtype": "bf16", "t": 32768, "e": 64, "k": 2048, "n": 2816},
        # a training micro-batch, fp32 weight gradients
        {"name": "experts grad", "op": "experts_grad", "dtype": "fp16", "t": 3989, "e": 16, "k": 1024, "n": 1536},
        # a full training batch through wide experts
        {"name": "experts grad large", "op": "experts_grad", "dtype": "bf16", "t": 32768, "e": 16, "k": 4096, "n": 2048},
        # one token against one quantised projection: latency
        {"name": "w4 token", "op": "w4", "dtype": "bf16", "t": 1, "e": 1, "k": 2048, "n": 2048, "group": 128, "zeros": False},
        # the same with odd sizes, small groups and zero points
        {"name": "w4 odd", "op": "w4", "dtype": "fp16", "t": 3, "e": 1, "k": 4256, "n": 4099, "group": 32, "zeros": True},
        # a decoding batch against a large projection: the weights' bytes
        {"name": "w4 batch", "op": "w4", "dtype": "fp16", "t": 8, "e": 1, "k": 8192, "n": 28672, "group": 128, "zeros": True},
        # a decoding batch through quantised experts
        {"name": "w4 experts", "op": "w4", "dtype": "bf16", "t": 24, "e": 64, "k": 2048, "n": 2816, "group": 64, "zeros": False},
        # updates of many small matrices, tall ones
        {"name": "orthogonalize small", "op": "orthogonalize", "dtype": "fp32", "batch": 12, "m": 250, "n": 64, "steps": 5},
        # the update of one expert layer in training precision
        {"name": "orthogonalize experts", "op": "orthogonalize", "dtype": "bf16", "batch": 4, "m": 2048, "n": 2816, "steps": 5},
        # a large square update kept in 32 bits
        {"name": "orthogonalize large", "op": "orthogonalize", "dtype": "fp32", "batch": 1, "m": 4096, "n": 4096, "steps": 5},
    ]


def _spread(rng, low, high, multiple=1):
    """A whole number between low and high, even over its logarithm."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return max(multiple, v // multiple * multiple)


def _drawn(rng):
    op = rng.choice(["experts", "experts_grad", "w4", "orthogonalize"])
    if op == "orthogonalize":
        return {"op": op, "dtype": rng.choice(["bf16", "fp32", "fp16"]), "batch": _spread(rng, 1, 16),
                "m": _spread(rng, 16, 4096), "n": _spread(rng, 16, 4096), "steps": rng.choice([3, 5, 6])}
    if op == "w4":
        group = rng.choice([32, 64, 128])
        return {"op": op, "dtype": rng.choice(["bf16", "fp16"]), "t": _spread(rng, 1, 32), "e": rng.choice([1, 1, 8, 64]),
                "k": _spread(rng, 256, 16384, group), "n": _spread(rng, 256, 32768), "group": group,
                "zeros": rng.choice([True, False])}
    return {"op": op, "dtype": rng.choice(["bf16", "fp16"]), "t": _spread(rng, 1, 32768), "e": _spread(rng, 1, 64),
            "k": _spread(rng, 64, 4096, rng.choice([1, 8, 64])), "n": _spread(rng, 64, 4096, rng.choice([1, 8, 64]))}


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        m = most.setdefault(c["op"], {"bytes": 0.0, "flops": 0.0})
        m["bytes"], m["flops"] = max(m["bytes"], w["bytes"]), max(m["flops"], w["flops"])
    while True:
        case = _drawn(rng)
        w, m = work(case), most[case["op"]]
        if 3072 not in case.values() and w["bytes"] <= m["bytes"] and w["flops"] <= m["flops"]:
            return case


def _routed(case, generator):
    """Row offsets of the experts' groups: rows routed at random to unevenly popular experts."""
    logits = 0.5 * torch.randn(case["e"], generator=generator, device="cuda")
    picks = torch.multinomial(torch.softmax(logits, 0), case["t"], replacement=True, generator=generator)
    offsets = torch.zeros(case["e"] + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = torch.cumsum(torch.bincount(picks, minlength=case["e"]), 0)
    return offsets


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    state = {"case": case}
    if case["op"] == "orthogonalize":
        # a gradient: a few strong directions over a noise floor
        b, m, n = case["batch"], case["m"], case["n"]
        rank = max(1, min(m, n) // 16)
        left = torch.randn(b, m, rank, generator=g, device="cuda")
        right = torch.randn(b, rank, n, generator=g, device="cuda")
        noise = torch.randn(b, m, n, generator=g, device="cuda")
        state["grad"] = (1e-3 * (left @ right / math.sqrt(rank) + 0.5 * noise)).to(dtype)
        return state
    t, e, k, n = case["t"], case["e"], case["k"], case["n"]
    state["offsets"] = _routed(case, g)
    state["x"] = normal(t, k)
    if case["op"] == "w4":
        groups = k // case["group"]
        state["packed"] = torch.randint(0, 256, (e, n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
        scale = 0.2 / math.sqrt(k)
        state["scales"] = ((0.5 + torch.rand(e, n, groups, generator=g, device="cuda")) * scale).to(dtype)
        state["zeros"] = (torch.randint(0, 16, (e, n, groups), generator=g, device="cuda", dtype=torch.uint8)
                          if case["zeros"] else None)
        return state
    state["w"] = normal(e, k, n, scale=1.0 / math.sqrt(k))
    state["capacity"] = int((state["offsets"][1:] - state["offsets"][:-1]).max())  # rows of the fullest expert
    if case["op"] == "experts_grad":
        state["dy"] = normal(t, n)
    return state


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _slots(state):
    """(experts, capacity) row of each slot and whether the slot holds one."""
    offsets, rows = state["offsets"].long(), state["x"].shape[0]
    j = torch.arange(state["capacity"], device="cuda")
    held = j < (offsets[1:] - offsets[:-1])[:, None]
    return torch.where(held, offsets[:-1, None] + j, rows), held


def _to_slots(v, row):
    """Rows of v in their slots, zeros in the empty ones, in 32 bits."""
    return torch.cat([v.float(), v.new_zeros(1, v.shape[1], dtype=torch.float32)])[row]


def _from_slots(v, row, rows):
    out = v.new_zeros(rows + 1, v.shape[-1])
    out[row] = v
    return out[:rows]


def _plain_experts(state):
    x, w = state["x"], state["w"]
    row, _ = _slots(state)
    return _from_slots(_to_slots(x, row) @ w.float(), row, x.shape[0]).to(x.dtype)


def _plain_experts_grad(state):
    x, w, dy = state["x"], state["w"], state["dy"]
    row, _ = _slots(state)
    xs, gs = _to_slots(x, row), _to_slots(dy, row)
    dx = _from_slots(gs @ w.float().transpose(1, 2), row, x.shape[0]).to(x.dtype)
    return dx, xs.transpose(1, 2) @ gs


def _plain_w4(state):
    case, x = state["case"], state["x"]
    rows = torch.arange(x.shape[0], device="cuda")
    expert = torch.searchsorted(state["offsets"].long(), rows, right=True) - 1
    if case["e"] == 1:
        expert = expert[:1]
    packed = state["packed"][expert]
    q = torch.stack([packed & 15, packed >> 4], -1).flatten(-2).float().unflatten(-1, (-1, case["group"]))
    zero = 8.0 if state["zeros"] is None else state["zeros"][expert].float().unsqueeze(-1)
    w = ((q - zero) * state["scales"][expert].float().unsqueeze(-1)).flatten(-2)
    if case["e"] == 1:
        return (x.float() @ w[0].t()).to(x.dtype)
    return (w @ x.float().unsqueeze(-1)).squeeze(-1).to(x.dtype)


def _plain_orthogonalize(state):
    grad = state["grad"]
    a, b, c = COEFFICIENTS
    x = grad.float()
    tall = x.shape[-2] > x.shape[-1]
    x = x.transpose(-2, -1) if tall else x
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + EPS)
    for _ in range(state["case"]["steps"]):
        s = x @ x.transpose(-2, -1)
        x = a * x + (b * s + c * (s @ s)) @ x
    return (x.transpose(-2, -1) if tall else x).to(grad.dtype).contiguous()


# ---------------------------------------------------------------------------
# the package's calls
# ---------------------------------------------------------------------------
def _own(state):
    import ozaki_triton_b200 as oz

    case = state["case"]
    if case["op"] == "experts":
        return oz.grouped_matmul(state["x"], state["w"], state["offsets"])
    if case["op"] == "experts_grad":
        return oz.grouped_matmul_backward(state["dy"], state["x"], state["w"], state["offsets"],
                                          dw_dtype=torch.float32)
    if case["op"] == "w4":
        if case["e"] == 1:
            return oz.matmul_w4(state["x"], state["packed"][0], state["scales"][0],
                                None if state["zeros"] is None else state["zeros"][0])
        return oz.matmul_w4(state["x"], state["packed"], state["scales"], state["zeros"],
                            offsets=state["offsets"])
    return oz.orthogonalize(state["grad"], steps=case["steps"], coefficients=COEFFICIENTS, eps=EPS)


def run(state):
    if own:
        return _own(state)
    return {"experts": _plain_experts, "experts_grad": _plain_experts_grad, "w4": _plain_w4,
            "orthogonalize": _plain_orthogonalize}[state["case"]["op"]](state)


def work(case):
    es = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "orthogonalize":
        m, n = sorted((case["m"], case["n"]))
        # XX^T and A^2 are symmetric: half of each product; then (bA + cA^2) X
        flops = case["steps"] * (m * m * n + m * m * m + 2 * m * m * n)
        return {"bytes": 2.0 * case["batch"] * m * n * es, "flops": float(case["batch"] * flops)}
    t, e, k, n = case["t"], case["e"], case["k"], case["n"]
    used = e * (1.0 - (1.0 - 1.0 / e) ** t)  # experts that rows are expected to reach
    offsets = 4 * (e + 1)
    if case["op"] == "w4":
        groups = k // case["group"]
        weight = n * k / 2 + n * groups * (es + (1 if case["zeros"] else 0))
        return {"bytes": used * weight + t * (k + n) * es + (offsets if e > 1 else 0), "flops": 2.0 * t * k * n}
    if case["op"] == "experts":
        return {"bytes": used * k * n * es + t * (k + n) * es + offsets, "flops": 2.0 * t * k * n}
    return {"bytes": used * k * n * es + t * (2 * k + n) * es + 4.0 * e * k * n + offsets, "flops": 4.0 * t * k * n}


# ---------------------------------------------------------------------------
# the definitions in 64 bits, expert by expert and matrix by matrix
# ---------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "orthogonalize":
        a, b, c = COEFFICIENTS
        found = []
        for grad in state["grad"].double():
            x = grad / (torch.sqrt((grad * grad).sum()) + EPS)
            for _ in range(case["steps"]):
                # the right-hand form X (aI + bA + cA^2) with A = X^T X where that is the smaller square
                if x.shape[0] > x.shape[1]:
                    s = x.t() @ x
                    x = x @ (a * torch.eye(len(s), dtype=s.dtype, device=s.device) + b * s + c * s @ s)
                else:
                    s = x @ x.t()
                    x = (a * torch.eye(len(s), dtype=s.dtype, device=s.device) + b * s + c * s @ s) @ x
            found.append(x)
        return torch.stack(found)
    bounds = state["offsets"].tolist()
    x = state["x"].double()
    if case["op"] == "w4":
        y = torch.zeros(case["t"], case["n"], dtype=torch.float64, device="cuda")
        for e in range(case["e"]):
            low, high = bounds[e], bounds[e + 1]
            if low == high:
                continue
            w = torch.empty(case["n"], case["k"], dtype=torch.float64, device="cuda")
            w[:, 0::2] = (state["packed"][e] % 16).double()
            w[:, 1::2] = (state["packed"][e] // 16).double()
            w -= 8.0 if state["zeros"] is None else state["zeros"][e].double().repeat_interleave(case["group"], 1)
            w *= state["scales"][e].double().repeat_interleave(case["group"], 1)
            y[low:high] = x[low:high] @ w.t()
        return y
    w = state["w"]
    if case["op"] == "experts":
        return torch.cat([x[bounds[e]:bounds[e + 1]] @ w[e].double() for e in range(case["e"])])
    dy = state["dy"].double()
    parts = [(x[bounds[e]:bounds[e + 1]], dy[bounds[e]:bounds[e + 1]]) for e in range(case["e"])]
    return (torch.cat([g @ w[e].double().t() for e, (_, g) in enumerate(parts)]),
            torch.stack([v.t() @ g for v, g in parts]))
