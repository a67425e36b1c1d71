"""A mixture-of-experts layer, trained and then served in 4 bits.

    python examples/expert_layer.py

Every token goes to one of the experts (two products with a SiLU between
them).  Training routes the tokens, runs the ragged products forward and
backward, clips the gradients by their common norm and updates each stack of
expert weights with an orthogonalised momentum; serving quantises the weights to
4 bits and runs a few tokens at a time.
"""

import os
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import ozaki_triton_b200 as oz  # noqa: E402


def layer(x, router, up, down):
    routing = oz.route(x.float() @ router, 1)
    hidden = F.silu(oz.grouped_matmul(oz.dispatch(x, routing), up, routing.offsets))
    return oz.combine(oz.grouped_matmul(hidden, down, routing.offsets), routing)


def layer_4bit(x, router, up4, down4):
    """The same with weights from quantize_w4."""
    routing = oz.route(x.float() @ router, 1)
    hidden = F.silu(oz.matmul_w4(oz.dispatch(x, routing), *up4, offsets=routing.offsets))
    return oz.combine(oz.matmul_w4(hidden, *down4, offsets=routing.offsets), routing)


def main(tokens=2048, width=256, hidden=512, experts=8, steps=60, seed=0, dtype=torch.bfloat16, log=print):
    """Fits a layer to a fixed random one; returns (first loss, last loss, relative error of 4 bits)."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda") / shape[-2] ** 0.5

    router = normal(width, experts)
    target = [normal(experts, width, hidden).to(dtype), normal(experts, hidden, width).to(dtype)]
    weights = [normal(experts, width, hidden), normal(experts, hidden, width)]          # fp32 masters
    momentum = [torch.zeros_like(w) for w in weights]
    clipped = [torch.empty_like(w) for w in weights]
    losses = []
    for step in range(steps):
        x = torch.randn(tokens, width, generator=g, device="cuda").to(dtype)
        with torch.no_grad():
            want = layer(x, router, *target)
        used = [w.to(dtype).requires_grad_() for w in weights]
        loss = F.mse_loss(layer(x, router, *used).float(), want.float())
        loss.backward()
        oz.clip_gradients([u.grad for u in used], 1.0, out=clipped)
        rate = 0.02 * (1 - step / steps)
        for w, m, c in zip(weights, momentum, clipped):
            m.mul_(0.9).add_(c)
            w.sub_(rate * oz.orthogonalize(m))
        losses.append(loss.detach())
        if step % 20 == 0:
            log(f"step {step}: loss {loss.item():.5f}")
    up4, down4 = (oz.quantize_w4(w.to(dtype), 64) for w in weights)
    few = torch.randn(3, width, generator=g, device="cuda").to(dtype)
    with torch.no_grad():
        full = layer(few, router, *(w.to(dtype) for w in weights))
        four = layer_4bit(few, router, up4, down4)
    error = ((four - full).float().norm() / full.float().norm()).item()
    log(f"loss {losses[0].item():.5f} -> {losses[-1].item():.5f}; 4-bit weights change 3 tokens by {100 * error:.1f}%")
    return losses[0].item(), losses[-1].item(), error


if __name__ == "__main__":
    main()
