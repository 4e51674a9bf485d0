"""Heal a pruned MoE layer and quantize it: the experts that stay are trained in 16 bits towards the
whole layer's output, and stored as 3-bit HEX with GPTQ rounding.

    python examples/heal_experts.py [--steps N]

The path through the operators of blackhole_b200.experts, and the two that the package had around them:

  expert_mlp               the layer's output and, backwards, the gradients of its stacks (grouped
                           products, their transposes, weight gradients, SwiGLU)
  clip_grad_norm           the gradients of both stacks clipped to a common norm
  grouped_mm, swiglu,      every expert's rows on the way through the layer, and from them the
  grouped_wgrad            Hessians sum x x^T of both projections' inputs
  quantize_stack(H=...)    the HEX parts, and hex_moe, which runs them
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "blackhole-harness_b200"))

from blackhole_b200 import experts  # noqa: E402
from blackhole_b200.hex_moe import HexTier, hex_moe, route_topk  # noqa: E402
from blackhole_b200.quant import quantize_stack  # noqa: E402

EXPERTS, KEPT, H, I, TOPK = 16, 12, 256, 128, 4


def quantized(w13: torch.Tensor, w2: torch.Tensor, hessians=(None, None)) -> HexTier:
    """The stacks as one 3-bit HEX tier; hessians: those of the inputs of w13 and of w2."""
    gate, up = w13.chunk(2, dim=1)
    parts = [quantize_stack(w.float(), levels=8, block=32, H=h)
             for w, h in ((gate, hessians[0]), (up, hessians[0]), (w2, hessians[1]))]
    return HexTier(3, torch.arange(len(w2), device=w2.device), *parts).prepare(len(w2))


def expert_hessians(batches, w13: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Every expert's sum of x x^T over its rows, for the inputs of w13 [E, H, H] and of w2 [E, I, I]."""
    E = len(w13)
    hx = torch.zeros(E, H, H, device=w13.device)
    ha = torch.zeros(E, I, I, device=w13.device)
    for x, _, ids in batches:
        offsets, slot, _, _ = experts.expert_plan(ids, E)
        rows = x[(slot // TOPK).clamp(max=len(x) - 1).long()]     # rows in expert order
        act = experts.swiglu(experts.grouped_mm(rows, w13, offsets))
        experts.grouped_wgrad(rows, rows, offsets, out=hx, accumulate=True)
        experts.grouped_wgrad(act, act, offsets, out=ha, accumulate=True)
    return hx, ha


def main(steps: int = 200, seed: int = 0) -> dict:
    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev).manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, generator=g, device=dev)  # noqa: E731
    w13 = (randn(EXPERTS, 2 * I, H) * H ** -0.5).bfloat16()
    w2 = (randn(EXPERTS, H, I) * I ** -0.5).bfloat16()
    # inputs of a layer are correlated: a few directions carry most of their energy
    mix = randn(H, H) * torch.logspace(0, -1.5, H, device=dev)[:, None] * 0.3
    router = randn(H, EXPERTS)

    def tokens(n: int) -> tuple:
        """Rows, their routing in the whole layer, and in the pruned one."""
        x = (randn(n, H) @ mix).bfloat16()
        logits = x.float() @ router
        return x, route_topk(logits, TOPK), lambda stay: (x, *route_topk(logits[:, stay], TOPK))

    x, (weights, ids), routed = tokens(2048)
    used = torch.bincount(ids.reshape(-1).long(), minlength=EXPERTS)
    stay = used.argsort(descending=True)[:KEPT].sort().values      # the experts that see the fewest rows go
    held = routed(stay)
    with torch.no_grad():
        want = experts.expert_mlp(x, weights, ids, w13, w2).float()
    calibration = [tokens(1024)[2](stay) for _ in range(8)]

    def error(out: torch.Tensor) -> float:
        return float((out.float() - want).norm() / want.norm())

    def stored(a: torch.Tensor, b: torch.Tensor) -> float:
        return error(hex_moe(*held, [quantized(a, b, expert_hessians(calibration, a))]))

    # the stacks are trained in 32 bits; the layer runs on their bf16 copies
    kept = w13[stay], w2[stay]
    masters = [t.float().requires_grad_() for t in kept]
    optimizer = torch.optim.Adam(masters, lr=2e-4)
    for _ in range(steps):
        x, (weights, ids), routed = tokens(1024)
        with torch.no_grad():
            target = experts.expert_mlp(x, weights, ids, w13, w2).float()
        optimizer.zero_grad()
        out = experts.expert_mlp(*routed(stay), *(m.bfloat16() for m in masters))
        loss = (out.float() - target).square().mean()
        loss.backward()
        experts.clip_grad_norm([m.grad for m in masters], 1.0)
        optimizer.step()
    with torch.no_grad():
        healed = [m.bfloat16() for m in masters]
        return {"pruned": error(experts.expert_mlp(*held, *kept)),
                "pruned and quantized to the nearest level": error(hex_moe(*held, [quantized(*kept)])),
                "pruned and quantized": stored(*kept),
                "pruned and healed": error(experts.expert_mlp(*held, *healed)),
                "pruned, healed and quantized": stored(*healed)}


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=200)
    for name, value in main(parser.parse_args().steps).items():
        print(f"{name}: relative error {value:.4f}")
