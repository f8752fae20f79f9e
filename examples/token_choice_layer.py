"""A layer whose tokens choose their experts: a few training steps on synthetic data with a load-balancing bias, then the same layer
served on 8-bit weights.

    python examples/token_choice_layer.py
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from expertscattergather_b200 import RoutedExperts, ops  # noqa: E402


def main(steps=30, tokens=4096, E=32, I=256, J=128, top_k=4):
    torch.manual_seed(0)
    layer = RoutedExperts(E, I, J, top_k, balance=True, score="sigmoid", groups=4, top_groups=2).cuda().bfloat16()
    target = torch.randn(I, I, device="cuda") / I ** 0.5
    opt = torch.optim.AdamW(layer.parameters(), lr=3e-3)
    first = last = None
    for step in range(steps):
        x = torch.randn(tokens, I, device="cuda").bfloat16()
        loss = (layer(x).float() - x.float() @ target).square().mean()
        opt.zero_grad()
        loss.backward()
        opt.step()
        layer.router.adjust(layer.plan, 1e-3)
        last = loss.item()
        first = last if first is None else first
        if step % 10 == 0 or step == steps - 1:
            counts = layer.plan.counts()
            print(f"step {step:3d}  loss {last:.4f}  rows of an expert {counts.min().item()} .. {counts.max().item()}")
    served = layer.quantized()
    x = torch.randn(16, I, device="cuda").bfloat16()
    with torch.no_grad():
        full, small = layer(x).float(), served(x).float()
    off = ((full - small).norm() / full.norm()).item()
    print(f"8-bit weights: {off:.3%} from the bf16 layer")
    ops.check_status()
    return first, last, off


if __name__ == "__main__":
    main()
