"""Point clouds as sequences: train a small classifier of shapes, then read a cloud point by point.

    python examples/point_sequence.py [--steps 60]

Clouds are sampled to equal coverage, brought into Morton order and run through two blocks of gated
recurrence and window attention; the causal blocks then answer the same cloud token by token from
their caches, which gives the same rows.
"""

import argparse
import os
import sys

import torch
from torch import nn

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from gdl_amd.functional import farthest_point_sampling, segment_reduce, sort_and_build_csr  # noqa: E402
from gdl_amd.sequence import PointSequenceBlock, serial_order  # noqa: E402


def clouds(batch, points, dev):
    """Spheres, cubes' surfaces and helices with jitter, unequal numbers of points: (pos, ptr, label)."""
    sizes = torch.randint(points // 2, points + 1, (batch,))
    label = torch.randint(0, 3, (batch,))
    parts = []
    for n, kind in zip(sizes.tolist(), label.tolist()):
        x = torch.randn(n, 3)
        if kind == 0:
            x = x / x.norm(dim=1, keepdim=True)
        elif kind == 1:
            x = x / x.abs().amax(1, keepdim=True)
        else:
            t = torch.rand(n) * 12
            x = torch.stack([t.cos(), t.sin(), t / 6 - 1], 1)
        parts.append(x + 0.05 * torch.randn(n, 3))
    ptr = torch.cat([torch.zeros(1, dtype=torch.int64), sizes.cumsum(0)])
    return torch.cat(parts).to(dev), ptr.to(dev), label.to(dev)


class Classifier(nn.Module):
    def __init__(self, channels=64):
        super().__init__()
        self.embed = nn.Linear(3, channels)
        self.blocks = nn.ModuleList(PointSequenceBlock(channels, 4, 32, kv_heads=2, sinks=2) for _ in range(2))
        self.head = nn.Linear(channels, 3)

    def forward(self, pos, ptr):
        x = self.embed(pos)
        for block in self.blocks:
            x = block(x, ptr)
        cloud = torch.repeat_interleave(ptr[1:] - ptr[:-1])
        csr = sort_and_build_csr(cloud, ptr.numel() - 1)
        return self.head(segment_reduce(x, *csr, ptr.numel() - 1, reduce="mean")), x


def main():
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--steps", type=int, default=60)
    steps = ap.parse_args().steps
    dev = torch.device("cuda")
    torch.manual_seed(0)
    model = Classifier().to(dev)
    opt = torch.optim.AdamW(model.parameters(), lr=2e-3)
    for step in range(steps):
        pos, ptr, label = clouds(32, 512, dev)
        keep = farthest_point_sampling(pos, 128, ptr=ptr)
        ptr = torch.arange(0, 32 * 128 + 1, 128, device=dev)
        pos = pos[keep]
        pos = pos[serial_order(pos, ptr)]
        logits, _ = model(pos, ptr)
        loss = nn.functional.cross_entropy(logits, label)
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
        if step % 20 == 0 or step == steps - 1:
            right = (logits.argmax(1) == label).float().mean()
            print(f"step {step:3d}  loss {loss.item():.3f}  right {right.item():.2f}", flush=True)
    with torch.no_grad():
        _, rows = model(pos, ptr)
        caches = [block.new_cache(32) for block in model.blocks]
        worst = 0.0
        for t in range(128):
            x = model.embed(pos[ptr[:-1] + t])
            for block, cache in zip(model.blocks, caches):
                x = block.step(x, torch.full((32,), t, device=dev), cache)
            worst = max(worst, (x - rows[ptr[:-1] + t]).abs().max().item())
    print(f"token by token: rows within {worst:.1e} of the forward's")


if __name__ == "__main__":
    main()
