"""Fine-tunes the decoder's kind of residual attention block on synthetic voxel features.

    python examples/finetune_block.py [--steps 50] [--channels 256] [--heads 4] [--state-bits 8]

Each step packs objects of different sizes, as a batch of sparse tensors is: group norm + swish per
object, a fused qkv projection, attention within each object, the output projection, the residual;
a mean squared error against a fixed target block, its gradients, and one AdamW step.  The norm, the
attention and the optimiser are hi3d_b200's; projections are torch's.
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch
from torch import nn

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "hi3dv1.0-mlx_b200"))
from hi3d_b200 import optim, training  # noqa: E402


class Block(nn.Module):
    """``x + proj(attention(qkv(swish(group_norm(x)))))`` over packed objects."""

    def __init__(self, channels: int, heads: int, groups: int = 32):
        super().__init__()
        self.heads, self.groups = heads, groups
        self.norm_weight = nn.Parameter(torch.ones(channels))
        self.norm_bias = nn.Parameter(torch.zeros(channels))
        self.qkv = nn.Linear(channels, 3 * channels)
        self.proj = nn.Linear(channels, channels)

    def forward(self, x: torch.Tensor, offsets: torch.Tensor, longest: int) -> torch.Tensor:
        h = training.group_norm_act(x, self.norm_weight, self.norm_bias, self.groups, offsets=offsets)
        qkv = self.qkv(h).view(x.shape[0], 3, self.heads, -1)
        a = training.flash_attn_varlen_qkvpacked(qkv, offsets, longest, qkv.shape[-1] ** -0.5)
        return x + self.proj(a.flatten(1))


def batch(sizes: list[int], channels: int, dtype: torch.dtype, generator: torch.Generator):
    """Packed features of objects of these sizes, their row offsets and the longest."""
    x = torch.randn(sum(sizes), channels, device="cuda", generator=generator).to(dtype)
    offsets = torch.tensor([0, *torch.tensor(sizes).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    return x, offsets, max(sizes)


def train(steps: int = 50, channels: int = 256, heads: int = 4, state_bits: int = 8, lr: float = 2e-3,
          dtype: torch.dtype = torch.bfloat16, seed: int = 0) -> list[float]:
    """The loss of each step."""
    torch.manual_seed(seed)
    generator = torch.Generator("cuda").manual_seed(seed)
    target, block = (Block(channels, heads).to("cuda", dtype) for _ in range(2))
    opt = optim.AdamW(block.parameters(), lr=lr, weight_decay=0.01, state_bits=state_bits)
    losses = []
    for step in range(steps):
        sizes = [64 + 97 * ((step + i) % 5) for i in range(4)]
        x, offsets, longest = batch(sizes, channels, dtype, generator)
        with torch.no_grad():
            want = target(x, offsets, longest)
        loss = (block(x, offsets, longest).float() - want.float()).square().mean()
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.detach())
    return [float(v) for v in losses]


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=50)
    ap.add_argument("--channels", type=int, default=256)
    ap.add_argument("--heads", type=int, default=4)
    ap.add_argument("--state-bits", type=int, default=8, choices=(8, 32))
    args = ap.parse_args()
    losses = train(args.steps, args.channels, args.heads, args.state_bits)
    for i in range(0, len(losses), max(1, len(losses) // 10)):
        print(f"step {i:4d}  loss {losses[i]:.5f}")
    print(f"last       loss {losses[-1]:.5f}")


if __name__ == "__main__":
    main()
