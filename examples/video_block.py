"""A murmurative block on video tokens: training steps with positions of three axes, then decoding.

    python examples/video_block.py [--steps 20]

A clip of frames x height x width patches becomes a sequence of tokens whose queries are normed per
head and rotated by time, height and width (``qk_norm_rope`` with sections); the block learns to
reconstruct the clip from a noisy copy. Afterwards a causal block takes tokens one by one over a
resident slot pool. Synthetic data, random weights.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from murmurative_attention_b200 import MurmurativeBlock  # noqa: E402


def video_positions(frames: int, height: int, width: int, device) -> torch.Tensor:
    """[frames * height * width, 3]: time, height and width of every token."""
    axes = [torch.arange(n, device=device) for n in (frames, height, width)]
    return torch.stack(torch.meshgrid(*axes, indexing="ij"), -1).reshape(-1, 3)


def train(steps: int = 20, frames: int = 4, height: int = 16, width: int = 16, dim: int = 256, heads: int = 4,
          batch: int = 2, dtype=torch.bfloat16, seed: int = 0):
    """Loss per step of a block that denoises a clip."""
    torch.manual_seed(seed)
    dev = torch.device("cuda")
    pairs = dim // heads // 2
    third = pairs // 3
    block = MurmurativeBlock(dim, heads, slots=64, sections=(pairs - 2 * third, third, third), device=dev, dtype=dtype)
    positions = video_positions(frames, height, width, dev)
    t = positions.float()
    waves = torch.stack([torch.sin(t @ torch.randn(3, dim, device=dev) * 0.3 + b) for b in range(batch)])
    noisy = (waves + 0.3 * torch.randn_like(waves)).to(dtype)
    opt = torch.optim.AdamW(block.parameters(), lr=3e-3, weight_decay=0.0)
    losses = []
    for _ in range(steps):
        opt.zero_grad(set_to_none=True)
        loss = (block(noisy, positions).float() - waves).square().mean()
        loss.backward()
        opt.step()
        losses.append(float(loss.detach()))
    return losses


def decode(tokens: int = 16, dim: int = 256, heads: int = 4, batch: int = 2, dtype=torch.bfloat16, seed: int = 0):
    """Outputs [tokens, batch, dim] of a causal block stepping over its slot pool."""
    torch.manual_seed(seed)
    block = MurmurativeBlock(dim, heads, slots=64, causal=True, device="cuda", dtype=dtype)
    pool = block.new_pool(batch)
    return torch.stack([block.step(torch.randn(batch, dim, device="cuda", dtype=dtype), pool) for _ in range(tokens)])


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=20)
    losses = train(ap.parse_args().steps)
    print("denoising loss: " + " ".join(f"{v:.3f}" for v in losses))
    print("decoded:", tuple(decode().shape))


if __name__ == "__main__":
    main()
