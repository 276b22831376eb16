"""Train a small restoration transformer against the SSIM loss.

Noisy frames are cut into patches; each block normalises and rotates its queries
and keys (``fa.qk_norm_rotary``), the loss is ``1 - SSIM`` plus a Charbonnier
term, and the weight matrices take orthogonalised updates (``fa.Muon``); norms,
biases and the position-free rest go to AdamW.

    python examples/train_restoration.py --steps 100
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch
import torch.nn.functional as F
from torch import nn

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))  # the package, from its checkout

import frame_analytics_b200 as fa  # noqa: E402


def angle_tables(rows: int, cols: int, rotary: int, device):
    """cos / sin of a (rows x cols) grid of patches: half of the pairs turn with
    the patch's row, half with its column."""
    per_axis = rotary // 4
    freq = 100.0 ** (-torch.arange(per_axis, device=device, dtype=torch.float64) / per_axis)
    y = torch.arange(rows, device=device, dtype=torch.float64)[:, None] * freq
    x = torch.arange(cols, device=device, dtype=torch.float64)[:, None] * freq
    angle = torch.cat((y[:, None].expand(rows, cols, per_axis),
                       x[None].expand(rows, cols, per_axis)), -1).reshape(rows * cols, -1)
    return angle.cos().float(), angle.sin().float()


class Block(nn.Module):
    def __init__(self, width: int, heads: int):
        super().__init__()
        self.heads, self.dim = heads, width // heads
        self.norm1, self.norm2 = nn.LayerNorm(width), nn.LayerNorm(width)
        self.qkv = nn.Linear(width, 3 * width, bias=False)
        self.proj = nn.Linear(width, width, bias=False)
        self.up = nn.Linear(width, 4 * width, bias=False)
        self.down = nn.Linear(4 * width, width, bias=False)
        self.q_weight = nn.Parameter(torch.ones(self.dim))
        self.k_weight = nn.Parameter(torch.ones(self.dim))

    def forward(self, x, cos, sin):
        b, n, w = x.shape
        packed = self.qkv(self.norm1(x)).view(b, n, 3 * self.heads, self.dim)
        q, k, v = packed.split(self.heads, dim=2)
        q, k = fa.qk_norm_rotary(q, k, cos, sin, q_weight=self.q_weight, k_weight=self.k_weight)
        y = F.scaled_dot_product_attention(q.transpose(1, 2), k.transpose(1, 2),
                                           v.transpose(1, 2))
        x = x + self.proj(y.transpose(1, 2).reshape(b, n, w))
        return x + self.down(F.gelu(self.up(self.norm2(x))))


class Restorer(nn.Module):
    def __init__(self, patch: int = 8, width: int = 192, heads: int = 6, depth: int = 2):
        super().__init__()
        self.patch, self.rotary = patch, width // heads
        self.embed = nn.Conv2d(3, width, patch, patch)
        self.blocks = nn.ModuleList(Block(width, heads) for _ in range(depth))
        self.head = nn.Linear(width, 3 * patch * patch)
        nn.init.zeros_(self.head.weight)
        nn.init.zeros_(self.head.bias)

    def forward(self, frames):
        x = self.embed(frames)
        rows, cols = x.shape[-2:]
        cos, sin = angle_tables(rows, cols, self.rotary, frames.device)
        x = x.flatten(2).mT
        for block in self.blocks:
            x = block(x, cos, sin)
        return frames + F.pixel_shuffle(self.head(x).mT.unflatten(2, (rows, cols)), self.patch)


def batch(n: int, size: int, generator, device):
    """Smooth synthetic frames in [0, 1] and their noisy versions."""
    coarse = torch.rand(n, 3, size // 8, size // 8, generator=generator, device=device)
    clean = F.interpolate(coarse, size=(size, size), mode="bicubic").clamp(0, 1)
    noise = 0.1 * torch.randn(clean.shape, generator=generator, device=device)
    return clean, (clean + noise).clamp(0, 1)


def train(steps: int = 100, size: int = 96, frames: int = 8, device="cuda", report=None):
    """Returns the loss of every step."""
    torch.manual_seed(0)
    g = torch.Generator(device=device).manual_seed(1)
    net = Restorer().to(device)
    matrices = [p for name, p in net.named_parameters() if p.dim() >= 2 and "head" not in name]
    chosen = {id(p) for p in matrices}
    others = [p for p in net.parameters() if id(p) not in chosen]
    muon = fa.Muon(matrices, lr=0.01, weight_decay=0.01)
    adam = torch.optim.AdamW(others, lr=2e-3)
    losses = []
    for i in range(steps):
        clean, noisy = batch(frames, size, g, device)
        out = net(noisy)
        loss = 1 - fa.ssim(clean, out, data_range=1.0) + fa.charbonnier(clean, out, eps=1e-3)
        muon.zero_grad(set_to_none=True)
        adam.zero_grad(set_to_none=True)
        loss.backward()
        muon.step()
        adam.step()
        losses.append(loss.detach())
        if report and (i + 1) % report == 0:
            print(f"step {i + 1}: loss {float(losses[-1]):.4f}")
    return [float(v) for v in losses]


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--steps", type=int, default=100)
    ap.add_argument("--size", type=int, default=96)
    ap.add_argument("--frames", type=int, default=8)
    args = ap.parse_args()
    train(args.steps, args.size, args.frames, report=10)
