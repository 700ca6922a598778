"""One attention block of a vision-language decoder, trained for a step and
then decoding from a cache, on the package's kernels.

    python examples/attention_block.py [--tokens 2048] [--dtype bf16]

hidden -> RMSNorm -> q, k, v projections -> q/k norm + rotary positions of
three axes (time, height, width) -> attention -> output projection + residual.
The step's loss and gradients are compared with the same block in plain torch
operations, and the last token's output with a decode step that reads the
others' keys and values from a cache. Exits with an error if they differ.
"""
from __future__ import annotations

import argparse
import math
import os
import sys

import torch
import torch.nn as nn
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import bloth_b200 as bloth  # noqa: E402


class Block(nn.Module):

    def __init__(self, hidden=512, heads=8, kv_heads=2, head_dim=64, sections=(12, 10, 10)):
        super().__init__()
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.norm = bloth.BlothRMSNorm(hidden)
        self.q = nn.Linear(hidden, heads * head_dim, bias=False)
        self.k = nn.Linear(hidden, kv_heads * head_dim, bias=False)
        self.v = nn.Linear(hidden, kv_heads * head_dim, bias=False)
        self.o = nn.Linear(heads * head_dim, hidden, bias=False)
        self.wq, self.wk = (nn.Parameter(torch.ones(head_dim)) for _ in range(2))
        self.axes = bloth.mrope_axes(sections, interleaved=True)
        half = head_dim // 2
        self.register_buffer("inv_freq", 1.0 / (1e6 ** (torch.arange(half) / half)))

    def project(self, x):
        y = self.norm(x)
        B, S, _ = x.shape
        return (p(y).view(B, S, -1, self.head_dim) for p in (self.q, self.k, self.v))

    def forward(self, x, positions, cache=None):
        """x [B, S, hidden], positions [3, B, S]; cache: (k, v, rows in use) to
        append to and attend over."""
        q, k, v = self.project(x)
        q, k = bloth.fused_qk_norm_mrope(q, k, self.wq, self.wk, positions,
                                         self.inv_freq.float(), self.axes)
        lens = None
        if cache is not None:
            ck, cv, used = cache
            ck[:, used:used + k.shape[1]], cv[:, used:used + k.shape[1]] = k, v
            lens = torch.full((x.shape[0],), used + k.shape[1], device=x.device,
                              dtype=torch.int32)
            k, v = ck, cv
        o = bloth.fused_attention(q, k, v, k_lens=lens)
        return x + self.o(o.flatten(2))

    def plain(self, x, positions):
        """The same block in plain torch operations."""
        y = F.rms_norm(x.float(), (x.shape[-1],), self.norm.weight.float(), self.norm.eps)
        y = y.to(x.dtype)
        B, S, _ = x.shape
        q, k, v = (p(y).view(B, S, -1, self.head_dim).float() for p in (self.q, self.k, self.v))
        ang = positions[list(self.axes)].permute(1, 2, 0).float() * self.inv_freq.float()
        cos, sin = ang.cos().unsqueeze(2), ang.sin().unsqueeze(2)

        def turn(t, w):
            t = F.rms_norm(t, (self.head_dim,), w.float(), 1e-6)
            a, b = t.chunk(2, -1)
            return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)

        q, k = turn(q, self.wq), turn(k, self.wk)
        g = self.heads // self.kv_heads
        k, v = (t.repeat_interleave(g, 2) for t in (k, v))
        s = torch.einsum("bqhd,bkhd->bhqk", q, k) / math.sqrt(self.head_dim)
        s = s.masked_fill(torch.ones(S, S, device=x.device, dtype=torch.bool).triu(1), -math.inf)
        o = torch.einsum("bhqk,bkhd->bqhd", s.softmax(-1), v)
        return x + self.o(o.to(x.dtype).flatten(2))


def relative(a, b):
    return float(((a.float() - b.float()).norm() / b.float().norm()).detach())


def run(tokens=512, dtype=torch.bfloat16, device="cuda"):
    """Relative differences from the plain block, by name."""
    torch.manual_seed(0)
    block = Block().to(device=device, dtype=dtype)
    x = torch.randn(2, tokens, 512, device=device).to(dtype).requires_grad_(True)
    grad = torch.randn(2, tokens, 512, device=device).to(dtype)
    t = torch.arange(tokens, device=device)
    pos = torch.stack([t // 64, t // 8 % 8, t % 8]).unsqueeze(1).expand(3, 2, tokens)
    names = [n for n, p in block.named_parameters()]
    leaves = [x] + [p for _, p in block.named_parameters()]
    y = block(x, pos)
    got = torch.autograd.grad(y, leaves, grad)
    z = block.plain(x, pos)
    want = torch.autograd.grad(z, leaves, grad)
    off = {"output": relative(y, z)}
    for n, a, b in zip(["input"] + names, got, want):
        off["gradient of " + n] = relative(a, b)
    with torch.no_grad():
        ck, cv = (torch.empty(2, tokens + 16, block.kv_heads, block.head_dim, device=device,
                              dtype=dtype) for _ in range(2))
        block(x[:, :-1], pos[:, :, :-1], (ck, cv, 0))
        last = block(x[:, -1:], pos[:, :, -1:], (ck, cv, tokens - 1))
    off["decoded token"] = relative(last, y[:, -1:])
    return off


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--tokens", type=int, default=512)
    ap.add_argument("--dtype", choices=("bf16", "f16", "f32"), default="bf16")
    a = ap.parse_args()
    dtype = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[a.dtype]
    off = run(a.tokens, dtype)
    # roundings to the type along the block, a dozen of them in a row at most
    bound = {"bf16": 12 * 2.0 ** -8, "f16": 12 * 2.0 ** -11, "f32": 1e-4}[a.dtype]
    for n, v in off.items():
        print(f"{n:24s} {v:.2e}")
    if max(off.values()) > bound:
        sys.exit(f"differs from the plain block by more than {bound:.1e}")


if __name__ == "__main__":
    main()
