"""Trains a small stack of fused MLP expert blocks and serves it.

Each block (FusedMLPExperts) norms its residual stream (fused_rms_norm), routes
every row to its two best experts (expert_sort, expert_dispatch), runs them
(FusedMLPSoftplus) and adds their weighted rows (expert_combine); FusedAdamW
steps all parameters in one launch, with its state in 8 bits.  At the end the
trained stream is normed into 8 bits with a scale for each 128 columns, as a
projection in 8 bits would take it.

    python examples/train_experts.py [--steps 200] [--rows 4096] [--state-bits 8]
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from mlp_megakernel_b200 import FusedAdamW, FusedMLPExperts, fused_rms_norm, fused_rms_norm_fp8  # noqa: E402


class Stack(torch.nn.Module):
    def __init__(self, width: int, hidden: int, blocks: int, experts: int):
        super().__init__()
        self.blocks = torch.nn.ModuleList(FusedMLPExperts(D=width, H=hidden, num_experts=experts, top=2)
                                          for _ in range(blocks))
        self.gain = torch.nn.Parameter(torch.ones(width))

    def forward(self, x):
        h = None
        for block in self.blocks:
            x, h = block(x, h)
        return x, h  # the stream is their sum

    def output(self, x):
        y, h = self(x)
        return fused_rms_norm(y, self.gain, residual=h)[0]


def main() -> int:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--rows", type=int, default=4096)
    ap.add_argument("--width", type=int, default=128)
    ap.add_argument("--blocks", type=int, default=2)
    ap.add_argument("--experts", type=int, default=8)
    ap.add_argument("--state-bits", type=int, choices=(8, 32), default=8)
    a = ap.parse_args()

    torch.manual_seed(0)
    model = Stack(a.width, a.width, a.blocks, a.experts).cuda()
    teacher = torch.randn(a.width, a.width, device="cuda") / a.width ** 0.5
    opt = FusedAdamW(model.parameters(), lr=2e-3, weight_decay=1e-3, state_bits=a.state_bits)
    first = last = None
    for step in range(a.steps):
        x = torch.randn(a.rows, a.width, device="cuda")
        loss = (model.output(x) - torch.tanh(x @ teacher)).square().mean()
        opt.zero_grad()
        loss.backward()
        opt.step()
        if step % max(1, a.steps // 5) == 0 or step == a.steps - 1:
            last = loss.item()
            first = last if first is None else first
            print(f"step {step:4d}  loss {last:.4f}")

    with torch.no_grad():
        y, h = model(x)
        want = fused_rms_norm(y, model.gain, residual=h)[0]
        q, scale, _ = fused_rms_norm_fp8(y, model.gain, residual=h, group=128)
        back = q.float() * scale.repeat_interleave(128, dim=1)[:, :a.width]
        off = ((back - want).norm() / want.norm()).item()
    print(f"8-bit output: relative error {off:.4f}")
    return 0 if last < first and off < 0.04 else 1


if __name__ == "__main__":
    sys.exit(main())
