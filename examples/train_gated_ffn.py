"""Train a small stack of gated feed-forward blocks: came_amd's block with its gradients, the clip by the global norm and
an optimizer step, as one loop.

    python examples/train_gated_ffn.py --optimizer adamw8bit --steps 200

The data are a random stack of the same shape's outputs for normal inputs; the loss is their mean squared error.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import came_amd  # noqa: E402

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
LRS = {"adamw": 1e-3, "adamw8bit": 1e-3, "came8bit": 2e-4}  # CAME's steps are larger at the same rate


class Block(torch.nn.Module):
    """x + gated_ffn(x / rms(x))"""

    def __init__(self, dim: int, hidden: int, dtype: torch.dtype, gen: torch.Generator):
        super().__init__()

        def weight(*shape):
            return torch.nn.Parameter((torch.randn(*shape, generator=gen) * shape[1] ** -0.5).to(dtype).cuda())

        self.w_gate, self.w_up, self.w_down = weight(hidden, dim), weight(hidden, dim), weight(dim, hidden)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        n = x * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-6).to(x.dtype)
        return x + came_amd.gated_ffn(n, self.w_gate, self.w_up, self.w_down)


def optimizer(name: str, params, lr: float):
    if name == "adamw":
        return came_amd.AdamW(params, lr=lr, max_grad_norm=1.0)
    if name == "adamw8bit":
        return came_amd.AdamW8bit(params, lr=lr, max_grad_norm=1.0)
    return came_amd.CAME8bit(params, lr=lr, weight_decay=1e-2)


def train(steps: int = 200, tokens: int = 512, dim: int = 256, hidden: int = 704, layers: int = 2, name: str = "adamw8bit",
          dtype: str = "bf16", lr: float | None = None, log=print) -> list[float]:
    """The losses of every tenth step and the last."""
    gen = torch.Generator().manual_seed(0)
    make = lambda: torch.nn.Sequential(*(Block(dim, hidden, DTYPES[dtype], gen) for _ in range(layers)))  # noqa: E731
    teacher, student = make(), make()
    params = list(student.parameters())
    opt = optimizer(name, params, lr or LRS[name])
    losses = []
    for step in range(steps):
        x = torch.randn(tokens, dim, generator=gen).to(DTYPES[dtype]).cuda()
        with torch.no_grad():
            want = teacher(x)
        loss = (student(x) - want).float().square().mean()
        loss.backward()
        if not hasattr(opt, "max_grad_norm"):  # CAME clips each update by itself; the gradients' norm is clipped here
            came_amd.clip_grad_norm_(params, 1.0)
        opt.step()
        opt.zero_grad()
        if step % 10 == 0 or step == steps - 1:
            losses.append(float(loss.detach()))
            log(f"step {step:4d}  loss {losses[-1]:.5f}")
    return losses


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--optimizer", choices=sorted(LRS), default="adamw8bit")
    ap.add_argument("--dtype", choices=sorted(DTYPES), default="bf16")
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--lr", type=float)
    a = ap.parse_args()
    train(a.steps, name=a.optimizer, dtype=a.dtype, lr=a.lr)


if __name__ == "__main__":
    main()
