"""Trains a small residual MLP in bfloat16 with the matrix operators: its layers are ``linear_act``
products, its weight matrices are orthogonalised at the start and stepped by ``Muon``, its biases by
``TurboAdam``.

    python examples/train_residual_mlp.py [--steps 200] [--width 256] [--depth 3]

The data is a fixed random teacher of the same shape; the printed loss is the mean squared error on
fresh batches.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

from turboadam_b200 import Muon, TurboAdam, linear_act, orthogonalize  # noqa: E402


class ResidualMLP(torch.nn.Module):
    """``depth`` blocks h + W2 gelu(W1 h + b1) + b2 between two plain layers."""

    def __init__(self, inputs, width, depth, outputs, generator, device):
        super().__init__()

        def matrix(rows, cols):
            w = torch.randn(rows, cols, device=device, generator=generator)
            # singular values near one, whatever the draw
            return torch.nn.Parameter(orthogonalize(w))

        def vector(n):
            return torch.nn.Parameter(torch.zeros(n, device=device, dtype=torch.bfloat16))

        self.first = matrix(width, inputs)
        self.up = torch.nn.ParameterList([matrix(2 * width, width) for _ in range(depth)])
        self.up_bias = torch.nn.ParameterList([vector(2 * width) for _ in range(depth)])
        self.down = torch.nn.ParameterList([matrix(width, 2 * width) for _ in range(depth)])
        self.down_bias = torch.nn.ParameterList([vector(width) for _ in range(depth)])
        self.last = matrix(outputs, width)

    def forward(self, x):
        h = linear_act(x, self.first)
        for up, up_bias, down, down_bias in zip(self.up, self.up_bias, self.down, self.down_bias):
            wide = linear_act(h, up, up_bias, activation="gelu")
            h = linear_act(wide, down, down_bias, residual=h)
        return linear_act(h, self.last)


def train(steps=200, width=256, depth=3, batch=512, inputs=64, outputs=32, seed=0, report=None):
    """Returns the loss of every step."""
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)
    teacher = ResidualMLP(inputs, width, 1, outputs, gen, device)
    model = ResidualMLP(inputs, width, depth, outputs, gen, device)
    matrices = [p for p in model.parameters() if p.dim() == 2]
    vectors = [p for p in model.parameters() if p.dim() == 1]
    optimizers = [Muon(matrices, lr=0.02, weight_decay=0.0, adjust_lr_fn="original"),
                  TurboAdam(vectors, lr=1e-3, seed=seed)]
    losses = []
    for step in range(steps):
        for opt in optimizers:  # the rate falls linearly over the last half
            for group in opt.param_groups:
                group.setdefault("start_lr", group["lr"])
                group["lr"] = group["start_lr"] * min(1.0, 2.0 * (1.0 - step / steps))
        x = torch.randn(batch, inputs, device=device, generator=gen).bfloat16()
        with torch.no_grad():
            target = teacher(x)
        loss = (model(x).float() - target.float()).square().mean()
        for opt in optimizers:
            opt.zero_grad()
        loss.backward()
        for opt in optimizers:
            opt.step()
        losses.append(loss.detach())
        if report and (step % report == 0 or step == steps - 1):
            print(f"step {step:4d}  loss {loss.item():.4f}", flush=True)
    return torch.stack(losses).tolist()


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--width", type=int, default=256)
    ap.add_argument("--depth", type=int, default=3)
    ap.add_argument("--batch", type=int, default=512)
    a = ap.parse_args()
    train(a.steps, a.width, a.depth, a.batch, report=20)
