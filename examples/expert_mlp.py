"""Trains a small layer of experts to follow a dense network, then serves it in 8-bit integers.

    python examples/expert_mlp.py [--steps 200]

Every step runs the expert operators together, as a program uses them: routing
with its gradient, the row order, products grouped by expert with both
gradients, the weighted sum; then the 8-bit form of the same layer.
"""

from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import einjax_b200 as E  # noqa: E402


def make_layer(d: int, f: int, experts: int, gen) -> dict:
    def weight(*shape):
        w = torch.randn(*shape, generator=gen, device="cuda") * shape[-2] ** -0.5
        return w.requires_grad_()
    return {"router": weight(d, experts), "w_in": weight(experts, d, 2 * f), "w_out": weight(experts, f, d)}


def forward(x, layer, top_k: int):
    w_in, w_out = layer["w_in"].to(torch.bfloat16), layer["w_out"].to(torch.bfloat16)
    return E.expert_mlp(x.to(torch.bfloat16), layer["router"], w_in, w_out, top_k)


def main(steps: int = 200, tokens: int = 1000, d: int = 256, f: int = 512, experts: int = 8, top_k: int = 2) -> dict:
    gen = torch.Generator(device="cuda")
    gen.manual_seed(0)
    teacher = [torch.randn(d, 2 * d, generator=gen, device="cuda") * d ** -0.5,
               torch.randn(2 * d, d, generator=gen, device="cuda") * (2 * d) ** -0.5]
    layer = make_layer(d, f, experts, gen)
    optimizer = torch.optim.Adam(layer.values(), lr=2e-3)
    losses = []
    for _ in range(steps):
        x = torch.randn(tokens, d, generator=gen, device="cuda")
        want = torch.relu(x @ teacher[0]) @ teacher[1]
        loss = (forward(x, layer, top_k).float() - want).square().mean()
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    with torch.no_grad():
        x = torch.randn(tokens, d, generator=gen, device="cuda")
        served = E.expert_mlp(x.to(torch.bfloat16), layer["router"], E.quantize_experts(layer["w_in"]),
                              E.quantize_experts(layer["w_out"]), top_k)
        trained = forward(x, layer, top_k)
        off = float((served.float() - trained.float()).norm() / trained.float().norm())
    E.check_device_errors()
    return {"first": float(losses[0]), "last": float(losses[-1]), "int8_off": off}


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__)
    parser.add_argument("--steps", type=int, default=200)
    result = main(parser.parse_args().steps)
    print(f"loss {result['first']:.4f} -> {result['last']:.4f}; "
          f"8-bit outputs differ by {100 * result['int8_off']:.2f}%")
