"""A residual block in 8-bit floating point: trained with dropout for some steps, then run as a server
runs it, a prompt first and single tokens after it, with the same weights in 8 bits.

    python examples/fp8_block.py [--width 1024] [--hidden 4096] [--tokens 2048] [--steps 20]

The block is h = x + dropout(down(gelu(up(norm(x))))), and its answer is head(norm(h)).  The linear layers'
operands are e4m3 numbers with a power of two for each block of 128; the masks are made again in the
backward pass.  Data are synthetic: the block learns a fixed map.
"""
from __future__ import annotations

import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tropical-gemm_amd"))

from tropical_gemm import fp8, layers  # noqa: E402
from tropical_gemm.pytorch import dropout_add_layer_norm_gpu, fp8_linear_gpu, layer_norm_gpu  # noqa: E402

gelu = torch.nn.functional.gelu


def train_forward(x, p, drop, seed):
    """The block with gradients; `seed` makes the step's mask."""
    up = fp8_linear_gpu(layer_norm_gpu(x, p["norm"], p["bias"]), p["up"])
    branch = fp8_linear_gpu(gelu(up), p["down"])
    y, _ = dropout_add_layer_norm_gpu(branch, x, p["norm2"], p["bias2"], drop, seed=seed)
    return fp8_linear_gpu(y, p["head"])


class Server:
    """The block for inference: weights rounded to 8 bits once, no dropout."""

    def __init__(self, p):
        self.p = {k: p[k].detach() for k in ("norm", "bias", "norm2", "bias2")}
        self.w = {k: fp8.quantize(p[k].detach(), fp8.BLOCK) for k in ("up", "down", "head")}

    def linear(self, x, name):
        return fp8.matmul(*fp8.quantize(x), *self.w[name], dtype=x.dtype)

    def __call__(self, x):
        y = layers.layer_norm(x, self.p["norm"], self.p["bias"])[0]
        branch = self.linear(gelu(self.linear(y, "up")), "down")
        y = layers.layer_norm(branch, self.p["norm2"], self.p["bias2"], x)[0]
        return self.linear(y, "head")


def run(width=1024, hidden=4096, tokens=2048, steps=20, drop=0.1, dtype=torch.bfloat16, verbose=True):
    """Trains the block, serves it; the losses, and how far a token served alone is from the prompt's."""
    dev = torch.device("cuda", 0)
    gen = torch.Generator(device=dev)
    gen.manual_seed(7)

    def randn(*shape, size=1.0):
        return torch.randn(*shape, generator=gen, device=dev) * size

    # Weights are kept in f32 and rounded to the activations' type for each step.
    master = {"norm": torch.ones(width, device=dev), "bias": torch.zeros(width, device=dev),
              "norm2": torch.ones(width, device=dev), "bias2": torch.zeros(width, device=dev),
              "up": randn(hidden, width, size=width ** -0.5), "down": randn(width, hidden, size=hidden ** -0.5),
              "head": randn(width, width, size=width ** -0.5)}
    for v in master.values():
        v.requires_grad_(True)
    teacher = randn(width, width, size=width ** -0.5)
    optimizer = torch.optim.Adam(master.values(), lr=3e-4)
    losses = []
    for step in range(steps):
        x = randn(tokens, width).to(dtype)
        target = torch.tanh(x.float() @ teacher.t())
        begun = time.perf_counter()
        y = train_forward(x, {k: v.to(dtype) for k, v in master.items()}, drop, seed=step)
        loss = (y.float() - target).square().mean()
        optimizer.zero_grad(set_to_none=True)
        loss.backward()
        optimizer.step()
        losses.append(loss.item())
        if verbose and (step % 5 == 0 or step == steps - 1):
            print(f"step {step:3d}  loss {losses[-1]:.4f}  {1e3 * (time.perf_counter() - begun):.2f} ms", flush=True)
    server = Server({k: v.to(dtype) for k, v in master.items()})
    x = randn(tokens, width).to(dtype)
    prompt = server(x)
    alone = torch.cat([server(x[i:i + 1]) for i in range(8)])
    apart = (alone.float() - prompt[:8].float()).abs().max().item()
    if verbose:
        print(f"prompt of {tokens} tokens served; single tokens differ from it by at most {apart:.2g}")
    return losses, apart


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--width", type=int, default=1024)
    ap.add_argument("--hidden", type=int, default=4096)
    ap.add_argument("--tokens", type=int, default=2048)
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--drop", type=float, default=0.1)
    a = ap.parse_args()
    run(a.width, a.hidden, a.tokens, a.steps, a.drop)
