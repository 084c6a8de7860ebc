"""A residual block of 8-bit linear layers: trained for some steps, then run as a server runs it,
a prompt first and single tokens after it, with the same weights in 8 bits.

    python examples/int8_block.py [--width 1024] [--hidden 4096] [--tokens 2048] [--steps 20]

The block is x -> x + down(silu(up(norm(x)))): the norm's output, the activations kept for the backward
pass and the weights are 8-bit rows with scales.  Data are synthetic: the block learns a fixed map.
"""
from __future__ import annotations

import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tropical-gemm_amd"))

from tropical_gemm import int8  # noqa: E402
from tropical_gemm.pytorch import int8_linear_gpu, rms_norm_int8_linear_gpu  # noqa: E402


def train_forward(x, p):
    """The block with gradients: the stream x, then the block's output added to it."""
    up, stream = rms_norm_int8_linear_gpu(x, None, p["norm"], p["up"])
    return stream + int8_linear_gpu(torch.nn.functional.silu(up), p["down"])


class Server:
    """The block for inference: weights rounded to 8-bit rows once."""

    def __init__(self, p):
        self.norm = p["norm"].detach()
        self.up, self.up_scale = int8.quantize(p["up"].detach())
        self.down, self.down_scale = int8.quantize(p["down"].detach())

    def __call__(self, x):
        q, scale, _ = int8.rms_norm(x, self.norm)
        up = int8.matmul(q, scale, self.up, self.up_scale, dtype=x.dtype)
        q, scale = int8.quantize(torch.nn.functional.silu(up))
        return x + int8.matmul(q, scale, self.down, self.down_scale, dtype=x.dtype)


def run(width=1024, hidden=4096, tokens=2048, steps=20, dtype=torch.bfloat16, verbose=True):
    """Trains the block, serves it; the losses, and how far a token served alone is from the prompt's."""
    dev = torch.device("cuda", 0)
    gen = torch.Generator(device=dev)
    gen.manual_seed(7)

    def randn(*shape, size=1.0):
        return torch.randn(*shape, generator=gen, device=dev) * size

    # Weights are kept in f32 and rounded to the activations' type for each step.
    master = {"norm": torch.ones(width, device=dev), "up": randn(hidden, width, size=width ** -0.5),
              "down": randn(width, hidden, size=hidden ** -0.5)}
    for v in master.values():
        v.requires_grad_(True)
    teacher = randn(width, width, size=width ** -0.5)
    optimizer = torch.optim.Adam(master.values(), lr=3e-4)
    losses = []
    for step in range(steps):
        x = randn(tokens, width).to(dtype)
        target = torch.tanh(x.float() @ teacher.t())
        begun = time.perf_counter()
        y = train_forward(x, {k: v.to(dtype) for k, v in master.items()})
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
    a = ap.parse_args()
    run(a.width, a.hidden, a.tokens, a.steps)
