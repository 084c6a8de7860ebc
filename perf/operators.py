"""The measured operators of the 8-bit linear layer: norm, checkpoint, product and gradients.

``listed()`` names fixed cases, ``draw(rng)`` gives one more of the same ranges.  With ``own`` false,
``run`` computes an operator in its plain form (elementary torch operations in 32 bits, rounded once);
with ``own`` true it calls ``tropical_gemm.int8``.  Sizes are generic.  Inputs live on the GPU and are
made from the seed alone.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

_DEV = "cuda"
_TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}
_EPS = 1e-6
_TINY = 1e-30  # the least row maximum a scale is made from
_int8 = None


def _framework():
    """tropical_gemm.int8, imported on the first call that needs it."""
    global _int8
    if _int8 is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "tropical-gemm_amd"))
        from tropical_gemm import int8

        _int8 = int8
    return _int8


# ---- cases ---------------------------------------------------------------------------------------


def _norm(name, dtype, rows, cols, residual=True):
    return dict(name=name, op="norm", dtype=dtype, rows=rows, cols=cols, residual=residual)


def _norm_backward(name, dtype, rows, cols, residual=True):
    return dict(name=name, op="norm_backward", dtype=dtype, rows=rows, cols=cols, residual=residual)


def _checkpoint(name, dtype, rows, cols):
    return dict(name=name, op="checkpoint", dtype=dtype, rows=rows, cols=cols)


def _matmul(name, dtype, m, n, k, bias=False):
    return dict(name=name, op="matmul", dtype=dtype, m=m, n=n, k=k, bias=bias)


def _backward(name, dtype, m, n, k):
    return dict(name=name, op="backward", dtype=dtype, m=m, n=n, k=k)


def listed():
    return [
        # One token of one sequence being decoded: the latency of a norm before a projection.
        _norm("norm_1x4096", "bf16", 1, 4096),
        # A long prompt's (or a training step's) tokens through the norm of a wide layer.
        _norm("norm_8192x8192", "bf16", 8192, 8192),
        # The norm in a training step, the residual stream's own gradient added.
        _norm_backward("norm_backward_8192x4096", "bf16", 8192, 4096),
        # A small model in full precision; no size a multiple of anything, no residual.
        _norm_backward("norm_backward_777x2501", "f32", 777, 2501, residual=False),
        # A layer's activations packed for the backward pass and restored there.
        _checkpoint("checkpoint_8192x8192", "bf16", 8192, 8192),
        # The same for a short batch whose rows are no whole vectors.
        _checkpoint("checkpoint_1001x3331", "f16", 1001, 3331),
        # One token against a large weight matrix: bound by reading the weights.
        _matmul("matmul_1x8192x8192", "bf16", 1, 8192, 8192),
        # A few sequences decoded together, with a bias, and rows that start at any address.
        _matmul("matmul_13x5003x4099", "f16", 13, 5003, 4099, bias=True),
        # A short prompt: fewer tiles than the GPU has room for.
        _matmul("matmul_512x4096x4096", "bf16", 512, 4096, 4096),
        # A long prompt or a training step's forward product.
        _matmul("matmul_8192x8192x8192", "bf16", 8192, 8192, 8192),
        # Both gradients of a small layer in full precision, odd sizes.
        _backward("backward_301x1031x2049", "f32", 301, 1031, 2049),
        # Both gradients in a training step of an ordinary layer.
        _backward("backward_8192x4096x4096", "bf16", 8192, 4096, 4096),
    ]


def _size(rng, lo, hi):
    """A size spread over its logarithm: a power of two, an odd multiple of 16, or any odd number."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    kind = rng.choice(["power", "sixteens", "odd", "odd"])
    if kind == "power":
        v = 2 ** round(math.log2(v))
    elif kind == "sixteens" and v >= 32:
        v = 16 * (int(v / 16) | 1)
    else:
        v = int(v) | 1
    return max(lo, min(hi, v))


def draw(rng):
    while True:
        c = _draw(rng)
        if work(c)["flops"] <= 2.0 * 8192 ** 3:
            c.pop("name")
            return c


def _draw(rng):
    op = rng.choice(["norm", "norm_backward", "checkpoint", "decode", "decode", "matmul", "matmul",
                     "backward", "backward"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op in ("norm", "norm_backward"):
        make = _norm if op == "norm" else _norm_backward
        return make("", dtype, _size(rng, 1, 8192), _size(rng, 64, 8192), rng.random() < 0.7)
    if op == "checkpoint":
        return _checkpoint("", dtype, _size(rng, 1, 8192), _size(rng, 64, 8192))
    m = _size(rng, 1, 32) if op == "decode" else _size(rng, 32, 8192)
    n, k = _size(rng, 64, 8192), _size(rng, 64, 8192)
    if op == "backward":
        return _backward("", dtype, m, n, k)
    return _matmul("", dtype, m, n, k, rng.random() < 0.3)


# ---- inputs --------------------------------------------------------------------------------------


def _activations(g, rows, cols, dtype):
    """A residual stream's values: most channels of order one, one in a hundred much larger, and one
    row in sixty-four zero, as a padded position is."""
    x = torch.randn(rows, cols, generator=g, device=_DEV)
    x *= torch.where(torch.rand(cols, generator=g, device=_DEV) < 0.01, 20.0, 1.0)
    if rows >= 8:
        x *= (torch.rand(rows, 1, generator=g, device=_DEV) >= 1 / 64).float()
    return x.to(dtype)


def _gradients(g, rows, cols, dtype):
    """Gradients: small, their size differing from token to token."""
    x = torch.randn(rows, cols, generator=g, device=_DEV) * 2e-2
    return (x * torch.exp(torch.randn(rows, 1, generator=g, device=_DEV))).to(dtype)


def _quantized(g, rows, cols):
    """8-bit rows and their scales, as rounding normal values to 127 steps of the row's maximum gives
    them."""
    q = torch.round(torch.randn(rows, cols, generator=g, device=_DEV) * 32).clamp_(-127, 127).to(torch.int8)
    scale = (torch.rand(rows, generator=g, device=_DEV) + 0.5) * 0.01
    return q, scale


def prepare(case, seed):
    g = torch.Generator(device=_DEV)
    g.manual_seed(seed)
    s = dict(case, dtype=_TORCH[case["dtype"]])
    if case["op"] in ("norm", "norm_backward"):
        rows, cols, dtype = case["rows"], case["cols"], s["dtype"]
        s["x"] = _activations(g, rows, cols, dtype)
        s["weight"] = (1 + 0.1 * torch.randn(cols, generator=g, device=_DEV)).to(dtype)
        other = _activations if case["op"] == "norm" else _gradients
        s["residual"] = other(g, rows, cols, dtype) if case["residual"] else None
        if case["op"] == "norm_backward":
            s["grad"] = _gradients(g, rows, cols, dtype)
    elif case["op"] == "checkpoint":
        s["x"] = _activations(g, case["rows"], case["cols"], s["dtype"])
    else:
        m, n, k = case["m"], case["n"], case["k"]
        s["a"], s["a_scale"] = _quantized(g, m, k)
        s["b"], s["b_scale"] = _quantized(g, n, k)
        if case["op"] == "backward":
            s["grad"] = _gradients(g, m, n, s["dtype"])
        else:
            bias = torch.randn(n, generator=g, device=_DEV) if case["bias"] else None
            s["bias"] = bias.to(s["dtype"]) if case["bias"] else None
    return s


# ---- one pass ------------------------------------------------------------------------------------


def run(state):
    return (_OWN if own else _PLAIN)[state["op"]](state)


def _own_norm(s):
    f = _framework()
    q, scale, h = f.rms_norm(s["x"], s["weight"], s["residual"], _EPS)
    out = {"values": f.dequantize(q, scale, s["dtype"]), "scale": scale}
    return dict(out, h=h) if s["residual"] is not None else out


def _own_norm_backward(s):
    # "residual" is here the gradient that reaches the stream behind the norm.
    return _framework().rms_norm_backward(s["grad"], s["x"], s["weight"], _EPS, s["residual"])


def _own_checkpoint(s):
    f = _framework()
    q, scale = f.quantize(s["x"])
    return {"values": f.dequantize(q, scale, s["dtype"]), "scale": scale}


def _own_matmul(s):
    return _framework().matmul(s["a"], s["a_scale"], s["b"], s["b_scale"], s["bias"], s["dtype"])


def _own_backward(s):
    f = _framework()
    return f.backward_a(s["grad"], s["b"], s["b_scale"]), f.backward_b(s["grad"], s["a"], s["a_scale"])


_OWN = {"norm": _own_norm, "norm_backward": _own_norm_backward, "checkpoint": _own_checkpoint,
        "matmul": _own_matmul, "backward": _own_backward}


def _round_rows(v):
    """The 8-bit rows nearest to v, as whole floating numbers, and the largest magnitude of each."""
    top = v.abs().amax(1, keepdim=True).clamp_min(_TINY)
    return torch.round(v * (127.0 / top)).clamp_(-127, 127), top


def _plain_norm(s):
    h = s["x"]
    if s["residual"] is not None:
        h = (h.float() + s["residual"].float()).to(s["dtype"])
    f = h.float()
    rstd = 1.0 / torch.sqrt((f * f).mean(1, keepdim=True) + _EPS)
    q, top = _round_rows(f * s["weight"].float())
    scale = top * rstd / 127.0
    out = {"values": (q * scale).to(s["dtype"]), "scale": scale[:, 0]}
    return dict(out, h=h) if s["residual"] is not None else out


def _plain_norm_backward(s):
    h, grad = s["x"].float(), s["grad"].float()
    rstd = 1.0 / torch.sqrt((h * h).mean(1, keepdim=True) + _EPS)
    xhat, u = h * rstd, grad * s["weight"].float()
    grad_x = rstd * (u - xhat * (u * xhat).mean(1, keepdim=True))
    if s["residual"] is not None:
        grad_x = grad_x + s["residual"].float()
    return grad_x.to(s["dtype"]), (grad * xhat).sum(0).to(s["dtype"])


def _plain_checkpoint(s):
    q, top = _round_rows(s["x"].float())
    scale = top / 127.0
    return {"values": (q * scale).to(s["dtype"]), "scale": scale[:, 0]}


def _plain_matmul(s):
    c = s["a"].float() @ s["b"].float().t()
    c = c * s["a_scale"][:, None] * s["b_scale"]
    if s["bias"] is not None:
        c = c + s["bias"].float()
    return c.to(s["dtype"])


def _plain_backward(s):
    grad = s["grad"].float()
    grad_a = grad @ (s["b"].float() * s["b_scale"][:, None])
    grad_b = grad.t() @ (s["a"].float() * s["a_scale"][:, None])
    return grad_a.to(s["dtype"]), grad_b.to(s["dtype"])


_PLAIN = {"norm": _plain_norm, "norm_backward": _plain_norm_backward, "checkpoint": _plain_checkpoint,
          "matmul": _plain_matmul, "backward": _plain_backward}


# ---- the definition in 64 bits -------------------------------------------------------------------


def _exact_rows(v, factor):
    top = torch.maximum(v.abs().max(1).values, torch.tensor(_TINY, dtype=torch.float64, device=_DEV))
    q = torch.round(v / top[:, None] * 127).clamp(-127, 127)
    scale = top * factor / 127
    return {"values": q * scale[:, None], "scale": scale}


def exact(case, seed):
    s = prepare(case, seed)
    wide = {key: v.double() for key, v in s.items() if isinstance(v, torch.Tensor)}
    op = case["op"]
    if op == "norm":
        h = wide["x"]
        if case["residual"]:  # the stream is stored in its own type, and the norm is of what is stored
            h = (h + wide["residual"]).to(s["dtype"]).double()
        factor = (h.pow(2).sum(1) / case["cols"] + _EPS).pow(-0.5)
        out = _exact_rows(h * wide["weight"], factor)
        return dict(out, h=h) if case["residual"] else out
    if op == "norm_backward":
        x, g, w = wide["x"], wide["grad"], wide["weight"]
        r = (x.pow(2).sum(1) / case["cols"] + _EPS).pow(-0.5)[:, None]
        dot = (g * w * x).sum(1, keepdim=True)
        grad_x = g * w * r - x * dot * r.pow(3) / case["cols"]
        if case["residual"]:
            grad_x = grad_x + wide["residual"]
        return grad_x, (g * x * r).sum(0)
    if op == "checkpoint":
        return _exact_rows(wide["x"], 1.0)
    a, b = wide["a"] * wide["a_scale"][:, None], wide["b"] * wide["b_scale"][:, None]
    if op == "backward":
        return torch.mm(wide["grad"], b), torch.mm(wide["grad"].t(), a)
    c = torch.mm(a, b.t())
    return c + wide["bias"] if case["bias"] else c


# ---- what a pass cannot do without ---------------------------------------------------------------


def work(case):
    """Each input read and each output written once; a product's multiply-adds count two."""
    size = _SIZE[case["dtype"]]
    if case["op"] in ("matmul", "backward"):
        m, n, k = case["m"], case["n"], case["k"]
        if case["op"] == "backward":
            return {"bytes": size * (m * n + m * k + n * k) + (m + n) * (k + 4), "flops": 4.0 * m * n * k}
        return {"bytes": (m + n) * (k + 4) + size * (m * n + case["bias"] * n), "flops": 2.0 * m * n * k}
    cells, edge = case["rows"] * case["cols"], 4 * case["rows"]
    if case["op"] == "checkpoint":  # read, packed, restored
        return {"bytes": cells * (2 * size + 1) + edge, "flops": 5.0 * cells}
    if case["op"] == "norm":  # x, residual and h; the 8-bit rows and their values
        streams = 4 if case["residual"] else 2
        return {"bytes": cells * (streams * size + 1) + edge + size * case["cols"], "flops": 9.0 * cells}
    streams = 4 if case["residual"] else 3
    return {"bytes": size * (streams * cells + 2 * case["cols"]), "flops": 12.0 * cells}
