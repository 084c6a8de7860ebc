"""The measured operators of a block in 8-bit floating point: layer norm, dropout and the linear layer.

``listed()`` names fixed cases, ``draw(rng)`` gives one more of the same ranges.  With ``own`` false,
``run`` computes an operator in its plain form (elementary torch operations in 32 bits, rounded once);
with ``own`` true it calls ``tropical_gemm.fp8`` and ``tropical_gemm.layers``.  Sizes are generic.
Inputs live on the GPU and are made from the seed alone.
"""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

_DEV = "cuda"
_TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}
_EPS = 1e-5
_BLOCK = 128
_E4M3, _E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
_MOST = 448.0          # the largest e4m3 number
_LEAST_EXPONENT = -100  # of a block's scale
_modules = None


def _framework():
    """tropical_gemm.fp8 and tropical_gemm.layers, imported on the first call that needs them."""
    global _modules
    if _modules is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "tropical-gemm_amd"))
        from tropical_gemm import fp8, layers

        _modules = fp8, layers
    return _modules


# ---- cases ---------------------------------------------------------------------------------------


def _quantize(name, dtype, rows, cols, block_rows):
    return dict(name=name, op="quantize", dtype=dtype, rows=rows, cols=cols, block_rows=block_rows)


def _matmul(name, dtype, m, n, k, bias=False):
    return dict(name=name, op="matmul", dtype=dtype, m=m, n=n, k=k, bias=bias)


def _backward(name, dtype, m, n, k):
    return dict(name=name, op="backward", dtype=dtype, m=m, n=n, k=k)


def _rows(op):
    def make(name, dtype, rows, cols, residual=True, p=0.0):
        return dict(name=name, op=op, dtype=dtype, rows=rows, cols=cols, residual=residual, p=p)
    return make


_norm, _norm_backward, _dropout = _rows("layer_norm"), _rows("layer_norm_backward"), _rows("dropout")


def listed():
    return [
        # A long prompt's (or a training step's) activations on their way into a product.
        _quantize("quantize_8192x8192", "bf16", 8192, 8192, 1),
        # A weight matrix after an optimizer's step; no size a multiple of a block.
        _quantize("quantize_weight_5003x4099", "f32", 5003, 4099, 128),
        # One token against a large weight matrix: bound by reading the weights.
        _matmul("matmul_1x8192x8192", "bf16", 1, 8192, 8192),
        # A short prompt through a layer of odd sizes, with a bias: rows at any address.
        _matmul("matmul_509x5003x4099", "f16", 509, 5003, 4099, bias=True),
        # A long prompt or a training step's forward product.
        _matmul("matmul_8192x8192x8192", "bf16", 8192, 8192, 8192),
        # Both gradients of a small layer in full precision, odd sizes.
        _backward("backward_301x1031x2049", "f32", 301, 1031, 2049),
        # Both gradients in a training step of an ordinary layer.
        _backward("backward_8192x4096x4096", "bf16", 8192, 4096, 4096),
        # One token of one sequence being decoded: the latency of a norm before a product.
        _norm("layer_norm_1x4096", "bf16", 1, 4096),
        # The norm in a training step of a wide layer, dropout on the branch that joins the stream.
        _norm("layer_norm_8192x8192", "bf16", 8192, 8192, p=0.1),
        # Its backward pass in an ordinary layer, the stream's own gradient added.
        _norm_backward("layer_norm_backward_8192x4096", "bf16", 8192, 4096, p=0.1),
        # Dropout of a sub-layer's output as it joins the stream.
        _dropout("dropout_16384x4096", "bf16", 16384, 4096, p=0.1),
        # A short batch of attention weights or embeddings, rows that are no whole vectors.
        _dropout("dropout_1001x3331", "f16", 1001, 3331, residual=False, p=0.3),
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
    op = rng.choice(["quantize", "decode", "matmul", "matmul", "backward", "layer_norm",
                     "layer_norm_backward", "dropout"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "quantize":
        return _quantize("", dtype, _size(rng, 1, 8192), _size(rng, 64, 8192), rng.choice([1, 128]))
    if op in ("layer_norm", "layer_norm_backward", "dropout"):
        p = round(rng.uniform(0.02, 0.5), 2)
        if op != "dropout" and rng.random() < 0.5:
            p = 0.0
        return _rows(op)("", dtype, _size(rng, 1, 8192), _size(rng, 64, 8192), rng.random() < 0.7, p)
    m = _size(rng, 1, 32) if op == "decode" else _size(rng, 32, 8192)
    n, k = _size(rng, 64, 8192), _size(rng, 64, 8192)
    if op == "backward":
        return _backward("", dtype, m, n, k)
    return _matmul("", dtype, m, n, k, rng.random() < 0.3)


# ---- inputs --------------------------------------------------------------------------------------


def _blocks(n):
    return -(-n // _BLOCK)


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


def _quantized(g, rows, cols, scale_rows, exponents):
    """8-bit numbers as rounding normal values to a block's scale gives them, and the scales, in the
    memory order that the quantizer gives them in: those of a block of columns are neighbours."""
    q = (torch.randn(rows, cols, generator=g, device=_DEV) * 120).clamp_(-_MOST, _MOST).to(_E4M3)
    e = torch.randint(*exponents, (_blocks(cols), scale_rows), generator=g, device=_DEV, dtype=torch.int32)
    return q, (e + 127).to(torch.uint8).view(_E8M0).t()


def prepare(case, seed):
    g = torch.Generator(device=_DEV)
    g.manual_seed(seed)
    op, dtype = case["op"], _TORCH[case["dtype"]]
    s = dict(case, dtype=dtype)
    if op in ("matmul", "backward"):
        m, n, k = case["m"], case["n"], case["k"]
        s["a"], s["a_scale"] = _quantized(g, m, k, m, (-9, -4))
        s["b"], s["b_scale"] = _quantized(g, n, k, _blocks(n), (-15, -12))
        if op == "backward":
            s["grad"] = _gradients(g, m, n, dtype)
        else:
            s["bias"] = torch.randn(n, generator=g, device=_DEV).to(dtype) if case["bias"] else None
        return s
    rows, cols = case["rows"], case["cols"]
    if op == "quantize":
        make = _gradients if case["block_rows"] > 1 else _activations  # a weight matrix: small, no outliers
        s["x"] = make(g, rows, cols, dtype)
        return s
    s["seed"], s["offset"] = (seed * 0x9E3779B97F4A7C15 + 12345) % 2 ** 63, seed % 97 * 2 ** 31
    s["x"] = _activations(g, rows, cols, dtype)
    other = _gradients if op == "layer_norm_backward" else _activations
    s["residual"] = other(g, rows, cols, dtype) if case["residual"] else None
    if op != "dropout":
        s["weight"] = (1 + 0.1 * torch.randn(cols, generator=g, device=_DEV)).to(dtype)
        s["bias"] = (0.1 * torch.randn(cols, generator=g, device=_DEV)).to(dtype)
    if op == "layer_norm_backward":  # x is the stored stream, with what the forward pass kept of its rows
        s["grad"] = _gradients(g, rows, cols, dtype)
        mean, rstd = _statistics(s["x"].float())
        s["mean"], s["rstd"] = mean[:, 0].contiguous(), rstd[:, 0].contiguous()
    return s


# ---- one pass ------------------------------------------------------------------------------------


def run(state):
    return (_OWN if own else _PLAIN)[state["op"]](state)


def _own_quantize(s):
    f, _ = _framework()
    q, scale = f.quantize(s["x"], s["block_rows"])
    return {"values": f.dequantize(q, scale, s["dtype"]), "scale": _powers(scale)}


def _own_matmul(s):
    return _framework()[0].matmul(s["a"], s["a_scale"], s["b"], s["b_scale"], s["bias"], s["dtype"])


def _own_backward(s):
    f, _ = _framework()
    return f.backward_a(s["grad"], s["b"], s["b_scale"]), f.backward_b(s["grad"], s["a"], s["a_scale"])


def _own_norm(s):
    y, h, mean, rstd = _framework()[1].layer_norm(s["x"], s["weight"], s["bias"], s["residual"], _EPS, s["p"],
                                                  s["seed"], s["offset"])
    return {"y": y, "h": h, "mean": mean, "rstd": rstd}


def _own_norm_backward(s):
    # "residual" is here the gradient that reaches the stream behind the norm.
    return _framework()[1].layer_norm_backward(s["grad"], s["x"], s["mean"], s["rstd"], s["weight"], s["residual"],
                                               s["p"], s["seed"], s["offset"])


def _own_dropout(s):
    return _framework()[1].dropout(s["x"], s["p"], s["seed"], s["offset"], s["residual"])


_OWN = {"quantize": _own_quantize, "matmul": _own_matmul, "backward": _own_backward, "layer_norm": _own_norm,
        "layer_norm_backward": _own_norm_backward, "dropout": _own_dropout}


def _powers(scale):
    """e8m0 scales as the f32 numbers they stand for."""
    return (scale.view(torch.uint8).to(torch.int32) << 23).view(torch.float32)


def _spread(scale, rows, cols):
    """Each element's scale of a matrix."""
    f = _powers(scale)
    if f.shape[0] != rows:
        f = f.repeat_interleave(_BLOCK, 0)[:rows]
    return f.repeat_interleave(_BLOCK, 1)[:, :cols]


def _plain_quantize(s):
    x, br = s["x"].float(), s["block_rows"]
    rows, cols = x.shape
    rb, cb = -(-rows // br), _blocks(cols)
    full = torch.nn.functional.pad(x.abs(), (0, cb * _BLOCK - cols, 0, rb * br - rows))
    top = full.view(rb, br, cb, _BLOCK).amax((1, 3))
    m, e = torch.frexp(top)  # top = m * 2^e, m in [0.5, 1): 448 = 0.875 * 2^9
    e = torch.where(m > 0.875, e - 8, e - 9).clamp_min(_LEAST_EXPONENT)
    e = torch.where(top == 0, _LEAST_EXPONENT, e)
    scale = ((e.to(torch.int32) + 127) << 23).view(torch.float32)
    each = scale.repeat_interleave(br, 0)[:rows].repeat_interleave(_BLOCK, 1)[:, :cols]
    return {"values": ((x / each).to(_E4M3).float() * each).to(s["dtype"]), "scale": scale}


def _plain_matmul(s):
    a = s["a"].float() * _spread(s["a_scale"], *s["a"].shape)
    b = s["b"].float() * _spread(s["b_scale"], *s["b"].shape)
    c = a @ b.t()
    if s["bias"] is not None:
        c = c + s["bias"].float()
    return c.to(s["dtype"])


def _plain_backward(s):
    grad = s["grad"].float()
    grad_a = grad @ (s["b"].float() * _spread(s["b_scale"], *s["b"].shape))
    grad_b = grad.t() @ (s["a"].float() * _spread(s["a_scale"], *s["a"].shape))
    return grad_a.to(s["dtype"]), grad_b.to(s["dtype"])


def _times(x, factor):
    """High and low 32 bits of x * factor, for 32-bit numbers held in 64."""
    low = x * (factor & 0xFFFF)
    high = x * (factor >> 16) + (low >> 16)
    return high >> 16, (high & 0xFFFF) << 16 | low & 0xFFFF


def _threshold(p):
    return int(np.rint(p * 65536))


def _kept(s, rows, cols):
    """Which elements dropout keeps: Philox4x32-10 with the seed as its key, counter (column / 8, row,
    offset) and 16 bits for each of eight columns."""
    groups = -(-cols // 8)
    c0 = torch.arange(groups, device=_DEV).expand(rows, groups)
    c1 = torch.arange(rows, device=_DEV)[:, None].expand(rows, groups)
    c2 = torch.full_like(c0, s["offset"] & 0xFFFFFFFF)
    c3 = torch.full_like(c0, s["offset"] >> 32)
    k0, k1 = s["seed"] & 0xFFFFFFFF, s["seed"] >> 32
    for _ in range(10):
        h0, l0 = _times(c0, 0xD2511F53)
        h1, l1 = _times(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    words = torch.stack([c0, c1, c2, c3], -1)
    halves = torch.stack([words & 0xFFFF, words >> 16], -1).view(rows, groups * 8)[:, :cols]
    return halves >= _threshold(s["p"])


def _dropped(s, x):
    if s["p"] == 0.0:
        return x
    keep = 65536.0 / (65536.0 - _threshold(s["p"]))
    return torch.where(_kept(s, *x.shape), x * float(np.float32(keep)), 0.0)


def _plain_dropout(s):
    y = _dropped(s, s["x"].float())
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["dtype"])


def _statistics(h):
    mean = h.mean(1, keepdim=True)
    return mean, 1.0 / torch.sqrt(((h - mean) * (h - mean)).mean(1, keepdim=True) + _EPS)


def _plain_norm(s):
    h = s["x"] if s["residual"] is None and s["p"] == 0.0 else _plain_dropout(s)
    mean, rstd = _statistics(h.float())
    y = (h.float() - mean) * rstd * s["weight"].float() + s["bias"].float()
    return {"y": y.to(s["dtype"]), "h": h, "mean": mean[:, 0], "rstd": rstd[:, 0]}


def _plain_norm_backward(s):
    grad, rstd = s["grad"].float(), s["rstd"][:, None]
    xhat, u = (s["x"].float() - s["mean"][:, None]) * rstd, grad * s["weight"].float()
    grad_h = rstd * (u - u.mean(1, keepdim=True) - xhat * (u * xhat).mean(1, keepdim=True))
    if s["residual"] is not None:
        grad_h = grad_h + s["residual"].float()
    dtype = s["dtype"]
    return (_dropped(s, grad_h).to(dtype), grad_h.to(dtype), (grad * xhat).sum(0).to(dtype), grad.sum(0).to(dtype))


_PLAIN = {"quantize": _plain_quantize, "matmul": _plain_matmul, "backward": _plain_backward,
          "layer_norm": _plain_norm, "layer_norm_backward": _plain_norm_backward, "dropout": _plain_dropout}


# ---- the definition in 64 bits -------------------------------------------------------------------


def _exact_factors(case, s):
    """Dropout's factor of each element (0 where it is dropped), by numpy in unsigned 64 bits, 1024
    rows at a time."""
    rows, cols = case["rows"], case["cols"]
    out = torch.empty(rows, cols, dtype=torch.float64, device=_DEV)
    low = np.uint64(0xFFFFFFFF)
    t = _threshold(case["p"])
    for first in range(0, rows, 1024):
        n = min(1024, rows - first)
        x = np.zeros((4, n, -(-cols // 8)), dtype=np.uint64)
        x[0] = np.arange(x.shape[2], dtype=np.uint64)
        x[1] = np.arange(first, first + n, dtype=np.uint64)[:, None]
        x[2], x[3] = s["offset"] % 2 ** 32, s["offset"] // 2 ** 32
        for turn in range(10):
            key = [(s["seed"] % 2 ** 32 + turn * 0x9E3779B9) % 2 ** 32, (s["seed"] // 2 ** 32 + turn * 0xBB67AE85) % 2 ** 32]
            p, q = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
            x = np.stack([(q >> np.uint64(32)) ^ x[1] ^ np.uint64(key[0]), q & low,
                          (p >> np.uint64(32)) ^ x[3] ^ np.uint64(key[1]), p & low])
        halves = np.ascontiguousarray(np.moveaxis(x.astype("<u4"), 0, -1)).view("<u2").reshape(n, -1)[:, :cols]
        out[first:first + n] = torch.from_numpy(halves >= t).to(_DEV).double()
    return out * (65536 / (65536 - t))


def _exact_power(e):
    """2^e in 64 bits from its bits: a power function rounds."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_exponent(v):
    """The largest e with 2^e <= v, for positive normal numbers."""
    return (v.view(torch.int64) >> 52) - 1023


def _exact_scaled(q, scale):
    """The numbers that a matrix of 8-bit numbers and its scales stand for."""
    rows, cols = q.shape
    f = _exact_power(scale.view(torch.uint8).to(torch.int64) - 127)
    per = 1 if f.shape[0] == rows else _BLOCK
    r = torch.arange(rows, device=_DEV) // per
    c = torch.arange(cols, device=_DEV) // _BLOCK
    return q.float().double() * f[r][:, c]


def _exact_quantize(case, s):
    x, br = s["x"].double(), case["block_rows"]
    rows, cols = x.shape
    values = torch.empty_like(x)
    scale = torch.empty(-(-rows // br), _blocks(cols), dtype=torch.float64, device=_DEV)
    for b in range(scale.shape[1]):
        part = x[:, b * _BLOCK:(b + 1) * _BLOCK]
        top = part.abs().max(1).values
        top = torch.cat([top, top.new_zeros(-rows % br)]).view(-1, br).max(1).values
        e = _exact_exponent(torch.clamp(top, min=2.0 ** (_LEAST_EXPONENT + 8))) - 8
        scale[:, b] = _exact_power(torch.where(_exact_power(e) * _MOST >= top, e, e + 1))
        each = scale[:, b].repeat_interleave(br)[:rows, None]
        v = part / each
        # e4m3: four significant bits down to 2^-6, steps of 2^-9 below.
        step = _exact_power(_exact_exponent(torch.clamp(v.abs(), min=2.0 ** -6)) - 3)
        values[:, b * _BLOCK:(b + 1) * _BLOCK] = torch.round(v / step) * step * each
    return {"values": values, "scale": scale}


def exact(case, seed):
    s = prepare(case, seed)
    wide = {key: v.double() for key, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()
            and v.dtype in (torch.float32, torch.float16, torch.bfloat16)}
    op = case["op"]
    if op == "quantize":
        return _exact_quantize(case, s)
    if op in ("matmul", "backward"):
        a, b = _exact_scaled(s["a"], s["a_scale"]), _exact_scaled(s["b"], s["b_scale"])
        if op == "backward":
            return torch.mm(wide["grad"], b), torch.mm(wide["grad"].t(), a)
        c = torch.mm(a, b.t())
        return c + wide["bias"] if case["bias"] else c
    factor = _exact_factors(case, s) if case["p"] > 0 else 1.0
    if op == "layer_norm_backward":
        xhat = (wide["x"] - wide["mean"][:, None]) * wide["rstd"][:, None]
        u = wide["grad"] * wide["weight"]
        inner = u - u.sum(1, keepdim=True) / case["cols"] - xhat * ((u * xhat).sum(1, keepdim=True) / case["cols"])
        grad_h = inner * wide["rstd"][:, None] + (wide["residual"] if case["residual"] else 0.0)
        return grad_h * factor, grad_h, (wide["grad"] * xhat).sum(0), wide["grad"].sum(0)
    h = wide["x"] * factor + (wide["residual"] if case["residual"] else 0.0)
    if op == "dropout":
        return h
    stored = _plain_dropout(s).double()  # the norm is of the stream as it is stored, rounded from 32 bits
    mean = stored.sum(1, keepdim=True) / case["cols"]
    rstd = ((stored - mean).pow(2).sum(1, keepdim=True) / case["cols"] + _EPS).pow(-0.5)
    return {"y": (stored - mean) * rstd * wide["weight"] + wide["bias"], "h": h, "mean": mean[:, 0], "rstd": rstd[:, 0]}


# ---- what a pass cannot do without ---------------------------------------------------------------


def work(case):
    """Each input read and each output written once; a product's multiply-adds count two."""
    size = _SIZE[case["dtype"]]
    if case["op"] in ("matmul", "backward"):
        m, n, k = case["m"], case["n"], case["k"]
        operands = (m + n) * k + _blocks(k) * (m + _blocks(n))
        if case["op"] == "backward":
            return {"bytes": size * (m * n + m * k + n * k) + operands, "flops": 4.0 * m * n * k}
        return {"bytes": operands + size * (m * n + case["bias"] * n), "flops": 2.0 * m * n * k}
    rows, cols = case["rows"], case["cols"]
    cells = rows * cols
    if case["op"] == "quantize":  # read, the 8-bit numbers, and their values
        scales = -(-rows // case["block_rows"]) * _blocks(cols)
        return {"bytes": cells * (2 * size + 1) + 4 * scales, "flops": 4.0 * cells}
    drop = case["p"] > 0
    if case["op"] == "dropout":
        return {"bytes": size * cells * (2 + case["residual"]), "flops": 15.0 * cells}
    edge = size * 2 * cols + 8 * rows
    if case["op"] == "layer_norm":  # x, residual, h, y
        streams = 2 + case["residual"] + (case["residual"] or drop)
        return {"bytes": size * streams * cells + edge, "flops": (8.0 + 15.0 * drop) * cells}
    # gradients of y and of h, h, the gradients of the residual and (another where elements drop) of x
    streams = 3 + case["residual"] + drop
    return {"bytes": size * streams * cells + edge + size * cols, "flops": (14.0 + 15.0 * drop) * cells}
