"""Layer norm and dropout: device tensors in, device tensors out.

What stands between the linear layers of a block, over ``tg_layer_norm``,
``tg_layer_norm_backward`` and ``tg_dropout`` of the C ABI.  No counterpart in the
reference.

* ``layer_norm``: dropout of a branch, the residual's addition and the norm in one
  pass; ``layer_norm_backward`` the gradients, of weight and bias too.
* ``dropout``: by itself, with or without the residual's addition.

Dropout stores no mask: a counter-based generator makes it from a seed, an offset
and an element's place, in the forward and again in the backward pass.  ``seed`` is
a whole number below 2**64, or an int64 tensor of one element on the GPU, read when
the kernel runs (a captured call then drops other elements in each replay if the
tensor changes).  Calls of one seed need different offsets, or they drop the same
elements.  The probability is ``p`` rounded to a multiple of 2**-16, and kept
elements are multiplied by the inverse of what it leaves.

Matrices are 2-D, bfloat16, float16 or float32; rows may be strided and start
anywhere, a row's elements must be neighbours.  Sums are f32.  Outputs and
workspaces come from torch's allocator, launches go to torch's current stream of
the inputs' device.  These functions do not record gradients themselves;
``tropical_gemm.pytorch`` joins them to autograd functions.
"""
from __future__ import annotations

import torch

from . import _native as nat
from .fp8 import _bytes
from .int8 import _F32, _FLOAT, _elsewhere, _matrix, _rows, _same_shape, _vector, _workspace
from .ops import _ptr, _stream


def _probability(p: float) -> float:
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p is {p}: a probability between 0 and 1 is expected")
    return p


def _random(seed, offset: int, dev: int):
    """(seed, address of the seed, offset)."""
    offset = int(offset)
    if not 0 <= offset < 1 << 64:
        raise ValueError(f"offset is {offset}: a number between 0 and 2**64 - 1 is expected")
    if isinstance(seed, torch.Tensor):
        if seed.get_device() != dev:
            _elsewhere("seed", seed, dev)
        if seed.dtype is not torch.int64 or seed.numel() != 1:
            raise ValueError(f"seed must be one int64 element, got {tuple(seed.shape)} of {seed.dtype}")
        return 0, seed.data_ptr(), offset
    seed = int(seed)
    if not 0 <= seed < 1 << 64:
        raise ValueError(f"seed is {seed}: a number between 0 and 2**64 - 1 is expected")
    return seed, None, offset


def dropout(x: torch.Tensor, p: float, seed, offset: int = 0, residual: torch.Tensor | None = None) -> torch.Tensor:
    """``dropout(x) + residual`` in x's type: elements are zero with probability
    ``p``, the others times ``1 / (1 - p)``.  Its gradient with respect to x is the
    same call on the gradient."""
    ldx = _rows("x", x)
    rows, cols = x.shape
    dev = x.device
    p = _probability(p)
    seed, seed_at, offset = _random(seed, offset, dev.index)
    ldr = 0
    if residual is not None:
        ldr = _rows("residual", residual, x.dtype, dev.index)
        _same_shape("residual", residual, x.shape)
    y = _matrix(rows, cols, x.dtype, dev)
    nat.check(nat.load().tg_dropout(dev.index, _FLOAT[x.dtype], x.data_ptr(), ldx, _ptr(residual), ldr, p, seed,
                                    seed_at, offset, y.data_ptr(), rows, cols, _stream(dev)))
    return y


def _drops(p: float) -> bool:
    return round(p * 65536) > 0


def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
               residual: torch.Tensor | None = None, eps: float = 1e-5, p: float = 0.0, seed=0, offset: int = 0):
    """``(y, h, mean, rstd)``: ``h = dropout(x) + residual`` in x's type (x itself
    where nothing is dropped or added), the mean and ``1 / sqrt(variance + eps)`` of
    its rows in f32, and ``y = (h - mean) * rstd * weight + bias`` in x's type.
    ``weight`` and ``bias`` are of x's type or both float32."""
    ldx = _rows("x", x)
    rows, cols = x.shape
    dev = x.device
    p = _probability(p)
    seed, seed_at, offset = _random(seed, offset, dev.index)
    _vector("weight", weight, cols, (x.dtype, torch.float32), dev.index)
    if bias is not None:
        _vector("bias", bias, cols, (weight.dtype,), dev.index)
    ldr, h = 0, x
    if residual is not None:
        ldr = _rows("residual", residual, x.dtype, dev.index)
        _same_shape("residual", residual, x.shape)
    if residual is not None or _drops(p):
        h = _matrix(rows, cols, x.dtype, dev)
    y = _matrix(rows, cols, x.dtype, dev)
    mean = torch.empty(rows, dtype=torch.float32, device=dev)
    rstd = torch.empty(rows, dtype=torch.float32, device=dev)
    if cols == 0:  # rows without a mean
        mean.fill_(float("nan"))
        rstd.fill_(float("nan"))
    nat.check(nat.load().tg_layer_norm(
        dev.index, _FLOAT[x.dtype], _FLOAT[weight.dtype], x.data_ptr(), ldx, _ptr(residual), ldr, weight.data_ptr(),
        _ptr(bias), eps, p, seed, seed_at, offset, y.data_ptr(), None if h is x else h.data_ptr(), mean.data_ptr(),
        rstd.data_ptr(), rows, cols, _stream(dev)))
    return y, h, mean, rstd


def layer_norm_backward(grad_y: torch.Tensor, h: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
                        weight: torch.Tensor, grad_h: torch.Tensor | None = None, p: float = 0.0, seed=0,
                        offset: int = 0):
    """``(grad_x, grad_residual, grad_weight, grad_bias)`` of ``layer_norm``, from
    the h, mean and rstd that it gave and the same p, seed and offset, with
    ``grad_h``, the gradient of h from elsewhere, added to grad_residual.  Without
    dropout grad_x is grad_residual itself.  Equal calls give equal bits."""
    ldh = _rows("h", h)
    rows, cols = h.shape
    dev = h.device
    p = _probability(p)
    seed, seed_at, offset = _random(seed, offset, dev.index)
    _same_shape("grad_y", grad_y, h.shape)
    ldg = _rows("grad_y", grad_y, h.dtype, dev.index)
    _vector("mean", mean, rows, _F32, dev.index)
    _vector("rstd", rstd, rows, _F32, dev.index)
    _vector("weight", weight, cols, (h.dtype, torch.float32), dev.index)
    ldgh = 0
    if grad_h is not None:
        _same_shape("grad_h", grad_h, h.shape)
        ldgh = _rows("grad_h", grad_h, h.dtype, dev.index)
    grad_residual = _matrix(rows, cols, h.dtype, dev)
    grad_x = _matrix(rows, cols, h.dtype, dev) if _drops(p) else grad_residual
    grad_weight = torch.empty(cols, dtype=weight.dtype, device=dev)
    grad_bias = torch.empty(cols, dtype=weight.dtype, device=dev)
    lib = nat.load()
    nbytes = _bytes(lib.tg_layer_norm_backward_workspace_size(rows, cols))
    ws = _workspace(nbytes, dev)
    nat.check(lib.tg_layer_norm_backward(
        dev.index, _FLOAT[h.dtype], _FLOAT[weight.dtype], grad_y.data_ptr(), ldg, h.data_ptr(), ldh, mean.data_ptr(),
        rstd.data_ptr(), weight.data_ptr(), _ptr(grad_h), ldgh, p, seed, seed_at, offset, grad_x.data_ptr(),
        grad_residual.data_ptr(), grad_weight.data_ptr(), grad_bias.data_ptr(), rows, cols, _ptr(ws), nbytes,
        _stream(dev)))
    return grad_x, grad_residual, grad_weight, grad_bias


__all__ = ["dropout", "layer_norm", "layer_norm_backward"]
