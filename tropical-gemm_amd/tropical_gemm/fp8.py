"""Linear layers in 8-bit floating point: device tensors in, device tensors out.

The operators of a linear layer whose operands are e4m3 numbers with one power
of two for each block of them, over the ``tg_f8_*`` entry points of the C ABI.
No counterpart in the reference.

* ``quantize`` / ``dequantize``: a matrix to 8-bit numbers with a scale for each
  1 x 128 (activations) or 128 x 128 elements (weights), and back.
* ``matmul``: 8-bit rows times the rows of an 8-bit weight matrix.
* ``backward_a`` / ``backward_b``: the gradients of that product, read from the
  8-bit operands.

8-bit numbers are ``torch.float8_e4m3fn``, scales ``torch.float8_e8m0fnu`` of
shape (row blocks, column blocks), in any strides.  ``quantize`` gives scales
whose rows are neighbours in memory (strides (1, rows)), which the products read
fastest.  Matrices are 2-D; rows may be strided and start anywhere, a row's
elements must be neighbours.  Activations and gradients are bfloat16, float16 or
float32, sums f32.  Outputs and workspaces come from torch's allocator, launches
go to torch's current stream of the inputs' device.  These functions do not
record gradients themselves; ``tropical_gemm.pytorch`` joins them to autograd
functions.
"""
from __future__ import annotations

import torch

from . import _native as nat
from .int8 import _FLOAT, _elsewhere, _float_type, _matrix, _rows, _vector, _workspace
from .ops import _ptr, _stream

BLOCK = 128
_E4M3, _E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _bytes(size: int) -> int:
    """A size function's answer; what it has none for is refused by the call."""
    return 0 if size == nat.SIZE_MAX else size


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


def _scale(name: str, t: torch.Tensor, rows: int, cols: int, dev: int):
    """Checks a matrix of scales; its strides."""
    if t.get_device() != dev:
        _elsewhere(name, t, dev)
    if t.dtype is not _E8M0:
        raise ValueError(f"{name} must be {_E8M0}, got {t.dtype}")
    if t.shape != (rows, _blocks(cols)):
        raise ValueError(f"Dimension mismatch: {name} has shape {tuple(t.shape)}, expected {(rows, _blocks(cols))}")
    row, col = t.stride()
    return (0 if rows <= 1 else row), col


def quantize(x: torch.Tensor, block_rows: int = 1):
    """``(q, scale)`` of the blocks of ``block_rows`` (1 or 128) x 128 elements of
    ``x``: ``scale = 2**e`` with the least e (at least -100) for which no
    magnitude of the block passes ``448 * 2**e``, ``q = x / scale`` rounded to
    e4m3.  A block that holds a NaN or an infinity becomes NaNs."""
    ld = _rows("x", x)
    rows, cols = x.shape
    if block_rows not in (1, BLOCK):
        raise ValueError(f"block_rows is {block_rows}: expected 1 or {BLOCK}")
    dev = x.device
    q = _matrix(rows, cols, _E4M3, dev)
    rb = rows if block_rows == 1 else _blocks(rows)
    scale = torch.empty_strided((rb, _blocks(cols)), (1, max(rb, 1)), dtype=_E8M0, device=dev)
    nat.check(nat.load().tg_f8_quantize(dev.index, _FLOAT[x.dtype], x.data_ptr(), ld, block_rows, q.data_ptr(),
                                        scale.data_ptr(), rows, cols, _stream(dev)))
    return q, scale


def dequantize(q: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The numbers that ``q`` and its scales stand for, rounded to ``dtype``; the
    blocks' height follows from the scales' shape."""
    ld = _rows("q", q, _E4M3)
    rows, cols = q.shape
    dev = q.device
    block_rows = 1 if scale.dim() > 0 and scale.shape[0] == rows else BLOCK
    row, col = _scale("scale", scale, rows if block_rows == 1 else _blocks(rows), cols, dev.index)
    kind = _float_type(dtype)
    y = _matrix(rows, cols, dtype, dev)
    nat.check(nat.load().tg_f8_dequantize(dev.index, kind, q.data_ptr(), ld, scale.data_ptr(), row, col, block_rows,
                                          y.data_ptr(), rows, cols, _stream(dev)))
    return y


def matmul(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor,
           bias: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``A @ B.T + bias`` in ``dtype``, of the numbers that the operands stand for:
    ``a`` (m, k) with scales for 1 x 128 elements, ``b`` (n, k) a weight matrix with
    one row for each output and scales for 128 x 128, ``bias`` of ``dtype``.

    For 16-bit outputs the matrix instructions add eight neighbouring products at a
    time and drop of them what lies 2**-13 below the largest, as it would be with
    operands that are not zero taken as 2**-6 at least (before their scales): up to
    2**-10 of the sum of the products' magnitudes so taken (more than float16's own
    rounding), 1.5e-5 of the result in the mean of normal values.  Where large
    products cancel, nothing bounds that by the result.  float32 outputs are made of exact products (scales of 2**-100
    to 2**111) and sums of f32; those of many rows take about twice the time."""
    dev = a.device
    lda = _rows("a", a, _E4M3)
    ldb = _rows("b", b, _E4M3, dev.index)
    m, k = a.shape
    n, k2 = b.shape
    if k != k2:
        raise ValueError(f"Dimension mismatch: a is {m}x{k}, b is {n}x{k2}")
    a_row, a_col = _scale("a_scale", a_scale, m, k, dev.index)
    b_row, b_col = _scale("b_scale", b_scale, _blocks(n), k, dev.index)
    kind = _float_type(dtype)
    if bias is not None:
        _vector("bias", bias, n, (dtype,), dev.index)
    c = _matrix(m, n, dtype, dev)
    lib = nat.load()
    pa, pb = a.data_ptr(), b.data_ptr()
    nbytes = _bytes(lib.tg_f8_gemm_workspace_size(kind, pa, lda, pb, ldb, m, n, k))
    ws = _workspace(nbytes, dev)
    nat.check(lib.tg_f8_gemm(dev.index, kind, pa, lda, a_scale.data_ptr(), a_row, a_col, pb, ldb, b_scale.data_ptr(),
                             b_row, b_col, _ptr(bias), c.data_ptr(), m, n, k, _ptr(ws), nbytes, _stream(dev)))
    return c


def _backward(which: str, grad_c: torch.Tensor, q: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    dev = grad_c.device
    ldg = _rows("grad_c", grad_c)
    other = "b" if which == "a" else "a"
    ldq = _rows(other, q, _E4M3, dev.index)
    m, n = grad_c.shape
    depth, k = q.shape
    if depth != (n if which == "a" else m):
        raise ValueError(f"Dimension mismatch: grad_c is {m}x{n}, {other} is {depth}x{k}")
    row, col = _scale(f"{other}_scale", scale, _blocks(n) if which == "a" else m, k, dev.index)
    out = _matrix(m if which == "a" else n, k, grad_c.dtype, dev)
    lib = nat.load()
    size, run = ((lib.tg_f8_backward_a_workspace_size, lib.tg_f8_backward_a) if which == "a" else
                 (lib.tg_f8_backward_b_workspace_size, lib.tg_f8_backward_b))
    kind = _FLOAT[grad_c.dtype]
    nbytes = _bytes(size(kind, grad_c.data_ptr(), ldg, m, n, k))
    ws = _workspace(nbytes, dev)
    nat.check(run(dev.index, kind, grad_c.data_ptr(), ldg, q.data_ptr(), ldq, scale.data_ptr(), row, col,
                  out.data_ptr(), m, n, k, _ptr(ws), nbytes, _stream(dev)))
    return out


def backward_a(grad_c: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor) -> torch.Tensor:
    """``grad_c @ B`` of the numbers that ``b`` stands for: the gradient of matmul's
    activations, in grad_c's type."""
    return _backward("a", grad_c, b, b_scale)


def backward_b(grad_c: torch.Tensor, a: torch.Tensor, a_scale: torch.Tensor) -> torch.Tensor:
    """``grad_c.T @ A`` of the numbers that ``a`` stands for: the gradient of
    matmul's weights, in grad_c's type, from the 8-bit activations that the
    forward pass kept."""
    return _backward("b", grad_c, a, a_scale)


__all__ = ["quantize", "dequantize", "matmul", "backward_a", "backward_b"]
