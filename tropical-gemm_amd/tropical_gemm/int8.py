"""Linear layers in 8 bits: device tensors in, device tensors out.

The operators a linear layer needs beside the tropical products, over the
``tg_i8_*`` entry points of the C ABI.  No counterpart in the reference.

* ``quantize`` / ``dequantize``: rows to 8-bit integers with one f32 scale each,
  and back: a layer's activations kept for its backward pass in half the bytes.
* ``rms_norm``: the residual's addition, the RMS norm and its 8-bit output in
  one pass; ``rms_norm_backward`` its gradients.
* ``matmul``: 8-bit rows times the rows of an 8-bit weight matrix, with a scale
  for each token and each output channel.
* ``backward_a`` / ``backward_b``: the gradients of that product, read from the
  8-bit operands.

``tropical_gemm.pytorch`` joins them to autograd functions.  Matrices are 2-D;
rows may be strided (a slice of a wider matrix) and start anywhere, a row's
elements must be neighbours.  Activations and gradients are bfloat16, float16
or float32; sums and scales are f32 (i32 for 8-bit products).  Outputs and
workspaces come from torch's allocator, launches go to torch's current stream
of the inputs' device.  These functions do not record gradients themselves.
"""
from __future__ import annotations

import torch

from . import _native as nat
from .ops import _ptr, _stream

_FLOAT = {torch.float32: nat.FLOAT["f32"], torch.bfloat16: nat.FLOAT["bf16"],
          torch.float16: nat.FLOAT["f16"]}
_F32 = (torch.float32,)


def _elsewhere(name: str, t: torch.Tensor, dev: int | None):
    if dev is None:
        raise ValueError("tropical_gemm GPU entry points need device tensors "
                         f"({name} is on {t.device.type}); move the tensors to the GPU first")
    raise ValueError(f"Tensors must be on the same device, cuda:{dev}: {name} is on {t.device}")


# The checks take the device as an index: comparing torch.device objects costs
# a small call as much as an allocation.
def _rows(name: str, t: torch.Tensor, dtype=None, dev: int | None = None) -> int:
    """Checks a matrix on a GPU (on `dev`) whose rows are neighbours; its row stride."""
    on = t.get_device()
    if on < 0 or dev is not None and on != dev:
        _elsewhere(name, t, dev)
    if t.dim() != 2:
        raise ValueError(f"Expected a 2D tensor for {name}, got {t.dim()} dims")
    if dtype is None:
        if t.dtype not in _FLOAT:
            raise ValueError(f"Unsupported dtype {t.dtype} of {name}: expected bfloat16, float16 or float32")
    elif t.dtype is not dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.is_contiguous():
        return t.shape[1]
    rows, cols = t.shape
    ld, step = t.stride()
    if rows <= 1:
        ld = cols
    if (cols > 1 and step != 1) or ld < cols:
        raise ValueError(f"The elements of a row of {name} must be neighbours and its rows apart, got strides "
                         f"{tuple(t.stride())} (call .contiguous() on PyTorch tensors)")
    return ld


def _vector(name: str, t: torch.Tensor, n: int, dtypes, dev: int) -> None:
    if t.shape != (n,):
        raise ValueError(f"Dimension mismatch: {name} has shape {tuple(t.shape)}, expected ({n},)")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must be {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")
    if t.get_device() != dev:
        _elsewhere(name, t, dev)
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous (call .contiguous() on PyTorch tensors)")


def _same_shape(name: str, t: torch.Tensor, shape) -> None:
    if t.shape != shape:
        raise ValueError(f"Dimension mismatch: {name} has shape {tuple(t.shape)}, expected {tuple(shape)}")


def _matrix(rows: int, cols: int, dtype, dev: torch.device) -> torch.Tensor:
    # Given strides, torch allocates in 1.3 us, not 1.6: a small call takes 9.
    return torch.empty_strided((rows, cols), (cols, 1), dtype=dtype, device=dev)


def _workspace(nbytes: int, dev: torch.device):
    return torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None


def quantize(x: torch.Tensor):
    """``(q, scale)`` of each row of ``x``: ``scale = max|x| / 127`` (f32) and
    ``q = rint(x / scale)`` (int8), so that ``q * scale`` is x to half a step.
    A row of zeros gives zeros; a row that holds a NaN or an infinity gives
    values that are NaN."""
    ld = _rows("x", x)
    rows, cols = x.shape
    dev = x.device
    q = _matrix(rows, cols, torch.int8, dev)
    scale = torch.empty(rows, dtype=torch.float32, device=dev)
    nat.check(nat.load().tg_i8_quantize(dev.index, _FLOAT[x.dtype], x.data_ptr(), ld, q.data_ptr(),
                                        scale.data_ptr(), rows, cols, _stream(dev)))
    return q, scale


def dequantize(q: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``q * scale[:, None]`` rounded to ``dtype``."""
    ld = _rows("q", q, torch.int8)
    rows, cols = q.shape
    dev = q.device
    _vector("scale", scale, rows, _F32, dev.index)
    _float_type(dtype)
    y = _matrix(rows, cols, dtype, dev)
    nat.check(nat.load().tg_i8_dequantize(dev.index, _FLOAT[dtype], q.data_ptr(), ld, scale.data_ptr(),
                                          y.data_ptr(), rows, cols, _stream(dev)))
    return y


def _float_type(dtype: torch.dtype) -> int:
    if dtype not in _FLOAT:
        raise ValueError(f"Unsupported dtype {dtype}: expected bfloat16, float16 or float32")
    return _FLOAT[dtype]


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, eps: float = 1e-6):
    """``(q, scale, h)``: ``h = x + residual`` in x's type (x itself without a
    residual), and ``h * rsqrt(mean(h^2) + eps) * weight`` as 8-bit rows with
    scales.  ``weight`` is of x's type or float32."""
    ldx = _rows("x", x)
    rows, cols = x.shape
    dev = x.device
    _vector("weight", weight, cols, (x.dtype, torch.float32), dev.index)
    ldr, h = 0, x
    if residual is not None:
        ldr = _rows("residual", residual, x.dtype, dev.index)
        _same_shape("residual", residual, x.shape)
        h = _matrix(rows, cols, x.dtype, dev)
    q = _matrix(rows, cols, torch.int8, dev)
    scale = torch.empty(rows, dtype=torch.float32, device=dev)
    nat.check(nat.load().tg_i8_rms_norm(
        dev.index, _FLOAT[x.dtype], _FLOAT[weight.dtype], x.data_ptr(), ldx, _ptr(residual), ldr,
        weight.data_ptr(), eps, q.data_ptr(), scale.data_ptr(), None if residual is None else h.data_ptr(), rows,
        cols, _stream(dev)))
    return q, scale, h


def rms_norm_backward(grad_y: torch.Tensor, h: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
                      grad_h: torch.Tensor | None = None):
    """``(grad_x, grad_weight)`` of ``rms_norm`` for the gradient of its
    normalised output (the rounding to 8 bits passes it on unchanged), with
    ``grad_h``, the gradient of the stream h from elsewhere, added to grad_x.
    grad_x is the gradient of x and of the residual.  Equal calls give equal
    bits."""
    dev = h.device
    ldh = _rows("h", h)
    rows, cols = h.shape
    _same_shape("grad_y", grad_y, h.shape)
    ldg = _rows("grad_y", grad_y, h.dtype, dev.index)
    _vector("weight", weight, cols, (h.dtype, torch.float32), dev.index)
    ldgh = 0
    if grad_h is not None:
        _same_shape("grad_h", grad_h, h.shape)
        ldgh = _rows("grad_h", grad_h, h.dtype, dev.index)
    grad_x = _matrix(rows, cols, h.dtype, dev)
    grad_weight = torch.empty(cols, dtype=weight.dtype, device=dev)
    lib = nat.load()
    nbytes = lib.tg_i8_rms_norm_backward_workspace_size(rows, cols)
    ws = _workspace(nbytes, dev)
    nat.check(lib.tg_i8_rms_norm_backward(
        dev.index, _FLOAT[h.dtype], _FLOAT[weight.dtype], grad_y.data_ptr(), ldg, h.data_ptr(), ldh,
        weight.data_ptr(), eps, _ptr(grad_h), ldgh, grad_x.data_ptr(), grad_weight.data_ptr(), rows, cols,
        _ptr(ws), nbytes, _stream(dev)))
    return grad_x, grad_weight


def matmul(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor,
           bias: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``(a @ b.T) * a_scale[:, None] * b_scale + bias`` in ``dtype``: ``a`` (m, k)
    int8 activations, ``b`` (n, k) an int8 weight matrix with one row for each
    output, f32 scales, ``bias`` of ``dtype``.  The integer sum is exact
    (k < 2**17)."""
    dev = a.device
    lda = _rows("a", a, torch.int8)
    ldb = _rows("b", b, torch.int8, dev.index)
    m, k = a.shape
    n, k2 = b.shape
    if k != k2:
        raise ValueError(f"Dimension mismatch: a is {m}x{k}, b is {n}x{k2}")
    _vector("a_scale", a_scale, m, _F32, dev.index)
    _vector("b_scale", b_scale, n, _F32, dev.index)
    kind = _float_type(dtype)
    if bias is not None:
        _vector("bias", bias, n, (dtype,), dev.index)
    c = _matrix(m, n, dtype, dev)
    lib = nat.load()
    pa, pb = a.data_ptr(), b.data_ptr()
    nbytes = lib.tg_i8_gemm_workspace_size(pa, lda, pb, ldb, m, n, k) if k < 1 << 17 else 0
    ws = _workspace(nbytes, dev)
    nat.check(lib.tg_i8_gemm(dev.index, kind, pa, lda, a_scale.data_ptr(), pb, ldb, b_scale.data_ptr(),
                             _ptr(bias), c.data_ptr(), m, n, k, _ptr(ws), nbytes, _stream(dev)))
    return c


def _backward(which: str, grad_c: torch.Tensor, q: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    dev = grad_c.device
    ldg = _rows("grad_c", grad_c)
    other = "b" if which == "a" else "a"
    ldq = _rows(other, q, torch.int8, dev.index)
    m, n = grad_c.shape
    depth, k = q.shape
    if depth != (n if which == "a" else m):
        raise ValueError(f"Dimension mismatch: grad_c is {m}x{n}, {other} is {depth}x{k}")
    _vector(f"{other}_scale", scale, depth, _F32, dev.index)
    out = _matrix(m if which == "a" else n, k, grad_c.dtype, dev)
    lib = nat.load()
    size, run = ((lib.tg_i8_backward_a_workspace_size, lib.tg_i8_backward_a) if which == "a" else
                 (lib.tg_i8_backward_b_workspace_size, lib.tg_i8_backward_b))
    kind = _FLOAT[grad_c.dtype]
    nbytes = size(kind, grad_c.data_ptr(), ldg, m, n, k)
    ws = _workspace(nbytes, dev)
    nat.check(run(dev.index, kind, grad_c.data_ptr(), ldg, q.data_ptr(), ldq, scale.data_ptr(),
                  out.data_ptr(), m, n, k, _ptr(ws), nbytes, _stream(dev)))
    return out


def backward_a(grad_c: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor) -> torch.Tensor:
    """``grad_c @ (b * b_scale[:, None])``: the gradient of matmul's activations
    ``a * a_scale[:, None]``, in grad_c's type."""
    return _backward("a", grad_c, b, b_scale)


def backward_b(grad_c: torch.Tensor, a: torch.Tensor, a_scale: torch.Tensor) -> torch.Tensor:
    """``grad_c.T @ (a * a_scale[:, None])``: the gradient of matmul's weights
    ``b * b_scale[:, None]``, in grad_c's type, from the 8-bit activations that
    the forward pass kept."""
    return _backward("b", grad_c, a, a_scale)


__all__ = ["quantize", "dequantize", "rms_norm", "rms_norm_backward", "matmul", "backward_a", "backward_b"]
