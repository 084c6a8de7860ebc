"""PyTorch autograd functions for tropical matmul on MI355X.

Mirrors the GPU and batched classes of the reference
(``crates/tropical-gemm-python/python/tropical_gemm/pytorch.py:338-860``):
same class and function names, same forward outputs, same gradient rules.

Differences that are deliberate:

* The backward runs the library's HIP scatter kernels (``tg_backward_*``)
  instead of ``torch.scatter_add_`` (reference ``pytorch.py:386-403``);
  the math is identical: ``grad_a[i, k*] += grad_c[i, j]``,
  ``grad_b[k*, j] += grad_c[i, j]`` and, for MaxMul, the multiplicative rule
  ``grad_a[i, k*] += grad_c[i, j] * B[k*, j]``, ``grad_b[k*, j] += grad_c[i, j] * A[i, k*]``
  (``pytorch.py:521-548``).
* float32 and float64 are both accepted on the GPU (the reference's DLPack
  path takes float32 only, ``python/src/lib.rs:2193-2197``).
* The argmax saved for backward stays int32 on the device (the reference
  widens it to int64 for ``scatter_add_``).
* The reference's CPU autograd classes (Rust SIMD backend) are not part of
  this backend; the batched classes require device tensors.
"""
from __future__ import annotations

import torch

from . import cuda_available, fp8, int8, layers, ops

GPU_AVAILABLE = cuda_available()
_DLPACK_AVAILABLE = True
_BATCHED_DLPACK_AVAILABLE = True

_GRAD_DTYPES = (torch.float32, torch.float64)


def _prep(a: torch.Tensor, b: torch.Tensor, name: str, cpu_name: str):
    if not a.is_cuda:
        raise RuntimeError(f"{name} requires GPU tensors. Use {cpu_name} for CPU tensors.")
    if a.device != b.device:
        raise RuntimeError(
            f"Tensors must be on the same device: a is on {a.device}, b is on {b.device}")
    if a.dtype not in _GRAD_DTYPES or b.dtype != a.dtype:
        raise RuntimeError(f"{name} supports float32/float64 tensors of one dtype, got "
                           f"{a.dtype} and {b.dtype}")
    return a.detach().contiguous(), b.detach().contiguous()


def _additive_forward(ctx, a, b, semiring: str, name: str, cpu_name: str):
    a_c, b_c = _prep(a, b, name, cpu_name)
    c, argmax = ops.gemm(semiring, a_c, b_c, True)
    ctx.save_for_backward(argmax)
    ctx.k = a.shape[1]
    ctx.m = a.shape[0]
    ctx.n = b.shape[1]
    return c


class _AdditiveGPU(torch.autograd.Function):

    @staticmethod
    def backward(ctx, grad_c: torch.Tensor):
        (argmax,) = ctx.saved_tensors
        grad_a = grad_b = None
        if ctx.needs_input_grad[0]:
            grad_a = ops.backward_a(grad_c, argmax, ctx.k)
        if ctx.needs_input_grad[1]:
            grad_b = ops.backward_b(grad_c, argmax, ctx.k)
        return grad_a, grad_b


class TropicalMaxPlusMatmulGPU(_AdditiveGPU):
    """GPU MaxPlus matmul ``C[i,j] = max_k A[i,k] + B[k,j]`` (pytorch.py:338-403)."""

    @staticmethod
    def forward(ctx, a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
        return _additive_forward(ctx, a, b, "maxplus", "TropicalMaxPlusMatmulGPU",
                                 "TropicalMaxPlusMatmul")


class TropicalMinPlusMatmulGPU(_AdditiveGPU):
    """GPU MinPlus matmul ``C[i,j] = min_k A[i,k] + B[k,j]`` (pytorch.py:406-468)."""

    @staticmethod
    def forward(ctx, a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
        return _additive_forward(ctx, a, b, "minplus", "TropicalMinPlusMatmulGPU",
                                 "TropicalMinPlusMatmul")


class TropicalMaxMulMatmulGPU(torch.autograd.Function):
    """GPU MaxMul matmul ``C[i,j] = max_k A[i,k] * B[k,j]`` with the
    multiplicative backward (pytorch.py:471-548)."""

    @staticmethod
    def forward(ctx, a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
        a_c, b_c = _prep(a, b, "TropicalMaxMulMatmulGPU", "TropicalMaxMulMatmul")
        c, argmax = ops.gemm("maxmul", a_c, b_c, True)
        ctx.save_for_backward(a_c, b_c, argmax)
        ctx.k = a.shape[1]
        ctx.m = a.shape[0]
        ctx.n = b.shape[1]
        return c

    @staticmethod
    def backward(ctx, grad_c: torch.Tensor):
        a, b, argmax = ctx.saved_tensors
        grad_a = grad_b = None
        if ctx.needs_input_grad[0]:
            grad_a = ops.backward_a(grad_c, argmax, ctx.k, b=b)
        if ctx.needs_input_grad[1]:
            grad_b = ops.backward_b(grad_c, argmax, ctx.k, a=a)
        return grad_a, grad_b


def _prep_batched(a: torch.Tensor, b: torch.Tensor):
    if not (a.is_cuda or b.is_cuda):
        raise RuntimeError("Batched tropical matmul on this backend requires GPU tensors; the "
                           "reference's CPU batched path is not part of it.")
    if a.device != b.device:
        raise RuntimeError(
            f"Tensors must be on the same device: a is on {a.device}, b is on {b.device}")
    if a.dtype not in _GRAD_DTYPES or b.dtype != a.dtype:
        raise RuntimeError(f"Batched GPU tropical matmul supports float32/float64 tensors of one "
                           f"dtype, got {a.dtype} and {b.dtype}")
    return a.detach().contiguous(), b.detach().contiguous()


def _additive_batched_forward(ctx, a, b, semiring: str):
    a_c, b_c = _prep_batched(a, b)
    c, argmax = ops.gemm_batched(semiring, a_c, b_c, True)
    ctx.save_for_backward(argmax)
    ctx.k = a.shape[2]
    ctx.batch = a.shape[0]
    ctx.m = a.shape[1]
    ctx.n = b.shape[2]
    return c


class _AdditiveBatched(torch.autograd.Function):

    @staticmethod
    def backward(ctx, grad_c: torch.Tensor):
        (argmax,) = ctx.saved_tensors
        grad_a = grad_b = None
        if ctx.needs_input_grad[0]:
            grad_a = ops.backward_a_batched(grad_c, argmax, ctx.k)
        if ctx.needs_input_grad[1]:
            grad_b = ops.backward_b_batched(grad_c, argmax, ctx.k)
        return grad_a, grad_b


class TropicalMaxPlusMatmulBatched(_AdditiveBatched):
    """Batched MaxPlus ``C[b,i,j] = max_k A[b,i,k] + B[b,k,j]`` (pytorch.py:556-640)."""

    @staticmethod
    def forward(ctx, a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
        return _additive_batched_forward(ctx, a, b, "maxplus")


class TropicalMinPlusMatmulBatched(_AdditiveBatched):
    """Batched MinPlus ``C[b,i,j] = min_k A[b,i,k] + B[b,k,j]`` (pytorch.py:643-730)."""

    @staticmethod
    def forward(ctx, a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
        return _additive_batched_forward(ctx, a, b, "minplus")


class TropicalMaxMulMatmulBatched(torch.autograd.Function):
    """Batched MaxMul with the multiplicative backward (pytorch.py:733-832)."""

    @staticmethod
    def forward(ctx, a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
        a_c, b_c = _prep_batched(a, b)
        c, argmax = ops.gemm_batched("maxmul", a_c, b_c, True)
        ctx.save_for_backward(a_c, b_c, argmax)
        ctx.k = a.shape[2]
        ctx.batch = a.shape[0]
        ctx.m = a.shape[1]
        ctx.n = b.shape[2]
        return c

    @staticmethod
    def backward(ctx, grad_c: torch.Tensor):
        a, b, argmax = ctx.saved_tensors
        grad_a = grad_b = None
        if ctx.needs_input_grad[0]:
            grad_a = ops.backward_a_batched(grad_c, argmax, ctx.k, b=b)
        if ctx.needs_input_grad[1]:
            grad_b = ops.backward_b_batched(grad_c, argmax, ctx.k, a=a)
        return grad_a, grad_b


def tropical_maxplus_matmul_gpu(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """GPU MaxPlus tropical matmul (pytorch.py:910-924)."""
    return TropicalMaxPlusMatmulGPU.apply(a, b)


def tropical_minplus_matmul_gpu(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """GPU MinPlus tropical matmul (pytorch.py:927-941)."""
    return TropicalMinPlusMatmulGPU.apply(a, b)


def tropical_maxmul_matmul_gpu(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """GPU MaxMul tropical matmul (pytorch.py:944-958)."""
    return TropicalMaxMulMatmulGPU.apply(a, b)


def tropical_maxplus_matmul_batched(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """Batched MaxPlus tropical matmul (pytorch.py:961-973)."""
    return TropicalMaxPlusMatmulBatched.apply(a, b)


def tropical_minplus_matmul_batched(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """Batched MinPlus tropical matmul (pytorch.py:976-988)."""
    return TropicalMinPlusMatmulBatched.apply(a, b)


def tropical_maxmul_matmul_batched(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """Batched MaxMul tropical matmul (pytorch.py:991-1003)."""
    return TropicalMaxMulMatmulBatched.apply(a, b)


# ---------------------------------------------------------------------------
# Linear layers in 8 bits (no counterpart in the reference)
# ---------------------------------------------------------------------------

def _prep_int8(name: str, x: torch.Tensor, weight: torch.Tensor):
    if not x.is_cuda or not weight.is_cuda:
        raise RuntimeError(f"{name} requires GPU tensors.")
    if x.dim() != 2 or weight.dim() != 2 or x.shape[1] != weight.shape[1]:
        raise RuntimeError(f"{name} expects activations (tokens, k) and weights (n, k), got "
                           f"{tuple(x.shape)} and {tuple(weight.shape)}")
    if x.dtype != weight.dtype:
        raise RuntimeError(f"{name} expects one dtype, got {x.dtype} and {weight.dtype}")
    return x.detach().contiguous(), weight.detach().contiguous()


def _int8_product_backward(grad, q, scale, qw, scale_w, want_x: bool, want_w: bool):
    grad = grad.contiguous()
    return (int8.backward_a(grad, qw, scale_w) if want_x else None,
            int8.backward_b(grad, q, scale) if want_w else None)


class _FirstDerivative(torch.autograd.Function):
    """A gradient as it is, whose own gradient is an error."""

    @staticmethod
    def forward(ctx, name: str, grad: torch.Tensor) -> torch.Tensor:
        ctx.name = name
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, _):
        raise RuntimeError(f"{ctx.name} has no second derivatives: its gradients cannot be differentiated again.")


def _first_derivatives(name: str, *grads):
    """The gradients of a backward pass whose kernels record nothing.  Where the
    caller asked for a graph of that pass (``create_graph=True``), they are part
    of one that refuses, or a loss that holds them would silently lack their
    derivatives.  (``once_differentiable`` marks them only where the incoming
    gradient needs one itself, which a loss's ones do not.)"""
    if not torch.is_grad_enabled():
        return grads
    return tuple(g if g is None else _FirstDerivative.apply(name, g.detach().requires_grad_()) for g in grads)


class Int8LinearGPU(torch.autograd.Function):
    """``y = x @ weight.T`` with both operands rounded to 8-bit rows, one scale
    for each token and each output channel.

    The backward pass reads the 8-bit rows, which are all that is kept of the
    operands (half of bfloat16's bytes): the gradients are those of the product
    of the rounded operands, passed through the rounding unchanged.  They have
    no gradients of their own: differentiating them is an error."""

    @staticmethod
    def forward(ctx, x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
        x, weight = _prep_int8("Int8LinearGPU", x, weight)
        q, scale = int8.quantize(x)
        qw, scale_w = int8.quantize(weight)
        ctx.save_for_backward(q, scale, qw, scale_w)
        return int8.matmul(q, scale, qw, scale_w, dtype=x.dtype)

    @staticmethod
    def backward(ctx, grad_y: torch.Tensor):
        with torch.no_grad():
            grads = _int8_product_backward(grad_y, *ctx.saved_tensors, *ctx.needs_input_grad)
        return _first_derivatives("Int8LinearGPU", *grads)


class RmsNormInt8LinearGPU(torch.autograd.Function):
    """``(y, h)`` of one step of a residual stream: ``h = x + residual``,
    ``y = rms_norm(h, norm_weight, eps) @ weight.T``, the norm's output rounded
    to 8-bit rows as it is made and the weights to 8-bit rows beside it.

    Kept for the backward pass: h, the 8-bit rows and the scales.  The gradients
    have no gradients of their own: differentiating them is an error."""

    @staticmethod
    def forward(ctx, x, residual, norm_weight, weight, eps: float = 1e-6):
        name = "RmsNormInt8LinearGPU"
        x, weight = _prep_int8(name, x, weight)
        norm_weight = norm_weight.detach().contiguous()
        residual = None if residual is None else residual.detach().contiguous()
        q, scale, h = int8.rms_norm(x, norm_weight, residual, eps)
        if residual is None:
            h = x.clone()  # an output that shares no memory with an input
        qw, scale_w = int8.quantize(weight)
        ctx.save_for_backward(h, norm_weight, q, scale, qw, scale_w)
        ctx.eps = eps
        ctx.set_materialize_grads(False)
        return int8.matmul(q, scale, qw, scale_w, dtype=x.dtype), h

    @staticmethod
    def backward(ctx, grad_y, grad_h):
        h, norm_weight, q, scale, qw, scale_w = ctx.saved_tensors
        want_x, want_r, want_nw, want_w, _ = ctx.needs_input_grad
        want_norm = want_x or want_r or want_nw
        if grad_y is None:
            return grad_h, grad_h if want_r else None, None, None, None
        with torch.no_grad():
            grad_n, grad_w = _int8_product_backward(grad_y, q, scale, qw, scale_w, want_norm, want_w)
            grad_x = grad_nw = None
            if want_norm:
                grad_h = None if grad_h is None else grad_h.contiguous()
                grad_x, grad_nw = int8.rms_norm_backward(grad_n, h, norm_weight, ctx.eps, grad_h)
        grad_x, grad_nw, grad_w = _first_derivatives("RmsNormInt8LinearGPU", grad_x, grad_nw, grad_w)
        return grad_x, grad_x if want_r else None, grad_nw, grad_w, None


def int8_linear_gpu(x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    """``x @ weight.T`` in 8 bits, with gradients (``Int8LinearGPU``)."""
    return Int8LinearGPU.apply(x, weight)


def rms_norm_int8_linear_gpu(x: torch.Tensor, residual: torch.Tensor | None, norm_weight: torch.Tensor,
                             weight: torch.Tensor, eps: float = 1e-6):
    """``(rms_norm(x + residual) @ weight.T, x + residual)`` in 8 bits, with
    gradients (``RmsNormInt8LinearGPU``)."""
    return RmsNormInt8LinearGPU.apply(x, residual, norm_weight, weight, eps)


# ---------------------------------------------------------------------------
# Blocks in 8-bit floating point (no counterpart in the reference)
# ---------------------------------------------------------------------------

class Fp8LinearGPU(torch.autograd.Function):
    """``y = x @ weight.T`` with both operands rounded to e4m3 numbers, one power of
    two for each 1 x 128 activations and 128 x 128 weights.

    The backward pass reads the 8-bit operands, which are all that is kept of them:
    the gradients are those of the product of the rounded operands, passed through
    the rounding unchanged.  They have no gradients of their own: differentiating
    them is an error."""

    @staticmethod
    def forward(ctx, x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
        x, weight = _prep_int8("Fp8LinearGPU", x, weight)
        q, scale = fp8.quantize(x)
        qw, scale_w = fp8.quantize(weight, fp8.BLOCK)
        ctx.save_for_backward(q, scale, qw, scale_w)
        return fp8.matmul(q, scale, qw, scale_w, dtype=x.dtype)

    @staticmethod
    def backward(ctx, grad_y: torch.Tensor):
        q, scale, qw, scale_w = ctx.saved_tensors
        want_x, want_w = ctx.needs_input_grad
        with torch.no_grad():
            grad_y = grad_y.contiguous()
            grads = (fp8.backward_a(grad_y, qw, scale_w) if want_x else None,
                     fp8.backward_b(grad_y, q, scale) if want_w else None)
        return _first_derivatives("Fp8LinearGPU", *grads)


def _prep_rows(name: str, x: torch.Tensor, residual: torch.Tensor | None):
    if not x.is_cuda:
        raise RuntimeError(f"{name} requires GPU tensors.")
    return x.detach().contiguous(), None if residual is None else residual.detach().contiguous()


def _save_seed(ctx, seed, p: float, offset: int, *tensors):
    """Keeps what makes the mask; a seed on the GPU as a tensor, so that changing it
    before the backward pass is an error."""
    at = isinstance(seed, torch.Tensor)
    ctx.save_for_backward(*tensors, *((seed,) if at else ()))
    ctx.random = (p, None if at else seed, offset)


def _saved_seed(ctx):
    """(the other tensors, (p, seed, offset)) that _save_seed kept."""
    p, seed, offset = ctx.random
    saved = ctx.saved_tensors
    return (saved[:-1], (p, saved[-1], offset)) if seed is None else (saved, (p, seed, offset))


class DropoutGPU(torch.autograd.Function):
    """``dropout(x) + residual``; nothing is kept for the backward pass but the
    seed.  The gradients have no gradients of their own: differentiating them is
    an error."""

    @staticmethod
    def forward(ctx, x, residual, p: float, seed, offset: int) -> torch.Tensor:
        x, residual = _prep_rows("DropoutGPU", x, residual)
        _save_seed(ctx, seed, p, offset)
        return layers.dropout(x, p, seed, offset, residual)

    @staticmethod
    def backward(ctx, grad_y: torch.Tensor):
        want_x, want_r = ctx.needs_input_grad[:2]
        _, random = _saved_seed(ctx)
        with torch.no_grad():
            grad_x = layers.dropout(grad_y.contiguous(), *random) if want_x else None
        (grad_x,) = _first_derivatives("DropoutGPU", grad_x)
        return grad_x, grad_y if want_r else None, None, None, None


class LayerNormGPU(torch.autograd.Function):
    """``(y, h)`` of one step of a residual stream: ``h = dropout(x) + residual``,
    ``y = layer_norm(h, weight, bias, eps)``.

    Kept for the backward pass: h, its rows' statistics and the seed.  The gradients
    have no gradients of their own: differentiating them is an error."""

    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps: float, p: float, seed, offset: int):
        x, residual = _prep_rows("LayerNormGPU", x, residual)
        weight, bias = weight.detach().contiguous(), None if bias is None else bias.detach().contiguous()
        y, h, mean, rstd = layers.layer_norm(x, weight, bias, residual, eps, p, seed, offset)
        _save_seed(ctx, seed, p, offset, h, mean, rstd, weight)
        ctx.set_materialize_grads(False)
        # An output that shares no memory with an input.
        return y, x.clone() if h is x else h

    @staticmethod
    def backward(ctx, grad_y, grad_h):
        (h, mean, rstd, weight), (p, seed, offset) = _saved_seed(ctx)
        want_x, want_r, want_w, want_b = ctx.needs_input_grad[:4]
        with torch.no_grad():
            grad_h = None if grad_h is None else grad_h.contiguous()
            if grad_y is not None:
                grads = layers.layer_norm_backward(grad_y.contiguous(), h, mean, rstd, weight, grad_h, p, seed, offset)
            elif grad_h is not None:
                grads = layers.dropout(grad_h, p, seed, offset), grad_h, None, None
            else:
                grads = None, None, None, None
            grads = tuple(g if want else None for g, want in zip(grads, (want_x, want_r, want_w, want_b)))
        return *_first_derivatives("LayerNormGPU", *grads), None, None, None, None


def _seed_of(x: torch.Tensor, p: float, seed):
    """The seed, drawn by torch's generator of x's device where none is given (in a
    captured graph, each replay draws another)."""
    if seed is None and p > 0:
        return torch.randint(0, 2 ** 63 - 1, (1,), dtype=torch.int64, device=x.device)
    return 0 if seed is None else seed


def fp8_linear_gpu(x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    """``x @ weight.T`` in 8-bit floating point, with gradients (``Fp8LinearGPU``)."""
    return Fp8LinearGPU.apply(x, weight)


def dropout_gpu(x: torch.Tensor, p: float, residual: torch.Tensor | None = None, seed=None,
                offset: int = 0) -> torch.Tensor:
    """``dropout(x) + residual`` with gradients (``DropoutGPU``)."""
    return DropoutGPU.apply(x, residual, p, _seed_of(x, p, seed), offset)


def layer_norm_gpu(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
                   eps: float = 1e-5) -> torch.Tensor:
    """``layer_norm(x)`` with gradients (``LayerNormGPU``)."""
    return _LayerNormOnlyGPU.apply(x, weight, bias, eps)


def dropout_add_layer_norm_gpu(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor,
                               bias: torch.Tensor | None = None, p: float = 0.0, eps: float = 1e-5, seed=None,
                               offset: int = 0):
    """``(layer_norm(h), h)`` of ``h = dropout(x) + residual``, with gradients
    (``LayerNormGPU``)."""
    return LayerNormGPU.apply(x, residual, weight, bias, eps, p, _seed_of(x, p, seed), offset)


class _LayerNormOnlyGPU(torch.autograd.Function):
    """``LayerNormGPU`` where the stream is x itself: y alone."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps: float):
        x, _ = _prep_rows("LayerNormGPU", x, None)
        weight, bias = weight.detach().contiguous(), None if bias is None else bias.detach().contiguous()
        y, _, mean, rstd = layers.layer_norm(x, weight, bias, None, eps)
        ctx.save_for_backward(x, mean, rstd, weight)
        return y

    @staticmethod
    def backward(ctx, grad_y):
        with torch.no_grad():
            grad_x, _, grad_w, grad_b = layers.layer_norm_backward(grad_y.contiguous(), *ctx.saved_tensors)
            grads = tuple(g if want else None for g, want in zip((grad_x, grad_w, grad_b), ctx.needs_input_grad))
        return *_first_derivatives("LayerNormGPU", *grads), None


__all__ = [
    "TropicalMaxPlusMatmulGPU",
    "TropicalMinPlusMatmulGPU",
    "TropicalMaxMulMatmulGPU",
    "TropicalMaxPlusMatmulBatched",
    "TropicalMinPlusMatmulBatched",
    "TropicalMaxMulMatmulBatched",
    "tropical_maxplus_matmul_gpu",
    "tropical_minplus_matmul_gpu",
    "tropical_maxmul_matmul_gpu",
    "tropical_maxplus_matmul_batched",
    "tropical_minplus_matmul_batched",
    "tropical_maxmul_matmul_batched",
    "Int8LinearGPU",
    "RmsNormInt8LinearGPU",
    "int8_linear_gpu",
    "rms_norm_int8_linear_gpu",
    "Fp8LinearGPU",
    "DropoutGPU",
    "LayerNormGPU",
    "fp8_linear_gpu",
    "dropout_gpu",
    "layer_norm_gpu",
    "dropout_add_layer_norm_gpu",
    "GPU_AVAILABLE",
    "_DLPACK_AVAILABLE",
]
