"""The 8-bit layer's autograd functions: gradients against torch's own for the
same rounded operands, and the example that trains and serves a block."""
import importlib.util
import os

import pytest
import torch

from tropical_gemm import int8
from tropical_gemm import pytorch as tgt

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda"


def _randn(seed, *shape):
    g = torch.Generator()
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g)


def _rel(a, b):
    return ((a.cpu().double() - b).norm() / b.norm()).item()


@pytest.mark.parametrize("m,n,k", [(1, 5, 7), (70, 130, 257), (300, 256, 512)])
def test_linear_f32(m, n, k):
    """In f32 the gradients are those of the rounded operands' product to 2e-6,
    the forward pass to two f32 roundings."""
    x, w = _randn(1, m, k).to(DEV).requires_grad_(), _randn(2, n, k).to(DEV).requires_grad_()
    g = _randn(3, m, n).to(DEV)
    y = tgt.int8_linear_gpu(x, w)
    y.backward(g)
    xr, wr = (int8.dequantize(*int8.quantize(t.detach()), torch.float32).cpu().double() for t in (x, w))
    assert _rel(y.detach(), xr @ wr.t()) < 1e-6
    assert _rel(x.grad, g.cpu().double() @ wr) < 2e-6
    assert _rel(w.grad, g.cpu().double().t() @ xr) < 2e-6


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("m,n,k", [(3, 40, 64), (130, 96, 300)])
def test_norm_linear_f32(m, n, k, residual):
    """Every gradient against torch's, in 64 bits, of the same function with the
    rounding passed through: y = (norm(h) + (rows - norm(h))) @ w."""
    x, nw = _randn(1, m, k), 1 + 0.1 * _randn(2, k)
    r, w = _randn(3, m, k) if residual else None, _randn(4, n, k)
    gy, gh = _randn(5, m, n), _randn(6, m, k)

    ours = [t.to(DEV).requires_grad_() if t is not None else None for t in (x, r, nw, w)]
    y, h = tgt.rms_norm_int8_linear_gpu(*ours, 1e-5)
    torch.autograd.backward([y, h], [gy.to(DEV), gh.to(DEV)])

    ref = [t.double().requires_grad_() if t is not None else None for t in (x, r, nw, w)]
    h64 = ref[0] if r is None else ref[0] + ref[1]
    norm = h64 * (h64.square().mean(1, keepdim=True) + 1e-5).rsqrt() * ref[2]
    q, s, _ = int8.rms_norm(x.to(DEV), nw.to(DEV), None if r is None else r.to(DEV), 1e-5)
    rows = int8.dequantize(q, s, torch.float32).cpu().double()
    wr = int8.dequantize(*int8.quantize(w.to(DEV)), torch.float32).cpu().double()
    y64 = (norm + (rows - norm).detach()) @ (ref[3] + (wr - ref[3]).detach()).t()
    torch.autograd.backward([y64, h64 * 1.0], [gy.double(), gh.double()])
    assert _rel(y.detach(), y64.detach()) < 1e-6 and _rel(h.detach(), h64.detach()) < 1e-6
    for a, b in zip(ours, ref):
        if a is not None:
            assert _rel(a.grad, b.grad) < 1e-5


def test_expanded_gradient_and_frozen_inputs():
    """A gradient whose rows are one row in memory, and inputs without one."""
    x, w = _randn(1, 20, 33).to(DEV).requires_grad_(), _randn(2, 12, 33).to(DEV)
    tgt.int8_linear_gpu(x, w).sum().backward()
    wr = int8.dequantize(*int8.quantize(w), torch.float32).cpu().double()
    assert _rel(x.grad, torch.ones(20, 12, dtype=torch.float64) @ wr) < 2e-6 and w.grad is None
    nw = torch.ones(33, device=DEV)
    w.requires_grad_()
    y, h = tgt.rms_norm_int8_linear_gpu(x.detach(), None, nw, w)
    y.sum().backward()
    assert w.grad is not None and nw.grad is None
    x.grad = None
    y, h = tgt.rms_norm_int8_linear_gpu(x, None, nw, w.detach())
    h.sum().backward()
    assert torch.equal(x.grad, torch.ones_like(x))


def test_refusals():
    x, w = torch.zeros(4, 8, device=DEV), torch.zeros(3, 8, device=DEV)
    with pytest.raises(RuntimeError, match="requires GPU tensors"):
        tgt.int8_linear_gpu(x.cpu(), w)
    with pytest.raises(RuntimeError, match="expects activations"):
        tgt.int8_linear_gpu(x, w[:, :7])
    with pytest.raises(RuntimeError, match="one dtype"):
        tgt.rms_norm_int8_linear_gpu(x, None, w[0], w.half())


def test_example_trains_and_serves():
    spec = importlib.util.spec_from_file_location("int8_block", os.path.join(ROOT, "examples", "int8_block.py"))
    block = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(block)
    losses, apart = block.run(width=256, hidden=512, tokens=512, steps=30, verbose=False)
    assert losses[-1] < 0.9 * losses[0]
    # The kernels of one token and of many give the same sums and roundings.
    assert apart == 0.0
