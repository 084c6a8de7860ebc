"""The autograd functions of the layer in 8-bit floating point, of layer norm and
dropout, by themselves and joined to a block: gradients against torch's own, in 64
bits, of the same function with the same rounded operands and masks."""
import importlib.util
import os

import pytest
import torch

from tropical_gemm import fp8, layers
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


def _mask(rows, cols, p, seed, offset=0):
    """Dropout's factors, from the operator itself (tested against its definition elsewhere)."""
    return layers.dropout(torch.ones(rows, cols, device=DEV), p, seed, offset).cpu().double()


def _rounded(t, br=1):
    return fp8.dequantize(*fp8.quantize(t.detach().to(DEV), br), torch.float32).cpu().double()


@pytest.mark.parametrize("m,n,k", [(1, 5, 7), (70, 130, 257), (300, 256, 512)])
def test_linear_f32(m, n, k):
    """Sums of at most 512 terms in f32: their 2-norms are off by less than
    512 * 2^-23 / 30 of the result, 2e-6."""
    x, w = _randn(1, m, k).to(DEV).requires_grad_(), _randn(2, n, k).to(DEV).requires_grad_()
    g = _randn(3, m, n).to(DEV)
    y = tgt.fp8_linear_gpu(x, w)
    y.backward(g)
    xr, wr = _rounded(x), _rounded(w, 128)
    assert _rel(y.detach(), xr @ wr.t()) < 2e-6
    assert _rel(x.grad, g.cpu().double() @ wr) < 2e-6
    assert _rel(w.grad, g.cpu().double().t() @ xr) < 2e-6


@pytest.mark.parametrize("seed", [5, None, "tensor"])
@pytest.mark.parametrize("residual", [False, True])
def test_dropout(residual, seed):
    if seed == "tensor":
        seed = torch.tensor([9], device=DEV)
    x, r = _randn(1, 40, 100).to(DEV).requires_grad_(), _randn(2, 40, 100).to(DEV).requires_grad_()
    g = _randn(3, 40, 100).to(DEV)
    y = tgt.dropout_gpu(x, 0.4, r if residual else None, seed)
    y.backward(g)
    f = (y.detach() - (r.detach() if residual else 0)) / x.detach()
    kept = f.abs() > 0.5
    assert torch.equal(x.grad != 0, kept)
    assert ((x.grad - g / 0.6)[kept].abs() <= 1e-4 * g.abs()[kept]).all()
    assert not residual or torch.equal(r.grad, g)
    if seed is None:
        assert not torch.equal(tgt.dropout_gpu(x, 0.4), tgt.dropout_gpu(x, 0.4))


@pytest.mark.parametrize("residual,p,bias", [(False, 0.0, True), (True, 0.0, False), (True, 0.3, True), (False, 0.3, True)])
def test_layer_norm_f32(residual, p, bias):
    m, k = 33, 300
    leaves = [_randn(1, m, k), _randn(2, m, k) if residual else None, 1 + 0.1 * _randn(3, k), _randn(4, k) if bias else None]
    gy, gh = _randn(5, m, k), _randn(6, m, k)
    ours = [t if t is None else t.to(DEV).requires_grad_() for t in leaves]
    y, h = tgt.dropout_add_layer_norm_gpu(*ours, p, 1e-5, 17, 3)
    torch.autograd.backward([y, h], [gy.to(DEV), gh.to(DEV)])
    ref = [t if t is None else t.double().requires_grad_() for t in leaves]
    h64 = ref[0] * (_mask(m, k, p, 17, 3) if p else 1) + (ref[1] if residual else 0)
    y64 = torch.nn.functional.layer_norm(h64, (k,), ref[2], ref[3], 1e-5)
    torch.autograd.backward([y64, h64], [gy.double(), gh.double()])
    assert _rel(y.detach(), y64.detach()) < 2e-6 and _rel(h.detach(), h64.detach()) < 2e-7
    for a, b in zip(ours, ref):
        assert a is None or _rel(a.grad, b.grad) < 1e-5
    # One output's gradient alone.
    for which in (0, 1):
        for t in (*ours, *ref):
            if t is not None:
                t.grad = None
        tgt.dropout_add_layer_norm_gpu(*ours, p, 1e-5, 17, 3)[which].backward((gy, gh)[which].to(DEV))
        h64 = ref[0] * (_mask(m, k, p, 17, 3) if p else 1) + (ref[1] if residual else 0)
        (torch.nn.functional.layer_norm(h64, (k,), ref[2], ref[3], 1e-5), h64)[which].backward((gy, gh)[which].double())
        for a, b in zip(ours, ref):
            if a is not None:
                assert (a.grad is None) == (b.grad is None) and (a.grad is None or _rel(a.grad, b.grad) < 1e-5)


def test_plain_layer_norm():
    x, w, b = (t.to(DEV).requires_grad_() for t in (_randn(1, 20, 130), _randn(2, 130), _randn(3, 130)))
    g = _randn(4, 20, 130)
    y = tgt.layer_norm_gpu(x, w, b)
    y.backward(g.to(DEV))
    ref = [t.detach().cpu().double().requires_grad_() for t in (x, w, b)]
    y64 = torch.nn.functional.layer_norm(ref[0], (130,), ref[1], ref[2], 1e-5)
    y64.backward(g.double())
    assert _rel(y.detach(), y64.detach()) < 2e-6
    for a, c in zip((x, w, b), ref):
        assert _rel(a.grad, c.grad) < 1e-5


@pytest.mark.parametrize("make", ["linear", "dropout", "norm", "stream"])
def test_second_derivatives_refuse(make):
    x, w = _randn(1, 8, 16).to(DEV).requires_grad_(), _randn(2, 16, 16).to(DEV).requires_grad_()
    v = torch.ones(16, device=DEV).requires_grad_()
    y = {"linear": lambda: tgt.fp8_linear_gpu(x, w), "dropout": lambda: tgt.dropout_gpu(x, 0.5, None, 1),
         "norm": lambda: tgt.layer_norm_gpu(x, v), "stream": lambda: tgt.dropout_add_layer_norm_gpu(x, x, v)[0]}[make]()
    (gx,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        gx.sum().backward()


def test_changed_seed_is_refused():
    seed = torch.tensor([4], device=DEV)
    x = _randn(1, 8, 16).to(DEV).requires_grad_()
    y = tgt.dropout_gpu(x, 0.5, None, seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def _block(x, p, drop, seed):
    y, h = tgt.dropout_add_layer_norm_gpu(x, None, p[0], p[1], 0.0)
    u = torch.tanh(tgt.fp8_linear_gpu(y, p[2]))
    branch = tgt.fp8_linear_gpu(u, p[3])
    z, h = tgt.dropout_add_layer_norm_gpu(branch, h, p[4], None, drop, seed=seed)
    return tgt.dropout_gpu(z, drop, h, seed, 1)


def test_block_gradients_f32():
    """A run of all operators together: every gradient against torch's, the
    rounding to 8 bits passed through, at the values that our own pass rounds
    to.  Each function's gradients are off by less than 1e-5; five of them follow
    one another."""
    m, k, n, drop, seed = 150, 256, 384, 0.2, 31
    leaves = [_randn(1, m, k), 1 + 0.1 * _randn(2, k), 0.1 * _randn(3, k), _randn(4, n, k) / 16, _randn(5, k, n) / 16,
              1 + 0.1 * _randn(6, k)]
    g = _randn(7, m, k)
    ours = [t.to(DEV).requires_grad_() for t in leaves]
    out = _block(ours[0], ours[1:], drop, seed)
    out.backward(g.to(DEV))

    ref = [t.double().requires_grad_() for t in leaves]
    with torch.no_grad():
        y = layers.layer_norm(ours[0], ours[1], ours[2])[0]
        u = torch.tanh(fp8.matmul(*fp8.quantize(y), *fp8.quantize(ours[3], 128), dtype=torch.float32))

    def linear(x64, w64, x, w):  # the product at the rounded operands, gradients passed through
        return (x64 + (_rounded(x) - x64).detach()) @ (w64 + (_rounded(w, 128) - w64).detach()).t()

    y64 = torch.nn.functional.layer_norm(ref[0], (k,), ref[1], ref[2], 1e-5)
    u64 = torch.tanh(linear(y64, ref[3], y, ours[3]))
    b64 = linear(u64, ref[4], u, ours[4])
    h64 = b64 * _mask(m, k, drop, seed) + ref[0]
    z64 = torch.nn.functional.layer_norm(h64, (k,), ref[5], None, 1e-5)
    o64 = z64 * _mask(m, k, drop, seed, 1) + h64
    o64.backward(g.double())
    assert _rel(out.detach(), o64.detach()) < 1e-5
    for a, b in zip(ours, ref):
        assert _rel(a.grad, b.grad) < 5e-5


def test_example():
    """The example runs: finite losses, and a token served alone answers as in the
    prompt, to what bf16 and the roundings to 8 bits make of another order of sums."""
    spec = importlib.util.spec_from_file_location("fp8_block", os.path.join(ROOT, "examples", "fp8_block.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    losses, apart = mod.run(width=256, hidden=512, tokens=200, steps=4, verbose=False)
    assert len(losses) == 4 and all(v == v and abs(v) < 1e6 for v in losses)
    assert apart < 0.5
