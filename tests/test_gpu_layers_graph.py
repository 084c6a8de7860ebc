"""The autograd functions of the 8-bit floating point layer, layer norm and dropout
in 16 bits, and captured into graphs: gradients element by element against 64 bits,
replays against eager calls, and masks drawn anew by each replay.

Tolerances, with u the unit roundoff of the type (2^-11, 2^-8): those of
test_gpu_fp8.py for products (f32 sums of r exact products: 3 * r * 2^-23 of the
magnitudes' sum S; 2^-10 S more for 16-bit outputs) and of test_gpu_layers.py for
the norm (2e-5 of the sum of the magnitudes), then u.
"""
import pytest
import torch

from tropical_gemm import fp8, layers
from tropical_gemm import pytorch as tgt

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}
HALF = [torch.bfloat16, torch.float16]
IDS = {torch.bfloat16: "bf16", torch.float16: "f16", torch.float32: "f32"}


def _randn(seed, *shape):
    g = torch.Generator()
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g)


def _leaf(seed, dtype, *shape, size=1.0, plus=0.0):
    return (plus + size * _randn(seed, *shape)).to(dtype).to(DEV).requires_grad_()


def _within(got, want, bound, dtype):
    assert got.dtype is dtype and got.shape == want.shape
    d = (got.detach().cpu().double() - want).abs()
    most = bound + U[dtype] * (want.abs() + bound) + LEAST[dtype]
    assert (d <= most).all(), (d - most).max()


def _rounded(t, br=1):
    return fp8.dequantize(*fp8.quantize(t.detach(), br), torch.float32).cpu().double()


@pytest.mark.parametrize("dtype", HALF, ids=IDS.get)
@pytest.mark.parametrize("m,n,k", [(1, 5, 7), (70, 130, 257), (300, 256, 512)])
def test_linear(dtype, m, n, k):
    x, w, g = _leaf(1, dtype, m, k), _leaf(2, dtype, n, k), _randn(3, m, n).to(dtype)
    y = tgt.fp8_linear_gpu(x, w)
    y.backward(g.to(DEV))
    xr, wr, g64 = _rounded(x), _rounded(w, 128), g.double()
    _within(y, xr @ wr.t(), ((k + 1) * 2.0 ** -23 + 2.0 ** -10) * (xr.abs() @ wr.abs().t()), dtype)
    _within(x.grad, g64 @ wr, 3 * n * 2.0 ** -23 * (g64.abs() @ wr.abs()), dtype)
    _within(w.grad, g64.t() @ xr, 3 * m * 2.0 ** -23 * (g64.t().abs() @ xr.abs()), dtype)


@pytest.mark.parametrize("dtype", HALF, ids=IDS.get)
@pytest.mark.parametrize("residual", [False, True])
def test_dropout(dtype, residual):
    x, r, g = _leaf(1, dtype, 40, 100), _leaf(2, dtype, 40, 100), _randn(3, 40, 100).to(dtype)
    y = tgt.dropout_gpu(x, 0.25, r if residual else None, 7, 3)
    y.backward(g.to(DEV))
    f = layers.dropout(torch.ones(40, 100, device=DEV), 0.25, 7, 3).cpu().double()
    want = x.detach().cpu().double() * f
    extra = r.detach().cpu().double() if residual else 0 * want
    _within(y, want + extra, 2.0 ** -23 * (want.abs() + extra.abs()), dtype)
    _within(x.grad, g.double() * f, 2.0 ** -23 * g.double().abs(), dtype)
    assert not residual or torch.equal(r.grad.cpu(), g)


@pytest.mark.parametrize("dtype", HALF, ids=IDS.get)
@pytest.mark.parametrize("residual,p,bias", [(False, 0.0, True), (True, 0.0, False), (True, 0.3, True), (False, 0.3, True)])
def test_layer_norm(dtype, residual, p, bias):
    m, k = 33, 300
    x, r = _leaf(1, dtype, m, k), _leaf(2, dtype, m, k) if residual else None
    w, b = _leaf(3, dtype, k, size=0.1, plus=1.0), _leaf(4, dtype, k) if bias else None
    gy, gh = _randn(5, m, k).to(dtype), _randn(6, m, k).to(dtype)
    y, h = tgt.dropout_add_layer_norm_gpu(x, r, w, b, p, 1e-5, 17, 3)
    torch.autograd.backward([y, h], [gy.to(DEV), gh.to(DEV)])
    f = layers.dropout(torch.ones(m, k, device=DEV), p, 17, 3).cpu().double() if p else torch.ones(m, k).double()
    want_h = x.detach().cpu().double() * f + (r.detach().cpu().double() if residual else 0)
    _within(h, want_h, 2.0 ** -22 * (want_h.abs() + 4), dtype)
    # Gradients at the stream as it is stored.
    h64, w64, g64 = h.detach().cpu().double(), w.detach().cpu().double(), gy.double()
    mean = h64.mean(1, keepdim=True)
    rstd = ((h64 - mean).square().mean(1, keepdim=True) + 1e-5).rsqrt()
    xh, u = (h64 - mean) * rstd, g64 * w64
    b64 = b.detach().cpu().double() if bias else 0 * w64
    _within(y, xh * w64 + b64, 4e-5 * (xh.abs() + 1) * w64.abs() + 2.0 ** -23 * b64.abs(), dtype)
    inner = u - u.mean(1, keepdim=True) - xh * (u * xh).mean(1, keepdim=True)
    size = rstd * (u.abs() + u.abs().mean(1, keepdim=True) + xh.abs() * (u * xh).abs().mean(1, keepdim=True)) + gh.double().abs()
    want = rstd * inner + gh.double()
    _within(x.grad, want * f, 4e-5 * size * f, dtype)
    if residual:
        _within(r.grad, want, 4e-5 * size, dtype)
    _within(w.grad, (g64 * xh).sum(0), 4e-5 * (g64 * xh).abs().sum(0), dtype)
    if bias:
        _within(b.grad, g64.sum(0), 4e-5 * g64.abs().sum(0), dtype)


def _leaves(dtype, m, k, n):
    return [_leaf(1, dtype, m, k), _leaf(2, dtype, k, size=0.1, plus=1.0), _leaf(3, dtype, k, size=0.1),
            _leaf(4, dtype, n, k, size=0.1), _leaf(5, dtype, k, n, size=0.1), _leaf(6, dtype, k, size=0.1, plus=1.0)]


def _step(p, grad, seed):
    """A block's forward and backward pass: its output and all its gradients."""
    y = tgt.layer_norm_gpu(p[0], p[1], p[2])
    branch = tgt.fp8_linear_gpu(torch.tanh(tgt.fp8_linear_gpu(y, p[3])), p[4])
    z, h = tgt.dropout_add_layer_norm_gpu(branch, p[0], p[5], None, 0.2, seed=seed)
    out = tgt.dropout_gpu(z, 0.1, h, seed, 1)
    return [out.detach(), *torch.autograd.grad(out, p, grad)]


@pytest.mark.parametrize("dtype", [*HALF, torch.float32], ids=IDS.get)
@pytest.mark.parametrize("m,k,n", [(40, 64, 96), (300, 256, 520)])
def test_captured_step(dtype, m, k, n):
    """Replays with other inputs and seeds give the bits of an eager step on leaves of
    its own, with eager work between them."""
    p = _leaves(dtype, m, k, n)
    grad = _randn(9, m, k).to(dtype).to(DEV)
    seed = torch.tensor([1], dtype=torch.int64, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(p, grad, seed)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(p, grad, seed)
    for turn in range(4):
        with torch.no_grad():
            p[0].copy_(_randn(20 + turn, m, k).to(dtype))
            grad.copy_(_randn(30 + turn, m, k).to(dtype))
            seed.fill_(100 + turn)
        want = _step([t.detach().clone().requires_grad_() for t in p], grad, seed.clone())
        graph.replay()
        torch.cuda.synchronize()
        assert len(out) == len(want) and all(torch.equal(a, b) for a, b in zip(out, want)), turn


@pytest.mark.parametrize("which", ["dropout", "norm"])
def test_replays_draw_other_masks(which):
    """Without a seed each call draws one; captured, each replay draws another, the
    same in its forward and its backward pass."""
    m, k, p = 64, 512, 0.3
    x, w = torch.ones(m, k, device=DEV).requires_grad_(), torch.ones(k, device=DEV).requires_grad_()
    one = torch.ones(m, k, device=DEV)

    def run():
        if which == "dropout":
            y = tgt.dropout_gpu(x, p)
            return y.detach(), torch.autograd.grad(y, x, one)[0]
        h = tgt.dropout_add_layer_norm_gpu(x, None, w, None, p)[1]
        return h.detach(), torch.autograd.grad(h, x, one)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, gx = run()
    masks = []
    for turn in range(4):
        eager = run()[0] != 0
        graph.replay()
        torch.cuda.synchronize()
        masks += [(y != 0).clone(), eager]
        assert torch.equal(y, gx)  # x and its gradient are ones
        # The share's deviation over n elements is sqrt(p (1 - p) / n): six of it, and p's rounding.
        assert abs((y == 0).float().mean().item() - p) < 6 * (p * (1 - p) / (m * k)) ** 0.5 + 2.0 ** -16
    assert all(not torch.equal(masks[i], masks[j]) for i in range(8) for j in range(i))
