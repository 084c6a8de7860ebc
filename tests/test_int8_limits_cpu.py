"""The 8-bit layer's autograd functions with plain host operators in place of the
kernels, and choices of a way at the limits of launches: no GPU needed."""
import pytest

torch = pytest.importorskip("torch")

from tropical_gemm import _native as nat  # noqa: E402
from tropical_gemm import int8  # noqa: E402
from tropical_gemm import pytorch as tgt  # noqa: E402


@pytest.fixture
def on_host(monkeypatch):
    """The int8 operators on the CPU, in 64 bits and without rounding to 8."""
    one = lambda t: torch.ones(t.shape[0], dtype=t.dtype)  # noqa: E731

    def rms_norm(x, weight, residual=None, eps=1e-6):
        h = x if residual is None else x + residual
        y = h * (h.square().mean(1, keepdim=True) + eps).rsqrt() * weight
        return y, one(y), h

    def rms_norm_backward(grad_y, h, weight, eps=1e-6, grad_h=None):
        rstd = (h.square().mean(1, keepdim=True) + eps).rsqrt()
        xh, u = h * rstd, grad_y * weight
        gx = rstd * (u - xh * (u * xh).mean(1, keepdim=True))
        return (gx if grad_h is None else gx + grad_h), (grad_y * xh).sum(0)

    for name, f in {"quantize": lambda x: (x.clone(), one(x)), "rms_norm": rms_norm,
                    "rms_norm_backward": rms_norm_backward,
                    "matmul": lambda a, sa, b, sb, bias=None, dtype=None: a @ b.t(),
                    "backward_a": lambda g, b, sb: g @ b, "backward_b": lambda g, a, sa: g.t() @ a}.items():
        monkeypatch.setattr(int8, name, f)
    monkeypatch.setattr(tgt, "_prep_int8", lambda name, x, weight: (x.detach(), weight.detach()))


def _randn(seed, *shape):
    g = torch.Generator()
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g, dtype=torch.float64)


def _layers():
    """(call, inputs) of both functions; the norm's with and without a residual."""
    x, r, w, nw = _randn(1, 5, 6), _randn(2, 5, 6), _randn(3, 4, 6), _randn(4, 6)
    leaf = lambda t: t.clone().requires_grad_()  # noqa: E731
    return [(lambda a, b: tgt.int8_linear_gpu(a, b), [leaf(x), leaf(w)]),
            (lambda a, n, b: tgt.rms_norm_int8_linear_gpu(a, None, n, b)[0], [leaf(x), leaf(nw), leaf(w)]),
            (lambda a, c, n, b: tgt.rms_norm_int8_linear_gpu(a, c, n, b)[0], [leaf(x), leaf(r), leaf(nw), leaf(w)])]


@pytest.mark.parametrize("i", range(3))
def test_second_derivatives_are_refused(on_host, i):
    """A loss that holds a gradient (a gradient penalty) is an error, not the loss
    without it; whichever input's gradient it is."""
    call, inputs = _layers()[i]
    for t in inputs:
        y = call(*inputs)
        grad, = torch.autograd.grad(y.square().sum(), t, create_graph=True)
        assert grad.requires_grad
        with pytest.raises(RuntimeError, match="no second derivatives"):
            (y.sum() + grad.square().sum()).backward()
        # Ones as the incoming gradient, which need none themselves.
        grad, = torch.autograd.grad(call(*inputs).sum(), t, create_graph=True)
        with pytest.raises(RuntimeError, match="no second derivatives"):
            grad.square().sum().backward()


@pytest.mark.parametrize("i", range(3))
def test_first_derivatives_with_a_graph(on_host, i):
    """create_graph changes no gradient, and without it nothing is recorded."""
    call, inputs = _layers()[i]
    plain = torch.autograd.grad(call(*inputs).square().sum(), inputs)
    graph = torch.autograd.grad(call(*inputs).square().sum(), inputs, create_graph=True)
    for a, b in zip(plain, graph):
        assert not a.requires_grad and torch.equal(a, b.detach())
    assert torch.autograd.gradcheck(call, inputs)


def test_gradient_of_the_stream_alone(on_host):
    """Only h is used: its gradient passes through, and on to a second derivative,
    which is that of the loss."""
    x, r = _randn(1, 5, 6).requires_grad_(), _randn(2, 5, 6).requires_grad_()
    h = tgt.rms_norm_int8_linear_gpu(x, r, torch.ones(6, dtype=torch.float64), _randn(3, 4, 6))[1]
    grads = torch.autograd.grad((h ** 3).sum(), (x, r), create_graph=True)
    second, = torch.autograd.grad(grads[0].sum(), x)
    assert torch.allclose(grads[1], 3 * (x + r) ** 2) and torch.allclose(second, 6 * (x + r))


@pytest.mark.parametrize("m,k", [(1, 16), (16, 16), (16, 17), (32, 17), (64, 17)])
def test_products_of_few_rows_launch_fewer_than_2_to_the_32_threads(m, k):
    """Sixteen columns take up to 1024 threads: 2^26 - 16 columns are the most."""
    lib = nat.load()
    most = (1 << 26) - 16
    plan = lambda n: lib.tg_i8_gemm_plan(4096, k, 4096, k, m, n, k).decode()  # noqa: E731
    if m <= 16:
        assert plan(most).startswith("stream")
    for n in (most + 1, most + 15, 1 << 26):
        assert not plan(n).startswith("stream") and plan(n) != "invalid"
