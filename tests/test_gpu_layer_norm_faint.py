"""Layer norm of rows whose deviations' squares lie below f32, with eps zero or
smaller still: statistics and outputs are those of the definition, as they are for
the same rows times a power of two.

Tolerances as in test_gpu_layers.py; beside them a step of 2^-149, half of which the
mean's rounding may take where it lies below f32's normal numbers, and its share of
the deviations.
"""
import pytest
import torch

from tropical_gemm import layers

pytestmark = pytest.mark.gpu

DEV = "cuda"
E = 2.0 ** -24
U = {torch.float32: E, torch.bfloat16: 2.0 ** -8}
IDS = {torch.bfloat16: "bf16", torch.float32: "f32"}


def _gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=IDS.get)
@pytest.mark.parametrize("eps", [0.0, 1e-38, 1e-32, 2e-30])
@pytest.mark.parametrize("cols", [5, 64, 300, 1500, 3100, 9000])
def test_faint_rows(dtype, eps, cols):
    sizes = [1.0, 2.0 ** -40, 2.0 ** -48, 2.0 ** -52, 2.0 ** -63, 2.0 ** -70, 2.0 ** -80, 2.0 ** -100, 2.0 ** -118]
    x = torch.randn(len(sizes), cols, generator=_gen(cols)).double() * torch.tensor(sizes, dtype=torch.float64)[:, None]
    x[:, 0] += 3 * torch.tensor(sizes, dtype=torch.float64)
    x = x.to(dtype)
    w = (1 + 0.2 * torch.randn(cols, generator=_gen(5))).to(dtype)
    b = (0.3 * torch.randn(cols, generator=_gen(6))).to(dtype)
    y, h, mean, rstd = layers.layer_norm(x.to(DEV), w.to(DEV), b.to(DEV), None, eps)
    x64, w64, b64 = x.double(), w.double(), b.double()
    m = x64.mean(1, keepdim=True)
    # eps as f32 holds it: below its normal numbers it has fewer bits.
    e = torch.tensor(eps, dtype=torch.float32).double()
    s = ((x64 - m).square().mean(1, keepdim=True) + e).rsqrt()
    size = x64.abs().mean(1, keepdim=True)
    assert ((mean.cpu().double()[:, None] - m).abs() <= 300 * E * size + 2.0 ** -149).all()
    off_by = 1e-5 + (300 * E * size * s) ** 2
    assert ((rstd.cpu().double()[:, None] - s).abs() <= off_by * s).all()
    core = (x64 - m) * s * w64
    bound = (off_by + 1e-5) * core.abs() + (300 * E * size + 2.0 ** -149) * s * w64.abs() + 2 * E * b64.abs()
    d = (y.cpu().double() - core - b64).abs()
    assert (d <= bound + U[dtype] * ((core + b64).abs() + bound)).all()


@pytest.mark.parametrize("cols", [8, 300, 5003, 9001])
def test_scaled_rows_give_the_same(cols):
    """A power of two on a row's values leaves its output as it is where eps is zero,
    through the ways of faint, ordinary and huge rows, to the roundings of the mean."""
    x = torch.randn(6, cols, generator=_gen(cols))
    w = torch.ones(cols, device=DEV)
    want = layers.layer_norm(x.to(DEV), w, eps=0.0)
    for power in (-100, -60, -50, 50, 70, 100):
        y, _, mean, rstd = layers.layer_norm((x.double() * 2.0 ** power).float().to(DEV), w, eps=0.0)
        assert ((y - want[0]).abs() <= 2e-5 * (want[0].abs() + 1)).all(), power
        assert ((mean * 2.0 ** -power - want[2]).abs() <= 300 * E * 2).all(), power
        assert ((rstd * 2.0 ** power - want[3]).abs() <= 2e-5 * want[3]).all(), power


@pytest.mark.parametrize("eps", [1e-38, 1e-32])
def test_equal_rows(eps):
    """Rows of equal values have no deviations, whatever eps: the bias, to the bit.
    (Between 1e-10 and 1e25 what rounding leaves of the first mean's error may be more
    than such an eps in rstd; it has no part in the output.)"""
    values = [0.0, 1e-38, 1e-30, 1e-10, 0.001, 0.1, 77.7, 1e25, 3e38]
    for cols in (7, 64, 1000, 5003, 9000):
        x = torch.tensor(values)[:, None].expand(-1, cols).contiguous()
        w, b = torch.randn(2, cols, generator=_gen(cols)).to(DEV)
        y, _, mean, rstd = layers.layer_norm(x.to(DEV), w, b, None, eps)
        assert torch.equal(y, b.expand(len(values), -1)) and torch.equal(mean.cpu(), x[:, 0])
        root = torch.tensor(eps, dtype=torch.float32).double().sqrt().item()
        assert ((rstd[[0, 1, 2, 8]].double() * root - 1).abs() < 1e-5).all()


@pytest.mark.parametrize("cols", [5, 300, 3100, 9000])
def test_gradients_of_faint_rows(cols):
    """From the statistics that the forward pass gives, with eps zero."""
    sizes = torch.tensor([1.0, 2.0 ** -52, 2.0 ** -63, 2.0 ** -80, 2.0 ** -100], dtype=torch.float64)
    x = (torch.randn(5, cols, generator=_gen(cols)).double() * sizes[:, None]).float()
    w, g = 1 + 0.2 * torch.randn(cols, generator=_gen(5)), torch.randn(5, cols, generator=_gen(6))
    y, h, mean, rstd = layers.layer_norm(x.to(DEV), w.to(DEV), eps=0.0)
    gr, _, gw, gb = layers.layer_norm_backward(g.to(DEV), h, mean, rstd, w.to(DEV))
    m, s = mean.cpu().double()[:, None], rstd.cpu().double()[:, None]
    xh, u = (x.double() - m) * s, g.double() * w.double()
    want = s * (u - u.mean(1, keepdim=True) - xh * (u * xh).mean(1, keepdim=True))
    size = s * (u.abs() + u.abs().mean(1, keepdim=True) + xh.abs() * (u * xh).abs().mean(1, keepdim=True))
    assert ((gr.cpu().double() - want).abs() <= 2e-5 * size).all()
    assert ((gw.cpu().double() - (g.double() * xh).sum(0)).abs() <= 2e-5 * (g.double() * xh).abs().sum(0)).all()
    assert ((gb.cpu().double() - g.double().sum(0)).abs() <= 2e-5 * g.double().abs().sum(0)).all()
