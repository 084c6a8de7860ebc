"""The mean that layer norm gives of a row, against sums of whole numbers.

Rows of whole numbers below 2^8, in any type, and of those times 2^100 (whose
squares pass f32), have sums that f32 holds exactly in any order: 2^8 * cols is
below 2^24.  Their mean is the sum times 1 / cols.  Where cols is a power of two
that is exact, and the mean has to be equal to the last bit; else 1 / cols and the
product are rounded once each, 2^-24 of the mean twice.

Rows whose mean is far above their deviations are wide numbers: the mean is rounded
once (2^-24 of it); before that the deviations are rounded, added up in a thread (at
most 24 in a row, 2 * 8 * 2 of them), over 64 lanes and 16 waves, 48 roundings of
at most 2^-24 of the magnitudes' sum.
"""
import pytest
import torch

from tropical_gemm import layers

pytestmark = pytest.mark.gpu

DEV = "cuda"
E = 2.0 ** -24
TYPES = [torch.bfloat16, torch.float16, torch.float32]
IDS = {torch.bfloat16: "bf16", torch.float16: "f16", torch.float32: "f32"}
ROWS = 60


def _whole(seed, rows, cols, most=64):
    g = torch.Generator()
    g.manual_seed(seed)
    return torch.randint(-most, most + 1, (rows, cols), generator=g)


def _check(mean, h, scale=1.0):
    """mean of the rows of whole numbers h, times scale."""
    cols = h.shape[1]
    sums, h64 = h.sum(1).double(), h.double()
    assert h.abs().max() <= 256 and (sums.abs() / cols < h64.std(1) / 2).all()
    got, want = mean.cpu().double(), sums / cols * scale
    if cols & (cols - 1) == 0:
        assert torch.equal(got, want)
    else:
        assert ((got - want).abs() <= 2.001 * E * want.abs()).all()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("cols", [512, 1024, 2048, 4096, 8192, 16384, 1031, 2501, 4099, 5003, 9001])
def test_whole_numbers(dtype, cols):
    x, r = _whole(cols, ROWS, cols), _whole(cols + 1, ROWS, cols)
    w = torch.ones(cols, dtype=dtype, device=DEV)
    xd, rd = x.to(dtype).to(DEV), r.to(dtype).to(DEV)
    _check(layers.layer_norm(xd, w)[2], x)
    _check(layers.layer_norm(xd, w, w, rd)[2], x + r)
    # Half are dropped, the others doubled: whole numbers again.
    for res in (None, rd):
        _, h, mean, _ = layers.layer_norm(xd, w, None, res, 1e-5, 0.5, 3, cols)
        _check(mean, h.cpu().double().long())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=IDS.get)
@pytest.mark.parametrize("cols", [512, 2048, 8192, 16384, 1031, 5003, 9001])
def test_whole_numbers_whose_squares_pass_f32(dtype, cols):
    x = _whole(cols, ROWS, cols)
    w = torch.ones(cols, dtype=dtype, device=DEV)
    _, h, mean, rstd = layers.layer_norm((x.double() * 2.0 ** 100).to(dtype).to(DEV), w)
    _check(mean, x, 2.0 ** 100)
    dev = x.double().std(1, correction=0) * 2.0 ** 100
    assert ((rstd.cpu().double() * dev - 1).abs() < 1e-5).all()


@pytest.mark.parametrize("cols", [512, 2048, 4096, 8192, 1031, 5003, 9001])
def test_mean_above_the_deviations(cols):
    """What rounding took from the first sum is given back."""
    g = torch.Generator()
    g.manual_seed(cols)
    x = torch.randn(400, cols, generator=g) + 1000
    mean = layers.layer_norm(x.to(DEV), torch.ones(cols, device=DEV))[2]
    want = x.double().mean(1)
    apart = (x.double() - want[:, None]).abs().mean(1)
    assert ((mean.cpu().double() - want).abs() <= E * (want + 48 * apart)).all()
