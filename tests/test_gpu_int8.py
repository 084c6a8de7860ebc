"""The 8-bit layer's operators against their definitions in 64 bits.

Tolerances, with u the unit roundoff of the output's type (2^-24, 2^-11, 2^-8
for f32, f16, bf16) and e = 2^-24:

* 8-bit rows: within half a step of the exact value, plus 127 * 4e of a step
  for the f32 product with 127 / top; a scale within 1e-5 (sums of fewer than
  160 f32 terms in a row, whose error the square root halves) or, without a
  norm, 2e.
* matmul: the integer sum is exact; its conversion, the two scales and the bias
  are four roundings of at most e of the largest of them, then one of u.
* norm backward: 2e-5 of the sum of the magnitudes added (sums of fewer than
  256 f32 terms in a row), then u.
* gradients of the product: each dequantized operand may be rounded to the
  gradient's type (u of every term; f32: 2e), the sum of r terms in f32 is off
  by less than r * e of the magnitudes, then u.  Their 2-norms are closer, as
  the roundings are independent: sqrt(2) u / sqrt(3) at most 0.9 u, with 1.2 u
  taken; f32: 2e-6.
"""
import numpy as np
import pytest
import torch

from tropical_gemm import _native as nat
from tropical_gemm import int8

pytestmark = pytest.mark.gpu

DEV = "cuda"
E = 2.0 ** -24
U = {torch.float32: E, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}
TYPES = [torch.bfloat16, torch.float16, torch.float32]
IDS = {torch.bfloat16: "bf16", torch.float16: "f16", torch.float32: "f32"}


def _say(*what):
    print("[case]", *what, flush=True)


def _gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def _values(seed, rows, cols, dtype, ld=None, offset=0):
    """A rows x cols matrix on the GPU whose rows are ld apart, `offset`
    elements into its storage."""
    ld = cols if ld is None else ld
    g = _gen(seed)
    store = torch.zeros(offset + max(rows, 1) * ld + 8, dtype=dtype, device=DEV)
    v = store[offset:].as_strided((rows, cols), (ld, 1))
    v.copy_((torch.randn(rows, cols, generator=g) * torch.exp(torch.randn(rows, 1, generator=g))).to(dtype))
    return v


def _int8(seed, rows, cols, ld=None, offset=0, full=False):
    ld = cols if ld is None else ld
    g = _gen(seed)
    store = torch.full((offset + max(rows, 1) * ld + 16,), 77, dtype=torch.int8, device=DEV)
    v = store[offset:].as_strided((rows, cols), (ld, 1))
    v.copy_(torch.randint(-128 if full else -127, 128, (rows, cols), generator=g).to(torch.int8))
    return v, (torch.rand(rows, generator=g) * 0.02 + 1e-3).to(DEV)


def _check_rows(q, scale, want):
    """q and scale against the exact values `want` (f64, on the CPU)."""
    top = want.abs().amax(1) if want.shape[1] else torch.zeros(want.shape[0], dtype=torch.float64)
    top = torch.clamp(top, min=1e-30)
    step = (top / 127)[:, None]
    q64 = q.cpu().double()
    assert q.dtype == torch.int8 and int(q.cpu().int().abs().max() if q.numel() else 0) <= 127
    assert ((q64 * step - want).abs() <= step * (0.5 + 127 * 4 * E + 1e-9)).all()
    live = top > 1e-29
    assert ((scale.cpu().double() - top / 127).abs() <= 1e-5 * top / 127)[live].all()
    assert (q64[~live] == 0).all()


COLS = [1, 7, 8, 9, 64, 511, 512, 513, 1024, 1025, 2048, 2051, 2501, 3081, 4096, 5003, 6145, 8185, 8192, 8200, 40001]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("cols", COLS)
def test_quantize_and_dequantize(dtype, cols):
    rows = 37 if cols < 8192 else 5
    for ld, offset in ((cols, 0), (cols + 3, 1)):
        _say("quantize", IDS[dtype], rows, cols, ld, offset)
        x = _values(cols, rows, cols, dtype, ld, offset)
        x[2] = 0
        q, scale = int8.quantize(x)
        _check_rows(q, scale, x.cpu().double())
        for out in TYPES:
            y = int8.dequantize(q, scale, out)
            assert torch.equal(y, (q.float() * scale[:, None]).to(out))
        wide = torch.zeros(rows, cols + 5, dtype=torch.int8, device=DEV)
        wide[:, 3:3 + cols] = q
        assert torch.equal(int8.dequantize(wide[:, 3:3 + cols], scale, dtype), int8.dequantize(q, scale, dtype))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("residual", [False, True])
def test_rms_norm(dtype, cols, residual):
    rows = 1 if cols in (7, 4096) else (33 if cols < 8192 else 5)
    for wtype in {dtype, torch.float32}:
        _say("rms_norm", IDS[dtype], IDS[wtype], rows, cols, residual)
        x = _values(cols + 1, rows, cols, dtype, cols + 1, 3)
        res = _values(cols + 2, rows, cols, dtype, cols + 8, 0) if residual else None
        w = (1 + 0.3 * torch.randn(cols, generator=_gen(3))).to(wtype).to(DEV)
        q, scale, h = int8.rms_norm(x, w, res, eps=1e-5)
        if residual:
            assert torch.equal(h, (x.float() + res.float()).to(dtype))
        else:
            assert h is x
        h64 = h.cpu().double()
        want = h64 * ((h64 * h64).mean(1, keepdim=True) + 1e-5).rsqrt() * w.cpu().double()
        _check_rows(q, scale, want)


def test_rows_that_are_not_finite():
    x = torch.randn(6, 600, generator=_gen(1)).to(DEV)
    x[1, 599] = float("nan")
    x[2, 3] = float("inf")
    x[3, 512] = -float("inf")
    x[4] = 0
    w = torch.ones(600, device=DEV)
    for q, scale in (int8.quantize(x), int8.rms_norm(x, w)[:2]):
        y = int8.dequantize(q, scale, torch.float32)
        assert torch.isnan(y[1:4]).all() and torch.isfinite(y[[0, 4, 5]]).all()
        assert (y[4] == 0).all() and (q[4] == 0).all()


def test_rows_of_tiny_and_huge_values():
    x = torch.randn(4, 100, generator=_gen(1))
    x[0] *= 1e-38  # below the least maximum a scale is made from: zeros
    x[1] *= 1e-20
    x[2] *= 1e37
    x = x.to(DEV)
    q, scale = int8.quantize(x)
    assert (q[0] == 0).all() and torch.isfinite(scale).all() and (scale > 0).all()
    _check_rows(q[1:], scale[1:], x[1:].cpu().double())


@pytest.mark.parametrize("rows,cols", [(0, 16), (16, 0), (0, 0)])
def test_empty_rows(rows, cols):
    x = torch.zeros(rows, cols, device=DEV, dtype=torch.bfloat16)
    w = torch.ones(cols, device=DEV, dtype=torch.bfloat16)
    q, scale = int8.quantize(x)
    assert q.shape == (rows, cols) and scale.shape == (rows,) and torch.isfinite(scale).all()
    assert int8.dequantize(q, scale).shape == (rows, cols)
    q, scale, h = int8.rms_norm(x, w, x)
    assert h.shape == (rows, cols) and torch.isfinite(scale).all()
    gx, gw = int8.rms_norm_backward(x, x, w)
    assert gx.shape == (rows, cols) and gw.shape == (cols,) and (gw == 0).all()


def _norm_grads(gy, h, w, eps, gh):
    gy, h, w = (t.cpu().double() for t in (gy, h, w))
    rstd = ((h * h).mean(1, keepdim=True) + eps).rsqrt()
    xh, u = h * rstd, gy * w
    gx = rstd * (u - xh * (u * xh).mean(1, keepdim=True))
    size = rstd * (u.abs() + xh.abs() * (u * xh).abs().mean(1, keepdim=True))
    if gh is not None:
        gx = gx + gh.cpu().double()
        size = size + gh.cpu().double().abs()
    return gx, size, (gy * xh).sum(0), (gy * xh).abs().sum(0)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 4096), (3, 7), (70, 512), (700, 129), (33, 2048), (20, 8192),
                                       (9, 8193), (5, 20011), (2500, 264), (1100, 2052), (40, 9), (600, 4095), (300, 8190),
                                       (700, 5001)])
def test_rms_norm_backward(dtype, rows, cols):
    for wtype, residual in ((dtype, True), (torch.float32, False)):
        _say("rms_norm_backward", IDS[dtype], IDS[wtype], rows, cols, residual)
        gy = _values(1, rows, cols, dtype, cols + 1, 1)
        h = _values(2, rows, cols, dtype, cols + 3, 0)
        if rows > 2:
            h[1] = 0
        gh = _values(3, rows, cols, dtype) if residual else None
        w = (1 + 0.3 * torch.randn(cols, generator=_gen(3))).to(wtype).to(DEV)
        gx, gw = int8.rms_norm_backward(gy, h, w, 1e-5, gh)
        assert gx.dtype == dtype and gw.dtype == wtype
        want, size, want_w, size_w = _norm_grads(gy, h, w, 1e-5, gh)
        assert ((gx.cpu().double() - want).abs() <= U[dtype] * want.abs() + 2e-5 * size + LEAST[dtype]).all()
        assert ((gw.cpu().double() - want_w).abs() <= U[wtype] * want_w.abs() + 2e-5 * size_w + LEAST[wtype]).all()
        again = int8.rms_norm_backward(gy, h, w, 1e-5, gh)
        assert torch.equal(gx, again[0]) and torch.equal(gw, again[1])


def test_rms_norm_backward_against_differences():
    """grad . d equals the central difference of sum(gy * norm(h)) along d, taken
    in 64 bits: its own error is of order 1e-8, the gradients' 2e-5."""
    rows, cols, eps, step = 9, 130, 1e-5, 1e-4
    gy, h, d = (_values(s, rows, cols, torch.float32) for s in (1, 2, 3))
    w, dw = (torch.randn(cols, generator=_gen(s)).to(DEV) for s in (4, 5))
    gx, gw = int8.rms_norm_backward(gy, h, w, eps)
    f64 = lambda t: t.cpu().double()  # noqa: E731

    def f(hh, ww):
        return (f64(gy) * hh * ((hh * hh).mean(1, keepdim=True) + eps).rsqrt() * ww).sum()

    slope = (f(f64(h) + step * f64(d), f64(w)) - f(f64(h) - step * f64(d), f64(w))) / (2 * step)
    _, size, _, size_w = _norm_grads(gy, h, w, eps, None)
    assert abs((f64(gx) * f64(d)).sum() - slope) <= 3e-5 * (size * f64(d).abs()).sum()
    slope = (f(f64(h), f64(w) + step * f64(dw)) - f(f64(h), f64(w) - step * f64(dw))) / (2 * step)
    assert abs((f64(gw) * f64(dw)).sum() - slope) <= 3e-5 * (size_w * f64(dw).abs()).sum()


def _check_matmul(c, a, sa, b, sb, bias, dtype):
    acc = a.cpu().double() @ b.cpu().double().t()
    want = acc * sa.cpu().double()[:, None] * sb.cpu().double()
    size = want.abs()
    if bias is not None:
        want = want + bias.cpu().double()
        size = size + bias.cpu().double().abs()
    assert c.dtype == dtype and c.shape == want.shape
    assert ((c.cpu().double() - want).abs() <= U[dtype] * want.abs() + 5 * E * size + LEAST[dtype]).all()


# Rows of a from one token on, around every tile edge; k around the steps of a
# tile and of a vector; odd and aligned sizes.
SIZES = [(1, 1, 1), (1, 64, 128), (1, 1000, 4096), (1, 333, 1001), (2, 17, 15), (3, 129, 257), (5, 4096, 512),
         (8, 250, 1024), (15, 48, 16), (16, 512, 4096), (16, 16, 33), (17, 100, 640), (31, 257, 2049), (32, 64, 64),
         (33, 65, 127), (48, 1024, 2048), (63, 63, 63), (64, 512, 1000), (65, 300, 144), (100, 1, 500),
         (128, 128, 128), (129, 127, 255), (200, 1000, 1600), (255, 257, 256), (256, 512, 1024), (257, 256, 130),
         (300, 600, 16), (511, 1030, 384), (513, 300, 4000), (1000, 1000, 1000), (1024, 768, 2304),
         (2049, 130, 272), (20, 300, 1040), (32, 48, 100), (40, 77, 515), (50, 200, 300), (64, 129, 2000), (90, 200, 17)]


@pytest.mark.parametrize("m,n,k", SIZES, ids=lambda v: str(v))
def test_matmul(m, n, k):
    for dtype, with_bias, lda, ldb, off in ((torch.bfloat16, False, k, k, 0), (torch.float16, True, k + 1, k, 1),
                                            (torch.float32, True, k + 16, k + 48, 16),
                                            (torch.bfloat16, True, k, k + 5, 3)):
        _say("matmul", m, n, k, IDS[dtype], with_bias, lda, ldb, off)
        a, sa = _int8(1, m, k, lda, off, full=True)
        b, sb = _int8(2, n, k, ldb, off, full=True)
        bias = torch.randn(n, generator=_gen(3)).to(dtype).to(DEV) if with_bias else None
        _check_matmul(int8.matmul(a, sa, b, sb, bias, dtype), a, sa, b, sb, bias, dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("m,n,k", [(8192, 4097, 128), (2048, 2049, 384), (4096, 2049, 128), (512, 4095, 640), (1024, 1023, 256)],
                         ids=lambda v: str(v))
def test_matmul_odd_columns(dtype, m, n, k):
    """Rows of the output that start at any half of a word, in every tile size:
    the same values as with one column more."""
    _say("matmul odd columns", IDS[dtype], m, n, k)
    a, sa = _int8(1, m, k, full=True)
    b, sb = _int8(2, n + 1, k, full=True)
    bias = torch.randn(n + 1, generator=_gen(3)).to(dtype).to(DEV)
    even = int8.matmul(a, sa, b, sb, bias, dtype)
    assert torch.equal(int8.matmul(a, sa, b[:n], sb[:n], bias[:n], dtype), even[:, :n])
    rows = torch.tensor([0, 1, m // 2 + 1, m - 1])
    want = (a[rows].cpu().double() @ b.cpu().double().t()) * sa[rows].cpu().double()[:, None] * sb.cpu().double() + bias.cpu().double()
    assert torch.allclose(even[rows].cpu().double(), want, rtol=1e-5 if dtype == torch.float32 else 1e-2, atol=1e-4)


@pytest.mark.parametrize("m,n", [(1, 40), (20, 40), (130, 70)])
def test_matmul_largest_sums(m, n):
    """-128 * -128 over the longest k: 2^14 (2^17 - 1), just inside i32."""
    k = (1 << 17) - 1
    a = torch.full((m, k), -128, dtype=torch.int8, device=DEV)
    b = torch.full((n, k), -128, dtype=torch.int8, device=DEV)
    b[1] = 127
    one = torch.ones(max(m, n), device=DEV)
    c = int8.matmul(a, one[:m], b, one[:n], dtype=torch.float32)
    want = torch.full((m, n), float((1 << 14) * k), device=DEV)
    want[:, 1] = float(-128 * 127 * k)
    assert torch.equal(c, want)
    with pytest.raises(nat.HipError, match="exact up to"):
        int8.matmul(torch.zeros(1, 1 << 17, dtype=torch.int8, device=DEV), one[:1],
                    torch.zeros(1, 1 << 17, dtype=torch.int8, device=DEV), one[:1])


@pytest.mark.parametrize("m,n,k", [(0, 8, 16), (8, 0, 16), (0, 0, 0), (5, 7, 0)])
def test_matmul_empty(m, n, k):
    a, sa = _int8(1, m, k)
    b, sb = _int8(2, n, k)
    bias = torch.randn(n, generator=_gen(3)).to(DEV)
    c = int8.matmul(a, sa, b, sb, bias, torch.float32)
    assert torch.equal(c, bias.expand(m, n))
    assert (int8.matmul(a, sa, b, sb) == 0).all()
    g = torch.ones(m, n, device=DEV)
    assert torch.equal(int8.backward_a(g, b, sb), torch.zeros(m, k, device=DEV))
    assert torch.equal(int8.backward_b(g, a, sa), torch.zeros(n, k, device=DEV))


def test_scales_that_are_not_finite_stay_in_their_rows():
    a, sa = _int8(1, 20, 300)
    b, sb = _int8(2, 30, 300)
    sa[3], sb[5] = float("nan"), float("inf")
    c = int8.matmul(a, sa, b, sb, dtype=torch.float32)
    bad = torch.zeros(20, 30, dtype=torch.bool, device=DEV)
    bad[3], bad[:, 5] = True, True
    assert torch.equal(~torch.isfinite(c), bad)


GRADS = [(1, 1, 1), (1, 70, 130), (2, 3, 5), (16, 64, 128), (17, 33, 65), (64, 64, 64), (100, 130, 70), (127, 129, 255),
         (128, 256, 128), (130, 1000, 520), (301, 515, 260), (512, 512, 512), (700, 96, 1040), (1031, 257, 129),
         (1536, 1024, 768), (40, 2050, 72), (2050, 40, 72), (300, 2100, 1030), (2100, 300, 1030), (1000, 1100, 1200),
         (9, 20, 8), (66, 8, 9), (65, 190, 63), (129, 7, 40), (7, 100, 40)]


def _check_grad(got, g, x, dtype):
    """got against g @ x (f64, on the CPU)."""
    want, size = g @ x, g.abs() @ x.abs()
    u = 2 * E if dtype == torch.float32 else U[dtype]
    off = (got.cpu().double() - want).abs()
    assert got.dtype == dtype and got.shape == want.shape
    assert (off <= (1.01 * u + g.shape[1] * E) * size + U[dtype] * want.abs() + LEAST[dtype]).all()
    if want.numel() >= 1000:
        assert off.norm() <= (2e-6 if dtype == torch.float32 else 1.2 * u) * want.norm()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("m,n,k", GRADS, ids=lambda v: str(v))
def test_gradients(dtype, m, n, k):
    for ldg, ldq, off in ((n, k, 0), (n + 1, k + 3, 1), (n + 8, k + 16, 8)):
        _say("backward", IDS[dtype], m, n, k, ldg, ldq, off)
        g = _values(1, m, n, dtype, ldg, off)
        a, sa = _int8(2, m, k, ldq, off)
        b, sb = _int8(3, n, k, ldq, off)
        f64 = lambda t: t.cpu().double()  # noqa: E731
        _check_grad(int8.backward_a(g, b, sb), f64(g), f64(b) * f64(sb)[:, None], dtype)
        _check_grad(int8.backward_b(g, a, sa), f64(g).t(), f64(a) * f64(sa)[:, None], dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("m,n,k", [(70, 90, 100), (300, 2100, 1030), (2100, 300, 1030), (40, 2050, 72), (2050, 40, 72)],
                         ids=lambda v: str(v))
def test_gradients_that_are_not_finite(dtype, m, n, k):
    """NaN and infinity in grad_c and in a scale reach the outputs that they are
    a term of, and no others."""
    nan, inf = float("nan"), float("inf")
    for pad in (0, 1):
        _say("backward not finite", IDS[dtype], m, n, k, pad)
        g = _values(1, m, n, dtype, n + pad)
        a, sa = _int8(2, m, k, k + pad)
        b, sb = _int8(3, n, k, k + pad)
        clean = int8.backward_a(g, b, sb), int8.backward_b(g, a, sa)
        g[1, n - 1], g[3, 4], g[m - 1, n - 2] = nan, inf, -inf
        b[4], b[n - 2], a[3], a[m - 1] = 3, 5, -2, 7  # no zeros where infinities meet them
        got_a, got_b = int8.backward_a(g, b, sb), int8.backward_b(g, a, sa)
        assert torch.isnan(got_a[1]).all() and torch.isnan(got_b[n - 1]).all()
        assert (got_a[3] == inf).all() and (got_a[m - 1] == -inf).all()
        assert (got_b[4] == -inf).all() and (got_b[n - 2] == -inf).all()
        for got, was, hit in ((got_a, clean[0], (1, 3, m - 1)), (got_b, clean[1], (n - 1, 4, n - 2))):
            rest = torch.ones(got.shape[0], dtype=torch.bool, device=DEV)
            rest[list(hit)] = False
            assert torch.isfinite(got[rest]).all()
        sb[n - 1], sa[0] = nan, nan
        assert torch.isnan(int8.backward_a(g, b, sb)).all() and torch.isnan(int8.backward_b(g, a, sa)).all()


def test_gradients_of_the_largest_numbers():
    """Close to the end of f32's range nothing overflows on the way."""
    top = float(torch.finfo(torch.float32).max)
    for m, n in ((64, 64), (2100, 300)):
        g = torch.zeros(m, n, device=DEV)
        g[:, 5] = top
        b = torch.ones(n, 72, dtype=torch.int8, device=DEV)
        out = int8.backward_a(g, b, torch.ones(n, device=DEV))
        assert torch.equal(out, torch.full_like(out, top))


def test_gradients_against_differences():
    """sum(G * (A B^T)) is linear in either operand, so its difference along any
    direction is the gradient's product with it."""
    m, n, k = 40, 72, 150
    g = _values(1, m, n, torch.float32)
    a, sa = _int8(2, m, k)
    b, sb = _int8(3, n, k)
    f64 = lambda t: t.cpu().double()  # noqa: E731
    av, bv, gv = f64(a) * f64(sa)[:, None], f64(b) * f64(sb)[:, None], f64(g)
    f = lambda x, y: (gv * (x @ y.t())).sum()  # noqa: E731
    da, db = torch.randn(m, k, generator=_gen(4)).double(), torch.randn(n, k, generator=_gen(5)).double()
    for grad, d, slope in ((int8.backward_a(g, b, sb), da, (f(av + da, bv) - f(av - da, bv)) / 2),
                           (int8.backward_b(g, a, sa), db, (f(av, bv + db) - f(av, bv - db)) / 2)):
        size = (f64(grad).abs() * d.abs()).sum()
        assert abs((f64(grad) * d).sum() - slope) <= 1e-5 * size


def test_gradients_of_wide_range():
    """Gradients and scales far from one: nothing is lost below or above the
    16-bit types' ranges on the way."""
    for m, n, k in ((130, 200, 96), (2050, 40, 72)):
        _check_wide_range(m, n, k)


def _check_wide_range(m, n, k):
    for dtype, gs, ss in ((torch.bfloat16, 1e-20, 1e-6), (torch.bfloat16, 1e15, 1e3), (torch.float16, 1e-3, 1e-5),
                          (torch.float16, 1e3, 1e-5), (torch.float16, 1e-4, 3e2), (torch.float32, 1e-15, 1e-10)):
        _say("wide", IDS[dtype], gs, ss)
        g = (torch.randn(m, n, generator=_gen(1)) * gs).to(dtype).to(DEV)
        a, sa = _int8(2, m, k)
        sa = sa * ss
        f64 = lambda t: t.cpu().double()  # noqa: E731
        want = f64(g).t() @ (f64(a) * f64(sa)[:, None])
        got = f64(int8.backward_b(g, a, sa))
        fine = want.abs() < 6e4 if dtype == torch.float16 else want.abs() < 1e38
        u = U[dtype] if dtype != torch.float32 else 2e-6
        floor = 2.0 ** -24 if dtype == torch.float16 else 0.0
        off = (got - want)[fine]
        assert torch.isfinite(got[fine]).all()
        assert off.norm() <= 1.2 * u * want[fine].norm() + floor * off.numel() ** 0.5


def test_rows_past_32_bits():
    """Row strides that put rows beyond 2^32 bytes and 2^31 elements."""
    k, ld = 640, (1 << 31) + 16
    store = torch.empty(2 * ld + k, dtype=torch.int8, device=DEV)
    b = store.as_strided((3, k), (ld, 1))
    small, sb = _int8(1, 3, k)
    b.copy_(small)
    for m in (1, 200):
        a, sa = _int8(2, m, k)
        assert torch.equal(int8.matmul(a, sa, b, sb), int8.matmul(a, sa, small, sb))
        assert torch.equal(int8.matmul(b, sb, a, sa), int8.matmul(small, sb, a, sa))
    g = _values(3, 50, 3, torch.bfloat16)
    assert torch.equal(int8.backward_a(g, b, sb), int8.backward_a(g, small, sb))
    assert torch.equal(int8.dequantize(b, sb), int8.dequantize(small, sb))
    x = store.view(torch.int8)[: 2 * ld + k // 2 * 2].view(torch.bfloat16).as_strided((3, k // 2), (ld // 2, 1))
    near = _values(4, 3, k // 2, torch.bfloat16)
    x.copy_(near)
    w = torch.ones(k // 2, dtype=torch.bfloat16, device=DEV)
    for far_out, near_out in ((int8.quantize(x), int8.quantize(near)), (int8.rms_norm(x, w, x), int8.rms_norm(near, w, near)),
                              (int8.rms_norm_backward(x, x, w), int8.rms_norm_backward(near, near, w)),
                              ([int8.backward_b(x, small, sb)], [int8.backward_b(near, small, sb)])):
        for u, v in zip(far_out, near_out):
            assert torch.equal(u, v)


def test_refusals():
    x = torch.zeros(4, 8, device=DEV)
    w = torch.ones(8, device=DEV)
    q, s = int8.quantize(x)
    with pytest.raises(ValueError, match="neighbours"):
        int8.quantize(x.t())
    with pytest.raises(ValueError, match="neighbours"):
        int8.quantize(x[:1].expand(4, 8))
    with pytest.raises(ValueError, match="2D"):
        int8.quantize(x[0])
    with pytest.raises(ValueError, match="Unsupported dtype"):
        int8.quantize(x.double())
    with pytest.raises(ValueError, match="Unsupported dtype"):
        int8.dequantize(q, s, torch.float64)
    with pytest.raises(ValueError, match="must be torch.int8"):
        int8.dequantize(x, s)
    with pytest.raises(ValueError, match="scale has shape"):
        int8.dequantize(q, s[:3])
    with pytest.raises(ValueError, match="weight must be"):
        int8.rms_norm(x.bfloat16(), w.half())
    with pytest.raises(ValueError, match="residual has shape"):
        int8.rms_norm(x, w, x[:3])
    with pytest.raises(ValueError, match="residual must be"):
        int8.rms_norm(x, w, x.half())
    with pytest.raises(nat.HipError, match="eps"):
        int8.rms_norm(x, w, eps=-1.0)
    with pytest.raises(ValueError, match="grad_y has shape"):
        int8.rms_norm_backward(x[:, :7], x, w)
    with pytest.raises(ValueError, match="grad_h must be"):
        int8.rms_norm_backward(x, x, w, grad_h=x.half())
    with pytest.raises(ValueError, match="Dimension mismatch: a is 4x8, b is 4x7"):
        int8.matmul(q, s, q[:, :7], s)
    with pytest.raises(ValueError, match="b_scale has shape"):
        int8.matmul(q, s, q[:3], s)
    with pytest.raises(ValueError, match="a_scale must be"):
        int8.matmul(q, s.half(), q, s)
    with pytest.raises(ValueError, match="bias must be"):
        int8.matmul(q, s, q, s, torch.zeros(4, device=DEV))
    with pytest.raises(ValueError, match="a must be torch.int8"):
        int8.matmul(x, s, q, s)
    with pytest.raises(ValueError, match="Dimension mismatch: grad_c is 4x8, b is 4x8"):
        int8.backward_a(x, q, s)
    with pytest.raises(ValueError, match="Dimension mismatch: grad_c is 8x4, a is 4x8"):
        int8.backward_b(x.t().contiguous(), q, s)
    with pytest.raises(ValueError, match="same device"):
        int8.matmul(q, s, q, s.cpu())


def test_other_stream():
    """Launches follow torch's current stream, workspaces too."""
    x = _values(1, 300, 1000, torch.bfloat16)
    w = torch.ones(1000, dtype=torch.bfloat16, device=DEV)
    b, sb = _int8(2, 200, 1000)

    def step():
        q, s, h = int8.rms_norm(x, w, x)
        c = int8.matmul(q, s, b, sb)
        ga, gb = int8.backward_a(c, b, sb), int8.backward_b(c, q, s)
        return [q, s, h, c, ga, gb, *int8.rms_norm_backward(ga, h, w, grad_h=x)]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    for u, v in zip(got, want):
        assert torch.equal(u, v)


@pytest.mark.parametrize("m", [1, 20, 300])
def test_graph(m):
    """A captured pass of all operators, replayed with eager work in between,
    equals the eager pass on the inputs of the moment."""
    k, n = 1000, 336
    x = _values(1, m, k, torch.bfloat16)
    w = torch.ones(k, dtype=torch.bfloat16, device=DEV)
    b, sb = _int8(2, n, k)

    def step():
        q, s, h = int8.rms_norm(x, w, x)
        c = int8.matmul(q, s, b, sb)
        ga, gb = int8.backward_a(c, b, sb), int8.backward_b(c, q, s)
        return [q, s, h, c, ga, gb, *int8.rms_norm_backward(ga, h, w, grad_h=x), int8.dequantize(*int8.quantize(x))]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        x.copy_(_values(10 + i, m, k, torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        for u, v in zip(got, step()):
            assert torch.equal(u, v)


def test_numbers_of_a_known_case():
    """A row whose rounding is known by hand, ties to even included."""
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -127.0, 126.5]], device=DEV)
    q, scale = int8.quantize(x)
    assert q.cpu().tolist() == [[127, 0, 2, 2, 0, -2, -127, 126]] and scale.item() == 1.0
    assert np.array_equal(int8.dequantize(q, scale, torch.float32).cpu().numpy(), q.cpu().numpy().astype(np.float32))


@pytest.mark.parametrize("m", [4, 5, 16, 17, 32, 33, 64])
def test_matmul_wide(m):
    """More columns than some of the ways for few rows take, aligned rows and not."""
    n, k = 12300, 144
    for ldb, off in ((k, 0), (k + 1, 1)):
        _say("matmul wide", m, n, k, ldb, off)
        a, sa = _int8(1, m, k, full=True)
        b, sb = _int8(2, n, k, ldb, off, full=True)
        _check_matmul(int8.matmul(a, sa, b, sb), a, sa, b, sb, None, torch.bfloat16)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_gradients_of_long_sums(dtype):
    """Few outputs and a long sum, which is cut into slices."""
    m, n, k = 5000, 40, 72
    g = _values(1, m, n, dtype)
    a, sa = _int8(2, m, k)
    f64 = lambda t: t.cpu().double()  # noqa: E731
    _check_grad(int8.backward_b(g, a, sa), f64(g).t(), f64(a) * f64(sa)[:, None], dtype)
    again = int8.backward_b(g, a, sa)
    assert torch.equal(again, int8.backward_b(g, a, sa))
