"""The layer in 8-bit floating point, layer norm and dropout where a form of a
kernel ends or another begins: sums split between waves or slices with a step
more on one side, numbers that are not finite on the matrix instructions' own
scales, the largest launches, columns at the limits of a row's threads.

Tolerances as in test_gpu_fp8.py and test_gpu_layers.py."""
import pytest
import torch

from tropical_gemm import _native as nat
from tropical_gemm import fp8, layers

pytestmark = pytest.mark.gpu

DEV = "cuda"
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def _operand(seed, rows, k, scale_rows):
    b = torch.randint(0, 256, (rows, k), generator=_gen(seed), dtype=torch.int32)
    b = torch.where((b & 127) == 127, b - 1, b).to(torch.uint8).to(DEV).view(E4M3)
    s = torch.randint(118, 126, (-(-k // 128), scale_rows), generator=_gen(seed + 1), dtype=torch.int32)
    return b, s.to(torch.uint8).to(DEV).view(E8M0).t()


def _exact(q, s, br):
    f = torch.pow(2.0, s.view(torch.uint8).double() - 127)
    return q.float().double() * f.repeat_interleave(br, 0)[:q.shape[0]].repeat_interleave(128, 1)[:, :q.shape[1]]


def _plan(m, n, k):
    return nat.load().tg_f8_gemm_plan(1, 256, k, 256, k, m, n, k).decode()


def _check(m, n, k):
    a, sa = _operand(m + k, m, k, m)
    b, sb = _operand(n + 7 * k, n, k, -(-n // 128))
    c = fp8.matmul(a, sa, b, sb, dtype=torch.bfloat16)
    da, db = _exact(a, sa, 1), _exact(b, sb, 128)
    want, size = torch.mm(da, db.t()), torch.mm(da.abs(), db.abs().t())
    bound = ((k + 1) * 2.0 ** -23 + 2.0 ** -10) * size
    assert ((c.double() - want).abs() <= bound + 2.0 ** -8 * (want.abs() + bound)).all(), _plan(m, n, k)


@pytest.mark.parametrize("form,sizes", [
    # Odd numbers of steps: one half of the waves has one more.
    ("tiles 64x64 halves", [(129, 1033, 4208), (128, 1024, 2944), (100, 2000, 1920 + 128), (128, 4096, 4224)]),
    ("tiles 128x64 halves", [(250, 8192, 4224), (256, 8000, 3968), (131, 8190, 2960)]),
    ("slices", [(65, 70, 8192), (100, 1000, 4224), (256, 256, 8320), (66, 128, 2064)]),
])
def test_split_sums(form, sizes):
    plans = [_plan(*s) for s in sizes]
    assert any(form in p for p in plans), plans
    for s, p in zip(sizes, plans):
        print("[case]", s, p, flush=True)
        _check(*s)


@pytest.mark.parametrize("dtype,u", [(torch.bfloat16, 2.0 ** -8), (torch.float32, 2.0 ** -24)], ids=["bf16", "f32"])
@pytest.mark.parametrize("m", [1, 16, 17, 33, 47, 48, 49, 64])
def test_few_rows(m, dtype, u):
    """Whole and part words, either side of the weights that the rows are given up at."""
    for n, k in [(1, 128), (19, 127), (130, 1156), (1000, 4112), (2064, 8192), (4128, 4096), (300, 1)]:
        print("[case]", m, n, k, flush=True)
        a, sa = _operand(m + k, m, k, m)
        b, sb = _operand(n + 7 * k, n, k, -(-n // 128))
        c = fp8.matmul(a, sa, b, sb, dtype=dtype)
        da, db = _exact(a, sa, 1), _exact(b, sb, 128)
        want, size = torch.mm(da, db.t()), torch.mm(da.abs(), db.abs().t())
        bound = ((k + 1) * 2.0 ** -23 + (2.0 ** -10 if dtype is torch.bfloat16 else 0)) * size
        assert ((c.double() - want).abs() <= bound + u * (want.abs() + bound)).all()


@pytest.mark.parametrize("m,n,k", [(300, 512, 129 * 16), (520, 777, 1600), (4096, 300, 256), (70, 4096, 144)])
def test_steps_of_every_count(m, n, k):
    """One step, two, three and more of each form that these sizes take."""
    for steps in (1, 2, 3, 4, 5):
        for kk in (steps * 128, steps * 128 - 112):
            print("[case]", m, n, kk, _plan(m, n, kk), flush=True)
            _check(m, n, kk)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,n", [(5, 66), (33, 66), (70, 66), (300, 300), (1500, 1400), (4096, 4096)])
def test_not_finite(dtype, m, n):
    """The NaN scale and NaN numbers reach their rows or columns, and no others."""
    k = 384
    one = 0x38
    for what in ("a scale", "b scale", "a", "b"):
        qa, qb = (torch.full((r, k), one, dtype=torch.uint8, device=DEV) for r in (m, n))
        sa = torch.full((3, m), 120, dtype=torch.uint8, device=DEV)
        sb = torch.full((3, -(-n // 128)), 120, dtype=torch.uint8, device=DEV)
        rows, cols = torch.zeros(m, dtype=torch.bool, device=DEV), torch.zeros(n, dtype=torch.bool, device=DEV)
        if what == "a scale":
            sa[1, 2], rows[2] = 255, True
            qa[2, 128:256] = 0
        elif what == "b scale":
            sb[2, 0], cols[:128] = 255, True
        elif what == "a":
            qa[m - 1, k - 1], rows[m - 1] = 0x7f, True
        else:
            qb[n - 1, 5], cols[n - 1] = 0xff, True
        print("[case]", what, m, n, flush=True)
        c = fp8.matmul(qa.view(E4M3), sa.view(E8M0).t(), qb.view(E4M3), sb.view(E8M0).t(), dtype=dtype)
        bad = rows[:, None] | cols[None, :]
        assert torch.equal(torch.isnan(c), bad), what
        assert (c[~bad] == k * 2.0 ** -14).all()


@pytest.mark.parametrize("m", [5, 40, 70, 300])
def test_scales_of_all_sizes_bf16(m):
    """Powers of two at both ends, alone and against each other."""
    n, k = 200, 256
    qa, qb = (torch.full((r, k), 0x38, dtype=torch.uint8, device=DEV).view(E4M3) for r in (m, n))
    for ea, eb in [(-100, 0), (0, -100), (100, -100), (-100, 100), (60, 59), (-60, -60), (111, 0), (119, -119), (0, 0)]:
        sa = torch.full((2, m), 127 + ea, dtype=torch.uint8, device=DEV).view(E8M0).t()
        sb = torch.full((2, 2), 127 + eb, dtype=torch.uint8, device=DEV).view(E8M0).t()
        c = fp8.matmul(qa, sa, qb, sb)
        assert (c.double() == k * 2.0 ** (ea + eb)).all(), (ea, eb)


def test_gradients_not_finite():
    """A NaN or an infinity in the gradient reaches its row or column alone, in each
    type and both ways."""
    for m, n, k in [(40, 70, 130), (300, 900, 1100)]:
        w, sw = fp8.quantize(torch.randn(n, k, generator=_gen(1)).to(DEV), 128)
        x, sx = fp8.quantize(torch.randn(m, k, generator=_gen(2)).to(DEV))
        for dtype in (torch.bfloat16, torch.float16, torch.float32):
            g = torch.randn(m, n, generator=_gen(3)).to(dtype).to(DEV)
            want_a, want_b = fp8.backward_a(g, w, sw), fp8.backward_b(g, x, sx)
            g2 = g.clone()
            g2[7, 9], g2[11, 20] = float("nan"), float("inf")
            ga, gb = fp8.backward_a(g2, w, sw), fp8.backward_b(g2, x, sx)
            ra, rb = torch.zeros(m, dtype=torch.bool), torch.zeros(n, dtype=torch.bool)
            ra[7] = ra[11] = rb[9] = rb[20] = True
            assert torch.equal(ga.cpu()[~ra], want_a.cpu()[~ra]) and torch.equal(gb.cpu()[~rb], want_b.cpu()[~rb])
            assert torch.isnan(ga[7]).all() and torch.isnan(gb[9]).all()
            assert not torch.isfinite(ga[11]).any() and not torch.isfinite(gb[20]).any()
            # NaN scales of the operand.
            bad = sw.clone()
            bad.view(torch.uint8)[0, 0] = 255
            ga = fp8.backward_a(g, w, bad)
            assert torch.isnan(ga[:, :128]).all() and torch.equal(ga[:, 128:], want_a[:, 128:])


def test_many_rows():
    """More rows than one launch takes: each part has its own rows' masks."""
    rows, cols, p = (1 << 21) + 300, 16, 0.25
    x = torch.randn(rows, cols, device=DEV).bfloat16()
    w = torch.ones(cols, device=DEV).bfloat16()
    y, h, mean, rstd = layers.layer_norm(x, w, None, None, 1e-5, p, 5, 1)
    assert torch.equal(h, layers.dropout(x, p, 5, 1))
    tail = 400  # rows of both launches, each as the others
    z = layers.layer_norm(h[-tail:].contiguous(), w)
    assert torch.equal(z[0], y[-tail:]) and torch.equal(z[2], mean[-tail:]) and torch.equal(z[3], rstd[-tail:])
    q, s = fp8.quantize(x)
    q2, s2 = fp8.quantize(x[-tail:])
    assert torch.equal(q[-tail:].view(torch.uint8), q2.view(torch.uint8))
    assert torch.equal(s[-tail:].view(torch.uint8), s2.view(torch.uint8))
    assert torch.equal(fp8.dequantize(q, s)[-tail:], fp8.dequantize(q2, s2))
    gx = layers.layer_norm_backward(x, h, mean, rstd, w, None, p, 5, 1)
    assert torch.equal(gx[0], layers.dropout(gx[1].float(), p, 5, 1).bfloat16()) or \
        ((gx[0].float() - layers.dropout(gx[1].float(), p, 5, 1)).abs() <= 2.0 ** -7 * gx[1].float().abs() * 1.34).all()


def test_wide_rows():
    """One row of many columns: blocks, norm, its gradients and masks."""
    cols = 300_001
    x = torch.randn(3, cols, generator=_gen(1))
    w = torch.randn(cols, generator=_gen(2))
    y, h, mean, rstd = layers.layer_norm(x.to(DEV), w.to(DEV), None, x.to(DEV), 1e-5, 0.5, 9, 3)
    drop = layers.dropout(x.to(DEV), 0.5, 9, 3, x.to(DEV))
    assert torch.equal(h, drop)
    h64 = h.cpu().double()
    m = h64.mean(1, keepdim=True)
    s = ((h64 - m).square().mean(1, keepdim=True) + 1e-5).rsqrt()
    want = (h64 - m) * s * w.double()
    assert ((y.cpu().double() - want).abs() <= 4e-5 * (want.abs() + w.double().abs())).all()
    g = torch.randn(3, cols, generator=_gen(4))
    gx, gr, gw, gb = layers.layer_norm_backward(g.to(DEV), h, mean, rstd, w.to(DEV), None, 0.5, 9, 3)
    xh, u = (h64 - m) * s, g.double() * w.double()
    want = s * (u - u.mean(1, keepdim=True) - xh * (u * xh).mean(1, keepdim=True))
    size = s * (u.abs() + u.abs().mean(1, keepdim=True) + xh.abs() * (u * xh).abs().mean(1, keepdim=True))
    assert ((gr.cpu().double() - want).abs() <= 1e-4 * size).all()
    assert ((gw.cpu().double() - (g.double() * xh).sum(0)).abs() <= 1e-4 * (g.double() * xh).abs().sum(0) + 1e-6).all()
    assert ((gb.cpu().double() - g.double().sum(0)).abs() <= 1e-6 * g.double().abs().sum(0)).all()
    q, sc = fp8.quantize(x.to(DEV))
    back = fp8.dequantize(q, sc, torch.float32).cpu()
    top = torch.nn.functional.pad(x.abs(), (0, -cols % 128)).view(3, -1, 128).amax(2).repeat_interleave(128, 1)[:, :cols]
    assert ((back - x).abs() <= torch.maximum(2.0 ** -4 * x.abs(), top * 2.0 ** -17)).all()


def test_on_another_stream():
    """Calls on a stream of their own, their inputs made there, outputs used on the
    default one after a wait."""
    side = torch.cuda.Stream()
    for turn in range(3):
        with torch.cuda.stream(side):
            x = torch.randn(500, 640, device=DEV).bfloat16()
            w = torch.randn(700, 640, device=DEV).bfloat16()
            q, s = fp8.quantize(x)
            qw, sw = fp8.quantize(w, 128)
            c = fp8.matmul(q, s, qw, sw)
            n, h, mean, rstd = layers.layer_norm(c, w.new_ones(700), None, None, 1e-5, 0.2, turn)
        torch.cuda.current_stream().wait_stream(side)
        for t in (x, w, q, s, qw, sw, c, n, h):
            t.record_stream(torch.cuda.current_stream())
        assert torch.equal(c, fp8.matmul(q, s, qw, sw))
        assert torch.equal(h, layers.dropout(c, 0.2, turn))


def test_refusals_on_the_gpu():
    x = torch.randn(4, 300, device=DEV)
    q, s = fp8.quantize(x)
    w, sw = fp8.quantize(x, 128)
    for call, message in [
        (lambda: fp8.quantize(x, 64), "block_rows"),
        (lambda: fp8.quantize(x.double()), "Unsupported dtype"),
        (lambda: fp8.quantize(x.t()), "neighbours"),
        (lambda: fp8.dequantize(q, s[:, :2]), "scale has shape"),
        (lambda: fp8.dequantize(q, s.view(torch.uint8)), "scale must be"),
        (lambda: fp8.dequantize(x, s), "q must be"),
        (lambda: fp8.matmul(q, s, w, s), "b_scale has shape"),
        (lambda: fp8.matmul(q, sw[:0], w, sw), "a_scale has shape"),
        (lambda: fp8.matmul(q[:, :100], s[:, :1], w, sw), "Dimension mismatch"),
        (lambda: fp8.matmul(q, s, w, sw, x[0]), "bias"),
        (lambda: fp8.matmul(q, s, w, sw, dtype=torch.float64), "Unsupported dtype"),
        (lambda: fp8.backward_a(x, w, sw), "Dimension mismatch"),
        (lambda: fp8.backward_b(x[:3], q, s), "Dimension mismatch"),
        (lambda: fp8.matmul(q.cpu(), s, w, sw), "device tensors"),
        (lambda: fp8.matmul(q, s.cpu(), w, sw), "same device"),
        (lambda: layers.dropout(x, 1.5, 1), "between 0 and 1"),
        (lambda: layers.dropout(x, float("nan"), 1), "between 0 and 1"),
        (lambda: layers.dropout(x, 0.5, -1), "seed is -1"),
        (lambda: layers.dropout(x, 0.5, 1 << 64), "seed is"),
        (lambda: layers.dropout(x, 0.5, 1, -1), "offset is -1"),
        (lambda: layers.dropout(x, 0.5, torch.zeros(2, dtype=torch.int64, device=DEV)), "one int64 element"),
        (lambda: layers.dropout(x, 0.5, torch.zeros(1, dtype=torch.int64)), "same device"),
        (lambda: layers.dropout(x, 0.5, 1, 0, x[:3]), "residual has shape"),
        (lambda: layers.layer_norm(x, x[0, :100]), "weight has shape"),
        (lambda: layers.layer_norm(x, x[0].half()), "weight must be"),
        (lambda: layers.layer_norm(x.half(), x[0], x[0].half()), "bias must be"),
        (lambda: layers.layer_norm_backward(x, x, x[0, :3], x[0, :4], x[0]), "mean has shape"),
        (lambda: layers.layer_norm_backward(x, x, x[0, :4].half(), x[0, :4], x[0]), "mean must be"),
    ]:
        with pytest.raises(ValueError, match=message):
            call()
    with pytest.raises(nat.HipError, match="eps"):
        layers.layer_norm(x, x[0], eps=-1.0)
