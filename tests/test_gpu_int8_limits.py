"""The 8-bit layer's operators at the limits of their definitions: ties, ranges,
rows in several workgroups, scales far from each other.  Expected values come
from integers, 64-bit sums or bits that have to be equal."""
import pytest
import torch

from tropical_gemm import int8
from tropical_gemm import pytorch as tgt

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16, torch.float32]
IDS = {torch.bfloat16: "bf16", torch.float16: "f16", torch.float32: "f32"}


def _say(*what):
    print("[case]", *what, flush=True)


def _gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def _rint_of_127ths(v, top):
    """rint(127 v / top), ties to even, of whole numbers v and top."""
    low = 127 * v.abs() // top
    rest = 2 * (127 * v.abs() - low * top)
    up = (rest > top) | ((rest == top) & (low % 2 == 1))
    return torch.sign(v) * (low + up.long())


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_ties_go_to_the_even_integer(dtype):
    """Every mantissa as a row's maximum (f32: maxima that 254 divides), beside the
    values nearest to a whole number and a half of its 127th parts.  All of
    them can be told from a tie: 127 v / top is one, or at least 1 / (2 top) of
    a step from one, 2^-12 in 16 bits."""
    bits = {torch.bfloat16: 8, torch.float16: 11, torch.float32: 24}[dtype]
    if dtype == torch.float32:
        top = torch.randint((1 << 23) // 254 + 1, (1 << 24) // 254, (2000, 1), generator=_gen(1)) * 254
    else:
        top = torch.arange(1 << (bits - 1), 1 << bits)[:, None]
    odd = 2 * torch.arange(-127, 127)[None] + 1
    v = (odd * top) // 254
    v = torch.where(v.abs() <= top, v, torch.zeros_like(v))
    v = torch.cat([top, -top // 2, v, (top + 1) // 2], 1)
    x = (v.double() * 2.0 ** -bits).to(dtype)
    v = (x.double() * 2.0 ** bits).long()  # what the type holds of them
    assert (x.double() * 2.0 ** bits == v.double()).all()
    want = _rint_of_127ths(v, v.abs().amax(1, keepdim=True))
    x = x.to(DEV)
    ones = torch.ones(x.shape[1], dtype=dtype, device=DEV)
    wide = torch.zeros(x.shape[0], 8200, dtype=dtype, device=DEV)  # the way of longer rows
    wide[:, :x.shape[1]] = x
    for q in (int8.quantize(x)[0], int8.rms_norm(x, ones)[0], int8.quantize(wide)[0][:, :x.shape[1]]):
        assert torch.equal(q.cpu().long(), want)


@pytest.mark.parametrize("cols", [8193, 8194, 8195, 8196, 8197, 8198, 8199, 16385, 16391])
def test_norm_backward_has_one_writer_for_each_column(cols):
    """Rows shared by workgroups of 8192 columns, the last one's fewer than eight:
    the columns before it belong to the workgroup before, bit for bit, and equal
    calls give equal bits."""
    rows, base = 3000, (cols - 1) // 8192 * 8192
    _say("norm backward", rows, cols)
    g, h = (torch.randn(rows, cols, generator=_gen(s)) * torch.exp(2 * torch.randn(rows, cols, generator=_gen(s + 2)))
            for s in (1, 2))
    w = torch.randn(cols, generator=_gen(5))
    last = slice(cols - 8, base)  # columns whose group the last workgroup loads too
    for t in (g, h, w):
        t[..., last] = t[..., base - 8192:base - 8191]  # as the first column of their workgroup
    g, h, w = g.to(DEV), h.to(DEV), w.to(DEV)
    gx, gw = int8.rms_norm_backward(g, h, w)
    first = slice(base - 8192, base - 8191)
    assert torch.equal(gx[:, last], gx[:, first].expand_as(gx[:, last]))
    assert torch.equal(gw[last], gw[first].expand_as(gw[last]))
    for _ in range(3):
        again = int8.rms_norm_backward(g, h, w)
        assert torch.equal(gx, again[0]) and torch.equal(gw, again[1])


def test_second_derivatives_are_refused():
    x, w = (torch.randn(8, 16, generator=_gen(s)).to(DEV).requires_grad_() for s in (1, 2))
    nw = torch.ones(16, device=DEV)
    for y in (tgt.int8_linear_gpu(x, w), tgt.rms_norm_int8_linear_gpu(x, None, nw, w)[0]):
        grad, = torch.autograd.grad(y.sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="no second derivatives"):
            (y.sum() + grad.square().sum()).backward()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("m,n,k", [(2100, 296, 1030), (296, 2100, 1030), (1000, 72, 4096), (520, 4008, 1024), (70, 90, 100),
                                   (300, 2100, 1030)], ids=lambda v: str(v))
def test_infinite_scales_make_infinite_gradients(dtype, m, n, k):
    """Where no term is zero, an infinite scale's term decides the sign, also in a
    sum whose length is no whole number of steps."""
    g = torch.rand(m, n, generator=_gen(1)) + 0.5
    a, b = (torch.randint(1, 128, (r, k), generator=_gen(r)).to(torch.int8) for r in (m, n))
    for at in (0, -1, -3, -9):
        _say("infinite scale", IDS[dtype], m, n, k, at)
        sa, sb = torch.full((m,), 0.01), torch.full((n,), 0.01)
        sa[at] = sb[at] = float("inf")
        g2, a2, b2 = g.clone(), a.clone(), b.clone()
        g2[::2, at] *= -1
        g2[at] *= -1
        b2[at, ::3] *= -1
        a2[at, ::3] *= -1
        g2, a2, b2 = g2.to(dtype).to(DEV), a2.to(DEV), b2.to(DEV)
        got = int8.backward_a(g2, b2, sb.to(DEV))
        want = torch.sign(g2[:, at].float())[:, None] * torch.sign(b2[at].float()) * float("inf")
        assert torch.equal(got.float(), want)
        got = int8.backward_b(g2, a2, sa.to(DEV))
        want = torch.sign(g2[at].float())[:, None] * torch.sign(a2[at].float()) * float("inf")
        assert torch.equal(got.float(), want)


def _huge_rows(seed, rows, cols, dtype):
    """Rows of ordinary values, of values whose squares pass f32, and of one such
    value among ordinary ones, in turn."""
    x = torch.randn(rows, cols, generator=_gen(seed))
    x[1::4] *= 1e19
    x[2::4] *= 5e36
    x[3::4, cols // 2] = 3e20
    return x.to(dtype)


HUGE = [(6, 1), (9, 7), (9, 8), (33, 300), (10, 513), (21, 1025), (21, 2051), (10, 3081), (10, 4096), (10, 6145), (10, 8192),
        (5, 8200), (5, 20011)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=IDS.get)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,cols", HUGE, ids=lambda v: str(v))
def test_norm_of_huge_rows(dtype, residual, rows, cols):
    """q within half a step (and f32's rounding of it), scales within 1e-5: f32 sums
    of squares, as for ordinary rows."""
    _say("norm of huge rows", IDS[dtype], rows, cols, residual)
    x = _huge_rows(cols, rows, cols, dtype)
    r = _huge_rows(cols + 1, rows, cols, dtype) if residual else None
    w = (1 + 0.3 * torch.randn(cols, generator=_gen(3))).to(dtype)
    q, scale, h = int8.rms_norm(x.to(DEV), w.to(DEV), None if r is None else r.to(DEV), 1e-5)
    h64 = h.cpu().double()
    assert torch.isfinite(h64).all()
    want = h64 * ((h64 * h64).mean(1, keepdim=True) + 1e-5).rsqrt() * w.double()
    step = want.abs().amax(1, keepdim=True) / 127
    assert ((scale.cpu().double()[:, None] - step).abs() <= 1e-5 * step).all()
    assert ((q.cpu().double() * step - want).abs() <= step * (0.5 + 127 * 4 * 2.0 ** -24 + 1e-9)).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=IDS.get)
@pytest.mark.parametrize("rows,cols", HUGE + [(1600, 264), (1025, 520), (1100, 4099), (600, 8195)], ids=lambda v: str(v))
def test_norm_backward_of_huge_rows(dtype, rows, cols):
    """Within 2e-5 of the magnitudes added, as for ordinary rows, then one rounding;
    numbers below f32's normal ones within their last bit.  More rows than
    workgroups, too."""
    _say("norm backward of huge rows", IDS[dtype], rows, cols)
    g = (torch.randn(rows, cols, generator=_gen(1)) * torch.exp(torch.randn(rows, 1, generator=_gen(2)))).to(dtype)
    h = _huge_rows(cols, rows, cols, dtype)
    w = (1 + 0.3 * torch.randn(cols, generator=_gen(3))).to(dtype)
    gx, gw = int8.rms_norm_backward(g.to(DEV), h.to(DEV), w.to(DEV), 1e-5)
    g64, h64, w64 = g.double(), h.double(), w.double()
    rstd = ((h64 * h64).mean(1, keepdim=True) + 1e-5).rsqrt()
    xh, u = h64 * rstd, g64 * w64
    want = rstd * (u - xh * (u * xh).mean(1, keepdim=True))
    size = rstd * (u.abs() + xh.abs() * (u * xh).abs().mean(1, keepdim=True))
    unit = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    least = 2.0 ** -133 if dtype == torch.bfloat16 else 2.0 ** -148
    assert ((gx.cpu().double() - want).abs() <= unit * want.abs() + 2e-5 * size + least).all()
    want, size = (g64 * xh).sum(0), (g64 * xh).abs().sum(0)
    again = int8.rms_norm_backward(g.to(DEV), h.to(DEV), w.to(DEV), 1e-5)
    assert torch.equal(gx, again[0]) and torch.equal(gw, again[1])
    assert ((gw.cpu().double() - want).abs() <= unit * want.abs() + 2e-5 * size).all()


F16_RANGES = [(64, 96, 80), (70, 90, 100), (300, 200, 264), (2100, 296, 1030), (296, 2100, 1030), (520, 4008, 1024),
              (5000, 40, 72)]


def _check_f16(got, g, x):
    """Each term's factor rounded once (2^-11 of it) and f32 sums, then one rounding;
    the 2-norm within 1.2 * 2^-11, as for the ordinary gradients."""
    want, size = g @ x, g.abs() @ x.abs()
    fine = want.abs() < 6e4
    off = (got.cpu().double() - want)[fine]
    u = 2.0 ** -11
    assert fine.any() and torch.isfinite(got.cpu()[fine]).all()
    assert (off.abs() <= ((1.01 * u + g.shape[1] * 2.0 ** -24) * size + u * want.abs())[fine] + 2.0 ** -24).all()
    assert off.norm() <= 1.2 * u * want[fine].norm() + 2.0 ** -24 * off.numel() ** 0.5


@pytest.mark.parametrize("m,n,k", F16_RANGES, ids=lambda v: str(v))
@pytest.mark.parametrize("spread", [-100, -40, -19, 15, 19, 21, 30, 36, 60, 100])
def test_f16_gradients_beside_a_scale_far_from_the_others(m, n, k, spread):
    """One scale 2^spread times the others; a large one meets a gradient of zero, or
    integers of zero (a padded position that holds anything)."""
    g = torch.randn(m, n, generator=_gen(1)).half()
    a, b = (torch.randint(-127, 128, (r, k), generator=_gen(r)).to(torch.int8) for r in (m, n))
    sa, sb = (torch.rand(r, generator=_gen(r + 1)) * 0.02 + 1e-3 for r in (m, n))
    sa[3] *= 2.0 ** spread
    sb[3] *= 2.0 ** spread
    for zero in ("gradient", "integers"):
        _say("f16 range", m, n, k, spread, zero)
        ga, gb, a2, b2 = g.clone(), g.clone(), a.clone(), b.clone()
        if zero == "gradient":
            ga[:, 3], gb[3] = 0, 0
        else:
            a2[3], b2[3] = 0, 0
        f64 = lambda q, s: q.double() * s.double()[:, None]  # noqa: E731
        _check_f16(int8.backward_a(ga.to(DEV), b2.to(DEV), sb.to(DEV)), ga.double(), f64(b2, sb))
        _check_f16(int8.backward_b(gb.to(DEV), a2.to(DEV), sa.to(DEV)), gb.double().t(), f64(a2, sa))


@pytest.mark.parametrize("m,n,k", F16_RANGES, ids=lambda v: str(v))
def test_f16_gradients_of_terms_of_one_size_from_scales_of_many(m, n, k):
    """Scales over 2^24 with gradients that make up for them: every term counts."""
    _say("f16 balanced", m, n, k)
    a, b = (torch.randint(-127, 128, (r, k), generator=_gen(r)).to(torch.int8) for r in (m, n))
    ea, eb = (torch.randint(-12, 13, (r,), generator=_gen(r + 1)).double() for r in (m, n))
    sa, sb = (0.01 * 2.0 ** -ea).float(), (0.01 * 2.0 ** -eb).float()
    g = torch.randn(m, n, generator=_gen(1)).double()
    ga, gb = (g * 2.0 ** eb).half(), (g * 2.0 ** ea[:, None]).half()
    f64 = lambda q, s: q.double() * s.double()[:, None]  # noqa: E731
    _check_f16(int8.backward_a(ga.to(DEV), b.to(DEV), sb.to(DEV)), ga.double(), f64(b, sb))
    _check_f16(int8.backward_b(gb.to(DEV), a.to(DEV), sa.to(DEV)), gb.double().t(), f64(a, sa))


@pytest.mark.parametrize("n", [(1 << 26) - 16, (1 << 26) - 15, (1 << 26) - 1])
def test_one_row_times_the_most_columns(n):
    """Both sides of the limit of one launch for few rows."""
    _say("matmul", 1, n, 16)
    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    b = torch.randint(-127, 128, (n, 16), generator=g, device=DEV, dtype=torch.int8)
    a = torch.randint(-127, 128, (1, 16), generator=g, device=DEV, dtype=torch.int8)
    sb = torch.rand(n, generator=g, device=DEV)
    c = int8.matmul(a, torch.full((1,), 0.5, device=DEV), b, sb, dtype=torch.float32)
    want = (b.float() * a.float()).sum(1) * 0.5 * sb  # whole numbers below 2^24
    assert torch.equal(c[0], want)


def _rel(a, b):
    return ((a.detach().cpu().double() - b).norm() / b.norm()).item()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=IDS.get)
@pytest.mark.parametrize("m,n,k", [(70, 130, 257), (300, 256, 512), (1100, 520, 1030)], ids=lambda v: str(v))
def test_linear_gradients_in_16_bits(dtype, m, n, k):
    """y: one rounding of every value, u.  Gradients: one of every value and one of
    every factor, 1.2 u in the 2-norm as for the operators alone."""
    u = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    x, w, g = (torch.randn(*s, generator=_gen(i)).to(dtype).to(DEV) for i, s in enumerate(((m, k), (n, k), (m, n))))
    x.requires_grad_()
    w.requires_grad_()
    y = tgt.int8_linear_gpu(x, w)
    y.backward(g)
    f64 = lambda q, s: q.cpu().double() * s.cpu().double()[:, None]  # noqa: E731
    xr, wr = f64(*int8.quantize(x.detach())), f64(*int8.quantize(w.detach()))
    g64 = g.cpu().double()
    assert y.dtype == x.grad.dtype == w.grad.dtype == dtype
    assert _rel(y, xr @ wr.t()) < 1.01 * u
    assert _rel(x.grad, g64 @ wr) < 1.2 * u
    assert _rel(w.grad, g64.t() @ xr) < 1.2 * u


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=IDS.get)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("m,n,k", [(130, 96, 300), (700, 512, 1024)], ids=lambda v: str(v))
def test_norm_linear_gradients_in_16_bits(dtype, residual, m, n, k):
    """As above, with the product's gradient rounded (1.2 u) before the norm's
    backward pass, which is linear in it and stretches it by at most the largest
    weight, 1.5, and its result rounded (u): less than 3 u.  The stream is what
    is stored of it."""
    u = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    shapes = ((m, k), (m, k), (k,), (n, k), (m, n), (m, k))
    x, r, nw, w, gy, gh = (torch.randn(*s, generator=_gen(i)) for i, s in enumerate(shapes))
    x, r, nw, w, gy, gh = (t.to(dtype) for t in (x, r, 1 + 0.1 * nw, w, gy, gh))
    ours = [t.to(DEV).requires_grad_() for t in (x, r, nw, w)]
    if not residual:
        ours[1] = None
    y, h = tgt.rms_norm_int8_linear_gpu(*ours, 1e-5)
    torch.autograd.backward([y, h], [gy.to(DEV), gh.to(DEV)])

    ref = [t.double().requires_grad_() for t in (x, r, nw, w)]
    h64 = ref[0] + ref[1] if residual else ref[0] * 1.0
    h64 = h64 + (h.detach().cpu().double() - h64).detach()
    norm = h64 * (h64.square().mean(1, keepdim=True) + 1e-5).rsqrt() * ref[2]
    f64 = lambda q, s: q.cpu().double() * s.cpu().double()[:, None]  # noqa: E731
    rows = f64(*int8.rms_norm(h.detach(), nw.to(DEV), None, 1e-5)[:2])
    wr = f64(*int8.quantize(w.to(DEV)))
    y64 = (norm + (rows - norm).detach()) @ (ref[3] + (wr - ref[3]).detach()).t()
    torch.autograd.backward([y64, h64], [gy.double(), gh.double()])
    assert _rel(y, y64.detach()) < 1.01 * u
    for a, b in zip(ours, ref):
        if a is not None:
            assert a.grad.dtype == dtype and _rel(a.grad, b.grad) < 3 * u


@pytest.mark.parametrize("m,n,k", [(64, 8191, 64), (8192, 64, 64), (1000, 1003, 5), (2048, 2048, 512), (2048, 2049, 2050),
                                   (4096, 4100, 520), (4096, 1024, 4096)], ids=lambda v: str(v))
@pytest.mark.parametrize("spread", [10, 40])
def test_f16_gradients_in_every_tile_size(m, n, k, spread):
    """As above, in slices, in larger tiles, in place and laid out; a gradient past
    its scale's row is zero.  The 64-bit products are torch's on the GPU."""
    _say("f16 tiles", m, n, k, spread)
    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    grad = torch.randn(m, n, generator=g, device=DEV).half()
    a, b = (torch.randint(-127, 128, (r, k), generator=g, device=DEV).to(torch.int8) for r in (m, n))
    sa, sb = (torch.rand(r, generator=g, device=DEV) * 0.02 + 1e-3 for r in (m, n))
    sa[3] *= 2.0 ** spread
    sb[3] *= 2.0 ** spread
    grad[3], grad[:, 3] = 0, 0
    f64 = lambda q, s: q.double() * s.double()[:, None]  # noqa: E731
    u = 2.0 ** -11
    for got, x, y in ((int8.backward_a(grad, b, sb), grad.double(), f64(b, sb)),
                      (int8.backward_b(grad, a, sa), grad.double().t().contiguous(), f64(a, sa))):
        want, size = torch.mm(x, y), torch.mm(x.abs(), y.abs())
        off = got.double() - want
        assert (off.abs() <= (1.01 * u + x.shape[1] * 2.0 ** -24) * size + u * want.abs() + 2.0 ** -24).all()
        assert off.norm() <= 1.2 * u * want.norm() + 2.0 ** -24 * off.numel() ** 0.5


@pytest.mark.parametrize("m,n,k", [(100, 96, 80), (520, 4008, 1024)], ids=lambda v: str(v))
def test_f16_gradients_in_a_graph_follow_their_scales(m, n, k):
    """Replays with scales of one size and far from each other, in turn."""
    _say("f16 graph", m, n, k)
    grad = torch.randn(m, n, generator=_gen(1)).half().to(DEV)
    a, b = (torch.randint(-127, 128, (r, k), generator=_gen(r)).to(torch.int8).to(DEV) for r in (m, n))
    sa, sb = (torch.rand(r, generator=_gen(r + 1)).to(DEV) * 0.02 + 1e-3 for r in (m, n))
    grad[3], grad[:, 3] = 0, 0
    step = lambda: (int8.backward_a(grad, b, sb), int8.backward_b(grad, a, sa))  # noqa: E731
    first = step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(5):
        sa[3] = sb[3] = 1e9 if i % 2 else 0.01
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        for u, v, w in zip(got, step(), first):
            assert torch.equal(u, v)
            assert (u.float() - w.float()).norm() <= 2.0 ** -9 * w.float().norm()
