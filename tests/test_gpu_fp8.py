"""The operators of the layer in 8-bit floating point against their definitions
in 64 bits, on the CPU.

Tolerances, with u the unit roundoff of the output's type (2^-24, 2^-11, 2^-8
for f32, f16, bf16):

* quantize, dequantize: exact (the scale is a power of two, the rounding is
  defined to the last bit).
* matmul to f32, and gradients: products are exact; each addition of a sum of r
  terms is off by at most one step of f32 at its result (2^-23; matrix instructions
  need not round to nearest), and no partial sum passes the magnitudes' sum S, so
  the sum is off by r * 2^-23 * S at most; a bias is one more addition, then u.
* matmul to 16 bits: the matrix instructions add groups of at most eight products
  first, each cut to a multiple of 2^-13 of the largest one's power of two, which
  is at most the group's part of S: 8 * 2^-13 * S more at most.
"""
import pytest
import torch

from tropical_gemm import _native as nat
from tropical_gemm import fp8

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}
TYPES = [torch.bfloat16, torch.float16, torch.float32]
IDS = {torch.bfloat16: "bf16", torch.float16: "f16", torch.float32: "f32"}
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _say(*what):
    print("[case]", *what, flush=True)


def _blocks(n):
    return -(-n // 128)


def _gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def _strided(v, ld=None, offset=0):
    """v on the GPU, its rows ld apart and `offset` elements into their storage,
    which holds NaNs elsewhere."""
    rows, cols = v.shape
    ld = cols if ld is None else ld
    nan = 0x7f if v.dtype is E4M3 else None
    n = offset + max(rows, 1) * ld + 16
    store = torch.full((n,), nan, dtype=torch.uint8, device=DEV).view(E4M3) if nan else torch.full((n,), float("nan"), dtype=v.dtype, device=DEV)
    out = store[offset:].as_strided((rows, cols), (ld, 1))
    if nan:
        out.view(torch.uint8).copy_(v.view(torch.uint8))
    else:
        out.copy_(v)
    return out


def _e4m3(seed, rows, cols):
    """Every finite e4m3 number, at random."""
    b = torch.randint(0, 256, (rows, cols), generator=_gen(seed), dtype=torch.int32)
    b = torch.where((b & 127) == 127, b - 1, b)
    return b.to(torch.uint8).view(E4M3)


def _scales(seed, rows, cols, lo=118, hi=132):
    return torch.randint(lo, hi, (rows, cols), generator=_gen(seed), dtype=torch.int32).to(torch.uint8)


def _laid(s, order):
    """Scales on the GPU in some memory order."""
    rows, cols = s.shape
    if order == "columns":
        t = s.t().contiguous().t()
    elif order == "rows":
        t = s.contiguous()
    else:  # a part of a larger one
        big = torch.full((rows + 3, cols + 2), 255, dtype=torch.uint8).t().contiguous().t()
        big[2:2 + rows, 1:1 + cols] = s
        return big.to(DEV)[2:2 + rows, 1:1 + cols].view(E8M0)
    return torch.empty_strided(t.shape, t.stride(), dtype=torch.uint8, device=DEV).copy_(t).view(E8M0)


def _exact(q, s, br):
    """The numbers that CPU bytes and scales stand for, in f64."""
    rows, cols = q.shape
    f = torch.pow(2.0, s.double() - 127)
    return q.float().double() * f.repeat_interleave(br, 0)[:rows].repeat_interleave(128, 1)[:, :cols]


def _close(got, want, bound, dtype):
    got = got.cpu().double()
    assert torch.isfinite(want).all() and got.shape == want.shape
    d = (got - want).abs()
    most = bound + U[dtype] * (want.abs() + bound) + LEAST[dtype]
    # What the type does not hold is infinite; near its end it may be.
    end = torch.finfo(dtype).max
    inf = torch.isinf(got) & (got.sign() == want.sign()) & (want.abs() + most > end)
    assert (inf | (d <= most)).all(), (d - most)[~inf].max()


# ---- blocks ----------------------------------------------------------------


def _quantized(x, br):
    """q (bytes) and scale (bytes) of the definition."""
    rows, cols = x.shape
    rb, cb = -(-rows // br), _blocks(cols)
    full = torch.zeros(rb * br, cb * 128, dtype=torch.float64)
    full[:rows, :cols] = x.double()
    blocks = full.view(rb, br, cb, 128)
    top = blocks.abs().amax((1, 3))
    e = torch.full(top.shape, -100, dtype=torch.int64)
    while True:
        more = top > 448 * torch.pow(2.0, e.double())
        if not more.any():
            break
        e += more.long()
    v = blocks / torch.pow(2.0, e.double())[:, None, :, None]
    q = v.float().to(E4M3).view(torch.uint8)  # exact in f32: a power of two
    return q.reshape(rb * br, cb * 128)[:rows, :cols], (e + 127).to(torch.uint8)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("br", [1, 128])
@pytest.mark.parametrize("rows,cols,ld,offset", [
    (1, 1, 1, 0), (1, 128, 128, 0), (3, 7, 7, 1), (128, 129, 129, 0), (129, 127, 140, 3), (130, 1000, 1003, 5),
    (257, 384, 384, 0), (5, 4099, 4099, 0), (1000, 8, 8, 0)])
def test_quantize(dtype, br, rows, cols, ld, offset):
    _say("quantize", dtype, br, rows, cols, ld, offset)
    g = _gen(rows * cols + br)
    x = torch.randn(rows, cols, generator=g) * torch.exp2(torch.randint(-20, 12, (rows, 1), generator=g).float())
    x = x.to(dtype)
    if rows > 2:
        x[1] = 0
    xs = _strided(x, ld, offset)
    q, s = fp8.quantize(xs, br)
    wq, ws = _quantized(x, br)
    assert q.dtype is E4M3 and s.dtype is E8M0
    assert torch.equal(s.cpu().view(torch.uint8), ws)
    got, zero = q.cpu().view(torch.uint8), (wq & 127) == 0
    assert torch.equal(torch.where(zero, 0, got & (127 + 128 * (~zero))), torch.where(zero, 0, wq))
    want = _exact(q.cpu(), ws, br)
    for out in TYPES:
        y = fp8.dequantize(q, s, out)
        assert torch.equal(y.cpu(), want.float().to(out)) and y.dtype is out


def test_quantize_every_number():
    """Every number between two neighbours of e4m3 and every tie, at every
    exponent of a scale that f32 has, and the borders of the scale's choice."""
    for e in (-100, -99, -9, 0, 1, 60, 119):
        v = torch.arange(0, 448 * 2 + 1, dtype=torch.float64) / 2  # multiples of 1/2: all ties above 8
        v = torch.cat([v, torch.arange(0, 1024, dtype=torch.float64) * 2.0 ** -11, -v])
        n = _blocks(v.numel()) * 128
        x = torch.full((n + 127 * (n // 127 + 1),), 448.0, dtype=torch.float64)[:n]
        x[:v.numel()] = v
        x = x.view(-1, 1).repeat(1, 2)
        x[:, 1] = 448.0  # the block's top
        x = (x * 2.0 ** e).float()
        q, s = fp8.quantize(x.to(DEV))
        wq, ws = _quantized(x, 1)
        assert torch.equal(s.cpu().view(torch.uint8), ws) and (ws == e + 127).all()
        assert torch.equal(q.cpu().float(), wq.view(E4M3).float()), e
    # One past 448 takes the next power of two; below 448 * 2^-100 nothing smaller is taken.
    x = torch.tensor([[448.0], [448.00003], [896.0], [2.0 ** -95], [2.0 ** -120], [0.0]], device=DEV)
    q, s = fp8.quantize(x)
    assert s.cpu().view(torch.uint8)[:, 0].tolist() == [127, 128, 128, 27, 27, 27]
    assert fp8.dequantize(q, s, torch.float32)[:, 0].tolist() == [448.0, 448.0, 896.0, 2.0 ** -95, 0.0, 0.0]


@pytest.mark.parametrize("br", [1, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_quantize_not_finite(br, bad):
    x = torch.randn(200, 300)
    x[3, 130] = bad
    q, s = fp8.quantize(x.to(DEV), br)
    y = fp8.dequantize(q, s, torch.float32).cpu()
    hit = torch.zeros(200, 300, dtype=torch.bool)
    hit[3:4 if br == 1 else 128, 128:256] = True
    if br == 128:
        hit[:128, 128:256] = True
    assert torch.isnan(y[hit]).all() and torch.isfinite(y[~hit]).all()
    # Products of it are NaN where the definition's are.
    w, sw = fp8.quantize(torch.randn(70, 300).to(DEV), 128)
    if br == 1:
        for rows in (16, 200):
            c = fp8.matmul(q[:rows].contiguous(), s[:rows], w, sw, dtype=torch.float32).cpu()
            assert torch.isnan(c[3]).all() and torch.isfinite(c[:3]).all() and torch.isfinite(c[4:]).all()


# ---- product ---------------------------------------------------------------

SIZES = [
    # Few rows: each form of the streamed product, whole and partial blocks.
    (1, 1, 1), (1, 16, 128), (1, 17, 129), (2, 100, 2048), (16, 127, 1000), (17, 130, 256), (32, 1000, 4099),
    (33, 129, 127), (48, 65, 640), (49, 300, 333), (64, 128, 2048),
    # Tiles: edges on every side, partial last blocks, slices, several tile forms.
    (65, 63, 128), (64, 64, 16), (100, 200, 144), (128, 128, 1024), (129, 257, 1040), (200, 300, 4096),
    (256, 256, 8192), (300, 130, 999), (513, 700, 272), (1000, 1100, 400),
]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_matmul(dtype, m, n, k):
    pick = (m + n + k) % 3
    lda, offa, ldb, offb = [(k, 0, k, 0), (k + 5, 3, k + 16, 0), (k + 16, 16, k + 1, 1)][pick]
    _say("matmul", dtype, m, n, k, pick)
    a, b = _e4m3(m + k, m, k), _e4m3(n + k, n, k)
    sa, sb = _scales(m, m, _blocks(k)), _scales(n, _blocks(n), _blocks(k))
    bias = torch.randn(n, generator=_gen(n)).to(dtype) if (m + n) % 2 else None
    c = fp8.matmul(_strided(a, lda, offa), _laid(sa, ["columns", "rows", "part"][pick]), _strided(b, ldb, offb),
                   _laid(sb, ["part", "columns", "rows"][pick]), None if bias is None else bias.to(DEV), dtype)
    da, db = _exact(a, sa, 1), _exact(b, sb, 128)
    want, size = da @ db.t(), da.abs() @ db.abs().t()
    if bias is not None:
        want, size = want + bias.double(), size + bias.double().abs()
    _close(c, want, ((k + 1) * 2.0 ** -23 + (dtype is not torch.float32) * 2.0 ** -10) * size, dtype)


@pytest.mark.parametrize("m,n,k", [(3, 100, 2048), (40, 129, 999), (200, 300, 1040), (513, 700, 272)])
def test_matmul_f16_in_range(m, n, k):
    """The same with scales that keep the sums inside f16."""
    a, b = _e4m3(m + k, m, k), _e4m3(n + k, n, k)
    sa, sb = _scales(m, m, _blocks(k), 112, 116), _scales(n, _blocks(n), _blocks(k), 118, 122)
    da, db = _exact(a, sa, 1), _exact(b, sb, 128)
    want, size = da @ db.t(), da.abs() @ db.abs().t()
    assert size.max() < 60000
    c = fp8.matmul(a.to(DEV), _laid(sa, "columns"), b.to(DEV), _laid(sb, "columns"), dtype=torch.float16)
    _close(c, want, (k * 2.0 ** -23 + 2.0 ** -10) * size, torch.float16)
    # In the mean the instructions' own rounding is far below f16's (1.5e-5 and 2e-4).
    assert (c.cpu().double() - want).norm() <= 3e-4 * want.norm()


@pytest.mark.parametrize("form", ["tiles 256x256", "tiles 128x256", "tiles 128x128", "tiles 128x64 halves",
                                  "tiles 64x64", "tiles 64x64 halves"])
def test_every_tile(form):
    """Each tile form is the plan of some product, whole and with edges."""
    found = 0
    for m, n, k in [(8192, 8192, 128), (8192 - 5, 4096 + 3, 144), (1500, 1400, 256), (1111, 1500, 384),
                    (4096, 1024, 512), (300, 256, 512), (2048, 2048, 144), (700, 900, 272), (5000, 6000, 128),
                    (4096, 4096, 2048), (4096 - 5, 4096 + 3, 1040), (8192, 4096, 1024), (2053, 4099, 4112),
                    (100, 1000, 4096), (129, 1033, 4240), (250, 8192, 4096), (131, 8190, 8080), (2048, 4096, 2048),
                    (2047, 4090, 2064), (3500, 6000, 1024), (2048, 2560, 4096), (2041, 2563, 4112)]:
        plan = nat.load().tg_f8_gemm_plan(1, 256, k, 256, k, m, n, k).decode()
        if plan.split(" slices")[0] != form:
            continue
        found += 1
        _say(plan, m, n, k)
        a, b = _e4m3(m, m, k), _e4m3(n, n, k)
        sa, sb = _scales(1, m, _blocks(k)), _scales(2, _blocks(n), _blocks(k))
        c = fp8.matmul(a.to(DEV), _laid(sa, "columns"), b.to(DEV), _laid(sb, "columns"), dtype=torch.bfloat16)
        da, db = _exact(a, sa, 1).to(DEV), _exact(b, sb, 128).to(DEV)
        want, size = torch.mm(da, db.t()), torch.mm(da.abs(), db.abs().t())
        assert ((c.double() - want).abs() <= ((k + 1) * 2.0 ** -23 + 2.0 ** -10) * size * (1 + 2.0 ** -8) + 2.0 ** -8 * want.abs()).all()
    assert found >= 1, form


def test_matmul_empty():
    q = lambda r, k: (torch.zeros(r, k, dtype=torch.uint8, device=DEV).view(E4M3),)
    s = lambda r, k: torch.full((r, _blocks(k)), 127, dtype=torch.uint8, device=DEV).view(E8M0)
    bias = torch.arange(5.0, device=DEV)
    c = fp8.matmul(*q(3, 0), s(3, 0), *q(5, 0), s(1, 0), bias, torch.float32)
    assert torch.equal(c, bias.expand(3, 5))
    assert fp8.matmul(*q(0, 8), s(0, 8), *q(5, 8), s(1, 8)).shape == (0, 5)
    assert fp8.matmul(*q(4, 8), s(4, 8), *q(0, 8), s(0, 8)).shape == (4, 0)
    x, t = fp8.quantize(torch.empty(0, 300, device=DEV))
    assert x.shape == (0, 300) and t.shape == (0, 3) and fp8.dequantize(x, t).shape == (0, 300)
    g = torch.zeros(0, 5, device=DEV)
    assert fp8.backward_a(g, *q(5, 8), s(1, 8)).shape == (0, 8)
    assert torch.equal(fp8.backward_b(g, *q(0, 8), s(0, 8)), torch.zeros(5, 8, device=DEV))


@pytest.mark.parametrize("m", [5, 70])
def test_scale_range(m):
    """Scales at both ends of what sums in f32 hold, and the NaN scale."""
    n, k = 66, 256
    a, b = torch.full((m, k), 0x38, dtype=torch.uint8).view(E4M3), torch.full((n, k), 0x38, dtype=torch.uint8).view(E4M3)
    for ea, eb in [(-100, 0), (100, -100), (60, 60), (-60, -60), (0, 0)]:
        sa = torch.full((m, 2), 127 + ea, dtype=torch.uint8)
        sb = torch.full((1, 2), 127 + eb, dtype=torch.uint8)
        c = fp8.matmul(a.to(DEV), sa.to(DEV).view(E8M0), b.to(DEV), sb.to(DEV).view(E8M0), dtype=torch.float32)
        # 256 * 2^120 = 2^128 lies beyond f32: infinite.
        assert (c.cpu() == torch.tensor(k * 2.0 ** (ea + eb), dtype=torch.float64).float()).all(), (ea, eb)
    sa[2, 1] = 255
    c = fp8.matmul(a.to(DEV), sa.to(DEV).view(E8M0), b.to(DEV), sb.to(DEV).view(E8M0), dtype=torch.float32).cpu()
    assert torch.isnan(c[2]).all() and torch.isfinite(c[:2]).all() and torch.isfinite(c[3:]).all()


# ---- gradients ---------------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (3, 130, 129), (65, 64, 128), (130, 70, 300), (64, 257, 16),
                                   (300, 200, 1000), (513, 129, 260), (1000, 1030, 520), (9, 8, 8), (7, 300, 200),
                                   (2100, 1500, 136), (700, 2300, 1100)])
def test_gradients(dtype, m, n, k):
    _say("gradients", dtype, m, n, k)
    a, b = _e4m3(m + k, m, k), _e4m3(n + k, n, k)
    sa, sb = _scales(m, m, _blocks(k)), _scales(n, _blocks(n), _blocks(k))
    g = (torch.randn(m, n, generator=_gen(m)) * torch.exp(torch.randn(m, 1, generator=_gen(n)))).to(dtype)
    odd = (m + n) % 2
    gs = _strided(g, n + 3 * odd, odd)
    da, db, g64 = _exact(a, sa, 1), _exact(b, sb, 128), g.double()
    ga = fp8.backward_a(gs, _strided(b, k + odd, odd), _laid(sb, "rows" if odd else "columns"))
    _close(ga, g64 @ db, n * 3 * 2.0 ** -23 * (g64.abs() @ db.abs()), dtype)
    gb = fp8.backward_b(gs, _strided(a, k + odd, odd), _laid(sa, "part" if odd else "columns"))
    _close(gb, g64.t() @ da, m * 3 * 2.0 ** -23 * (g64.t().abs() @ da.abs()), dtype)


def test_gradients_exact_products():
    """Gradients of one term are exact products, rounded once: f16 and f32 keep
    all their bits."""
    for dtype in TYPES:
        g = torch.randn(70, 1, generator=_gen(3)).to(dtype)
        b, sb = _e4m3(4, 1, 300), _scales(5, 1, 3, 100, 127)
        ga = fp8.backward_a(g.to(DEV), b.to(DEV), _laid(sb, "rows"))
        want = g.double() @ _exact(b, sb, 128)
        least = 2.0 ** -24 if dtype is torch.float16 else 0
        assert ((ga.cpu().double() - want).abs() <= U[dtype] * want.abs() + least / 2 + (2.0 ** -23 * 2) * want.abs() * (dtype is torch.float32)).all()


# ---- how calls are made ------------------------------------------------------


def _product(m, n, k, dtype=torch.bfloat16):
    x = torch.randn(m, k, generator=_gen(m)).to(dtype).to(DEV)
    w = torch.randn(n, k, generator=_gen(n)).to(dtype).to(DEV)
    g = torch.randn(m, n, generator=_gen(k)).to(dtype).to(DEV)
    return x, w, g


def _all(x, w, g):
    q, s = fp8.quantize(x)
    qw, sw = fp8.quantize(w, 128)
    return [fp8.dequantize(q, s, x.dtype), fp8.matmul(q, s, qw, sw, dtype=x.dtype), fp8.backward_a(g, qw, sw),
            fp8.backward_b(g, q, s)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("m,n,k", [(5, 300, 512), (200, 260, 333)])
def test_graph(dtype, m, n, k):
    """A captured run, replayed with other inputs and eager work between."""
    x, w, g = _product(m, n, k, dtype)
    _all(x, w, g)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _all(x, w, g)
    for turn in range(3):
        x.copy_(torch.randn(m, k, generator=_gen(turn)).to(dtype))
        want = _all(x, w, g)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), turn


def test_streams_and_repeats():
    """Two streams at once, and equal calls give equal bits."""
    x, w, g = _product(300, 520, 700)
    want = _all(x, w, g)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for turn in range(4):
        with torch.cuda.stream(streams[turn % 2]):
            got.append(_all(x, w, g))
    torch.cuda.synchronize()
    for outs in got:
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_outputs_stay_inside():
    """Nothing is written before or behind an output."""
    lib = nat.load()
    for m, n, k in [(5, 33, 130), (70, 75, 144), (300, 259, 256), (513, 261, 128)]:
        a, b = _e4m3(1, m, k).to(DEV), _e4m3(2, n, k).to(DEV)
        sa, sb = _laid(_scales(1, m, _blocks(k)), "columns"), _laid(_scales(2, _blocks(n), _blocks(k)), "columns")
        store = torch.full((m * n + 128,), 7.0, dtype=torch.bfloat16, device=DEV)
        out = store[63:63 + m * n]
        need = lib.tg_f8_gemm_workspace_size(1, a.data_ptr(), k, b.data_ptr(), k, m, n, k)
        ws = torch.full((max(need, 1) + 256,), 77, dtype=torch.uint8, device=DEV)
        nat.check(lib.tg_f8_gemm(0, 1, a.data_ptr(), k, sa.data_ptr(), *sa.stride(), b.data_ptr(), k, sb.data_ptr(),
                                 *sb.stride(), None, out.data_ptr(), m, n, k, ws.data_ptr(), need,
                                 torch.cuda.current_stream().cuda_stream))
        torch.cuda.synchronize()
        assert torch.equal(out.view(m, n), fp8.matmul(a, sa, b, sb))
        assert (store[:63] == 7).all() and (store[63 + m * n:] == 7).all() and (ws[need:] == 77).all()
