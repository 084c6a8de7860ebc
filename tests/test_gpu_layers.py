"""Layer norm and dropout against their definitions in 64 bits, on the CPU.

Which elements are dropped is compared exactly, with a generator written in
numpy.  Tolerances, with u the unit roundoff of the type and e = 2^-24:

* dropout: one product and one sum in f32, 2e of their magnitudes, then u.
* mean: sums in f32 of fewer than 300 terms in a row, 300e of the mean magnitude.
* rstd: the variance's sum likewise, 300e, and the mean's error squared; the
  square root halves both: 1e-5, where deviations are not below a thousandth of
  the mean (they are not here).
* y: (h - mean) is off by the mean's error and e of itself, rstd by 1e-5, then
  three roundings: 2e-5 of |(h - mean) rstd w| plus 300e * mean|h| rstd |w| plus e
  of the bias, then u.
* gradients: 2e-5 of the sum of the magnitudes added, then u.
"""
import numpy as np
import pytest
import torch

from tropical_gemm import _native as nat
from tropical_gemm import layers

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


def _strided(v, ld=None, offset=0):
    rows, cols = v.shape
    ld = cols if ld is None else ld
    store = torch.full((offset + max(rows, 1) * ld + 16,), float("nan"), dtype=v.dtype, device=DEV)
    out = store[offset:].as_strided((rows, cols), (ld, 1))
    out.copy_(v)
    return out


def _factors(rows, cols, p, seed, offset, first_row=0):
    """Dropout's factor of each element, in f64."""
    c = [np.zeros((rows, -(-cols // 8)), dtype=np.uint64) for _ in range(4)]
    c[0] += np.arange(c[0].shape[1], dtype=np.uint64)
    c[1] += np.arange(first_row, first_row + rows, dtype=np.uint64)[:, None]
    c[2] += np.uint64(offset & 0xFFFFFFFF)
    c[3] += np.uint64(offset >> 32)
    k = [seed & 0xFFFFFFFF, seed >> 32]
    low = np.uint64(0xFFFFFFFF)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    bits = np.stack([c[j % 8 // 2] >> np.uint64(16 * (j % 2)) & np.uint64(0xFFFF) for j in range(8)], -1)
    t = int(np.rint(p * 65536))
    keep = (bits.reshape(rows, -1)[:, :cols] >= t).astype(np.float64)
    return torch.from_numpy(keep * (65536 / (65536 - t) if t < 65536 else 0))


def _within(got, want, bound, dtype):
    got = got.cpu().double()
    assert got.shape == want.shape
    assert torch.isfinite(want).all()
    d = (got - want).abs()
    most = bound + U[dtype] * (want.abs() + bound) + LEAST[dtype]
    assert (d <= most).all(), (d - most).max()


def test_generator():
    """Philox4x32-10 at the counters and keys its authors publish values for."""
    # counter 0, key 0: 6627e8d5 e169c58d bc57ac4c 9b00dbd8: row 0, column group 0.
    words = [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    halves = [w >> (16 * h) & 0xFFFF for w in words for h in range(2)]
    x = torch.ones(1, 8, device=DEV)
    for j, h in enumerate(halves):
        for t, kept in ((h, True), (h + 1, False)):
            y = layers.dropout(x, t / 65536, 0)
            assert bool(y[0, j] != 0) == kept, (j, t)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("rows,cols,ld,offset,p", [
    (1, 1, 1, 0, 0.5), (3, 7, 9, 1, 0.25), (1, 8, 8, 0, 0.9), (5, 9, 9, 0, 0.1), (70, 1000, 1000, 0, 0.1),
    (33, 513, 517, 3, 0.3), (2, 4099, 4099, 0, 0.5), (1000, 24, 24, 0, 0.01), (17, 100, 100, 0, 0.0), (17, 100, 100, 0, 1.0)])
def test_dropout(dtype, rows, cols, ld, offset, p):
    _say("dropout", dtype, rows, cols, ld, offset, p)
    seed, off = (rows * 0x123456789ABCDEF + 1) % 2 ** 64, cols * (2 ** 31 + 1)
    x = (torch.randn(rows, cols, generator=_gen(1)) + 3).to(dtype)
    r = torch.randn(rows, cols, generator=_gen(2)).to(dtype)
    f = _factors(rows, cols, p, seed, off)
    y = layers.dropout(_strided(x, ld, offset), p, seed, off)
    want = x.double() * f
    assert torch.equal(y.cpu() != 0, want != 0)
    _within(y, want, 2 * E * want.abs(), dtype)
    y = layers.dropout(_strided(x, ld, offset), p, seed, off, _strided(r, cols + 2, 1))
    _within(y, want + r.double(), 2 * E * (want.abs() + r.double().abs()), dtype)
    at = torch.tensor([seed - 2 ** 64 if seed >= 2 ** 63 else seed], dtype=torch.int64, device=DEV)
    assert torch.equal(layers.dropout(_strided(x, ld, offset), p, at, off, _strided(r, cols + 2, 1)), y)


def test_dropout_drops_what_is_not_finite():
    x = torch.full((50, 64), float("nan"), device=DEV)
    y = layers.dropout(x, 0.5, 11)
    f = _factors(50, 64, 0.5, 11, 0)
    assert torch.equal(torch.isnan(y).cpu(), f > 0) and (y[(f == 0).to(DEV)] == 0).all()


def test_dropout_share():
    """Seeds and offsets give other masks, each with its share of zeros: the
    share's deviation over n elements is sqrt(p (1 - p) / n), six of it allowed."""
    x = torch.ones(512, 1024, device=DEV)
    masks = [layers.dropout(x, 0.2, s, o) == 0 for s, o in [(1, 0), (2, 0), (1, 1), (1, 2 ** 32), (2 ** 32 + 1, 0)]]
    n = x.numel()
    for m in masks:
        assert abs(m.float().mean().item() - 0.2) < 6 * (0.16 / n) ** 0.5 + 2 ** -17
    for i in range(len(masks)):
        for j in range(i):
            assert abs((masks[i] & masks[j]).float().mean().item() - 0.04) < 6 * (0.04 * 0.96 / n) ** 0.5 + 2 ** -16


COLS = [1, 2, 7, 8, 9, 64, 511, 512, 513, 1024, 1025, 2048, 2051, 2501, 4096, 5003, 8185, 8192, 8200, 20001]


def _norm_case(rows, cols, dtype, seed, spread=True):
    x = torch.randn(rows, cols, generator=_gen(seed)) + 0.5
    if spread:
        x = x * torch.exp(torch.randn(rows, 1, generator=_gen(seed + 1)))
    r = torch.randn(rows, cols, generator=_gen(seed + 2))
    return x.to(dtype), r.to(dtype)


def _check_norm(x, r, w, b, p, seed, off, eps, outs, dtype):
    y, h, mean, rstd = outs
    rows, cols = x.shape
    want_h = x.double() * (_factors(rows, cols, p, seed, off) if p > 0 else 1)
    if r is not None:
        want_h = want_h + r.double()
    _within(h, want_h, 2 * E * (want_h.abs() + (r.double().abs() if r is not None else 0)) if r is not None or p > 0 else 0 * want_h, dtype)
    h64 = h.cpu().double()
    m = h64.mean(1, keepdim=True)
    s = ((h64 - m).square().mean(1, keepdim=True) + eps).rsqrt()
    size = h64.abs().mean(1, keepdim=True)
    assert ((mean.cpu().double()[:, None] - m).abs() <= 300 * E * size).all()
    off_by = 1e-5 + (300 * E * size * s) ** 2
    assert ((rstd.cpu().double()[:, None] - s).abs() <= off_by * s).all()
    w64 = w.cpu().double()
    b64 = b.cpu().double() if b is not None else torch.zeros_like(w64)
    core = (h64 - m) * s * w64
    bound = (off_by + 1e-5) * core.abs() + 300 * E * size * s * w64.abs() + 2 * E * b64.abs()
    _within(y, core + b64, bound, dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("cols", COLS)
def test_layer_norm(dtype, cols):
    rows = 37 if cols < 3000 else 5
    wide = cols % 2 == 0 and dtype is not torch.float32
    x, r = _norm_case(rows, cols, dtype, cols)
    wt = torch.float32 if wide else dtype
    w = (1 + 0.2 * torch.randn(cols, generator=_gen(5))).to(wt).to(DEV)
    b = (0.3 * torch.randn(cols, generator=_gen(6))).to(wt).to(DEV)
    for p, res, bias, ld, at in [(0.0, False, True, cols, 0), (0.0, True, True, cols + 3, 1), (0.3, True, False, cols, 0),
                                 (0.5, False, True, cols + 5, 2)]:
        _say("layer_norm", dtype, rows, cols, p, res, bias, ld, at)
        outs = layers.layer_norm(_strided(x, ld, at), w, b if bias else None, _strided(r, cols + 1, at) if res else None,
                                 1e-5, p, 77 + cols, 5)
        _check_norm(x, r if res else None, w, b if bias else None, p, 77 + cols, 5, 1e-5, outs, dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("cols", COLS)
def test_layer_norm_backward(dtype, cols):
    wide = cols % 2 == 0 and dtype is not torch.float32
    wt = torch.float32 if wide else dtype
    for rows, p, gh, ld, at in [(1, 0.0, False, cols, 0), (70 if cols < 3000 else 9, 0.3, True, cols + 3, 1),
                                (1100 if cols < 600 else 11, 0.0, True, cols, 0), (6, 0.5, False, cols + 1, 3)]:
        _say("layer_norm_backward", dtype, rows, cols, p, gh, ld, at)
        h, extra = _norm_case(rows, cols, dtype, cols + rows, spread=False)
        g = (torch.randn(rows, cols, generator=_gen(9)) * 0.1).to(dtype)
        w = (1 + 0.2 * torch.randn(cols, generator=_gen(5))).to(wt)
        h64 = h.double()
        mean = h64.mean(1)
        rstd = ((h64 - mean[:, None]).square().mean(1) + 1e-5).rsqrt()
        m32, r32 = mean.float(), rstd.float()
        gx, gr, gw, gb = layers.layer_norm_backward(
            _strided(g, ld, at), _strided(h, cols + 2, at), m32.to(DEV), r32.to(DEV), w.to(DEV),
            _strided(extra, cols + 4, at) if gh else None, p, 99, 2 ** 40)
        xh, u = (h64 - m32.double()[:, None]) * r32.double()[:, None], g.double() * w.double()
        want = r32.double()[:, None] * (u - u.mean(1, keepdim=True) - xh * (u * xh).mean(1, keepdim=True))
        size = r32.double()[:, None] * (u.abs() + u.abs().mean(1, keepdim=True) + xh.abs() * (u * xh).abs().mean(1, keepdim=True))
        if gh:
            want, size = want + extra.double(), size + extra.double().abs()
        _within(gr, want, 2e-5 * size, dtype)
        f = _factors(rows, cols, p, 99, 2 ** 40) if p > 0 else torch.ones(rows, cols, dtype=torch.float64)
        _within(gx, want * f, 2e-5 * size * f, dtype)
        _within(gw, (g.double() * xh).sum(0), 2e-5 * (g.double() * xh).abs().sum(0), wt)
        _within(gb, g.double().sum(0), 2e-5 * g.double().abs().sum(0), wt)


def test_layer_norm_differences():
    """The gradients against differences of the forward pass in 64 bits: along a
    direction, the loss's difference at both sides."""
    rows, cols, p, seed = 9, 40, 0.3, 5
    x, r = _norm_case(rows, cols, torch.float32, 3, spread=False)
    w, b = 1 + 0.2 * torch.randn(cols, generator=_gen(1)), torch.randn(cols, generator=_gen(2))
    gy, gh = torch.randn(rows, cols, generator=_gen(3)), torch.randn(rows, cols, generator=_gen(4))
    f = _factors(rows, cols, p, seed, 0)

    def loss(x, r, w, b):
        h = x * f + r
        m = h.mean(1, keepdim=True)
        y = (h - m) * ((h - m).square().mean(1, keepdim=True) + 1e-5).rsqrt() * w + b
        return (y * gy.double()).sum() + (h * gh.double()).sum()

    ins = [t.to(DEV) for t in (x, r, w, b)]
    y, h, mean, rstd = layers.layer_norm(ins[0], ins[2], ins[3], ins[1], 1e-5, p, seed)
    grads = layers.layer_norm_backward(gy.to(DEV), h, mean, rstd, ins[2], gh.to(DEV), p, seed)
    for i in range(4):
        at = [t.double() for t in (x, r, w, b)]
        d = torch.randn(at[i].shape, generator=_gen(10 + i)).double() * 1e-5
        up, down = list(at), list(at)
        up[i], down[i] = at[i] + d, at[i] - d
        want = (loss(*up) - loss(*down)).item() / 2
        got = (grads[i].cpu().double() * d).sum().item()
        scale = (grads[i].cpu().double() * d).abs().sum().item()
        assert abs(got - want) <= 1e-4 * scale, i


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=IDS.get)
@pytest.mark.parametrize("cols", [5, 64, 300, 1500, 3100, 9000])
def test_layer_norm_huge(dtype, cols):
    """Deviations whose squares, and sums that pass f32, and small ones beside."""
    rows = 5
    x = torch.randn(rows, cols, generator=_gen(cols))
    x[0] *= 1e25
    x[1] = torch.where(torch.arange(cols) % 2 == 0, 3e38, -3e38)
    x[2] *= 1e-3
    x[3] = 3e38 * (1 - 1e-2 * torch.rand(cols, generator=_gen(1)))
    x = x.to(dtype)
    w, b = torch.ones(cols, device=DEV).to(dtype), torch.zeros(cols, device=DEV).to(dtype)
    y, h, mean, rstd = layers.layer_norm(x.to(DEV), w, b)
    x64 = x.double()
    m = x64.mean(1, keepdim=True)
    s = ((x64 - m).square().mean(1, keepdim=True) + 1e-5).rsqrt()
    size = x64.abs().mean(1, keepdim=True)
    # rstd itself may lie below f32's normal numbers, with 21 bits left.
    assert ((mean.cpu().double()[:, None] - m).abs() <= 300 * E * size).all()
    off_by = 1e-5 + (300 * E * size * s) ** 2
    assert ((rstd.cpu().double()[:, None] - s).abs() <= (off_by + 2.0 ** -21) * s).all()
    want = (x64 - m) * s
    _within(y, want, (off_by + 1e-5) * want.abs() + 300 * E * size * s, dtype)
    g = torch.randn(rows, cols, generator=_gen(7)).to(dtype)
    gx = layers.layer_norm_backward(g.to(DEV), h, mean, rstd, w)[0].cpu().double()
    m, s = mean.cpu().double()[:, None], rstd.cpu().double()[:, None]
    xh, u = (x64 - m) * s, g.double()
    want = s * (u - u.mean(1, keepdim=True) - xh * (u * xh).mean(1, keepdim=True))
    size = s * (u.abs() + u.abs().mean(1, keepdim=True) + xh.abs() * (u * xh).abs().mean(1, keepdim=True))
    # Below f32's normal numbers a step is 2^-149 (bf16: 2^-133).
    assert ((gx - want).abs() <= (2e-5 + U[dtype]) * size + 8 * LEAST[dtype]).all()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("cols", [1, 7, 64, 300, 1000, 2501, 3100, 5003, 9000])
def test_layer_norm_of_equal_values(dtype, cols):
    """y is the bias, to the bit.  The first mean is off by k steps of f32, k below
    300; the deviations are k steps each, exactly, and so is their sum, k * cols < 2^24
    of them; its mean is k (1 + 2^-23) steps, which added to the first mean rounds to
    the value.  The variance left is below 300e * (300 steps)^2: nothing beside eps up
    to 1000, and none where the sum passes f32 and the row is done again."""
    values = [0.1, -77.7, 1000.0, 65504.0] + ([1e25, 3e38] if dtype is not torch.float16 else [])
    x = torch.tensor(values).to(dtype)[:, None].expand(-1, cols).contiguous()
    w, b = torch.randn(2, cols, generator=_gen(cols)).to(dtype).to(DEV)
    y, _, mean, rstd = layers.layer_norm(x.to(DEV), w, b)
    assert torch.equal(y, b.expand(len(values), -1))
    assert torch.equal(mean.cpu(), x[:, 0].float())
    for i in [0, 1, 2] + ([5] if dtype is not torch.float16 else []):
        assert abs(rstd[i].item() * 1e-5 ** 0.5 - 1) < 1e-3


def test_layer_norm_of_no_columns():
    w = torch.ones(0, device=DEV)
    y, h, mean, rstd = layers.layer_norm(torch.ones(4, 0, device=DEV), w, w)
    assert y.shape == h.shape == (4, 0) and torch.isnan(mean).all() and torch.isnan(rstd).all()
    assert [tuple(g.shape) for g in layers.layer_norm_backward(y, h, mean, rstd, w)] == [(4, 0), (4, 0), (0,), (0,)]


def test_layer_norm_not_finite_rows_stay_apart():
    x = torch.randn(200, 100, generator=_gen(1))
    x[3, 5], x[7, 9] = float("nan"), float("inf")
    w = torch.ones(100, device=DEV)
    y, h, mean, rstd = layers.layer_norm(x.to(DEV), w)
    good = torch.ones(200, dtype=torch.bool)
    good[3] = good[7] = False
    assert torch.isnan(y.cpu()[~good]).all() and torch.isfinite(y.cpu()[good]).all()
    assert torch.equal(y.cpu()[good], layers.layer_norm(x[good].to(DEV), w)[0].cpu())


def test_empty():
    w = torch.ones(16, device=DEV)
    y, h, mean, rstd = layers.layer_norm(torch.empty(0, 16, device=DEV), w, w)
    assert y.shape == (0, 16) and mean.shape == (0,)
    gx, gr, gw, gb = layers.layer_norm_backward(torch.empty(0, 16, device=DEV), y, mean, rstd, w)
    assert gx.shape == (0, 16) and torch.equal(gw, torch.zeros(16, device=DEV)) and torch.equal(gb, gw)
    assert layers.dropout(torch.empty(0, 16, device=DEV), 0.5, 1).shape == (0, 16)
    e = torch.empty(4, 0, device=DEV)
    assert layers.layer_norm(e, torch.empty(0, device=DEV))[0].shape == (4, 0)
    assert layers.dropout(e, 0.5, 1).shape == (4, 0)


def test_constant_rows():
    """A row without deviations gives the bias (its mean is exact here)."""
    w, b = torch.randn(256, device=DEV), torch.randn(256, device=DEV)
    y, _, mean, rstd = layers.layer_norm(torch.full((3, 256), 4.0, device=DEV), w, b, eps=0.25)
    assert torch.equal(y, b.expand(3, 256)) and (mean == 4).all() and (rstd == 2).all()


@pytest.mark.parametrize("cols", [100, 4096, 9001])
def test_graph_follows_the_seed(cols):
    """A captured forward and backward pass, replayed with other seeds and inputs."""
    x = torch.randn(40, cols, device=DEV)
    r, g = torch.randn_like(x), torch.randn_like(x)
    w, b = torch.randn(cols, device=DEV), torch.randn(cols, device=DEV)
    seed = torch.tensor([1], dtype=torch.int64, device=DEV)

    def run():
        y, h, mean, rstd = layers.layer_norm(x, w, b, r, 1e-5, 0.3, seed, 7)
        return [y, h, mean, rstd, *layers.layer_norm_backward(g, h, mean, rstd, w, g, 0.3, seed, 7),
                layers.dropout(x, 0.3, seed, 8, r)]

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    seen = []
    for turn in range(3):
        seed.fill_(100 + turn)
        x.copy_(torch.randn(40, cols, generator=_gen(turn)))
        want = run()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, want)), turn
        seen.append(out[1].clone())
    assert not torch.equal(seen[0], seen[1])


def test_repeats_and_streams():
    x = torch.randn(3000, 1000, device=DEV).bfloat16()
    w = torch.randn(1000, device=DEV).bfloat16()
    y, h, mean, rstd = layers.layer_norm(x, w, None, x, 1e-5, 0.2, 3)
    want = layers.layer_norm_backward(x, h, mean, rstd, w, x, 0.2, 3)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for turn in range(4):
        with torch.cuda.stream(streams[turn % 2]):
            got.append(layers.layer_norm_backward(x, h, mean, rstd, w, x, 0.2, 3))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for outs in got for a, b in zip(outs, want))


def test_outputs_stay_inside():
    lib = nat.load()
    for rows, cols in [(3, 5), (5, 77), (9, 1031), (4, 4099), (3, 8199), (2, 9001)]:
        x, r = (t.to(DEV) for t in _norm_case(rows, cols, torch.bfloat16, cols))
        w = torch.ones(cols, dtype=torch.bfloat16, device=DEV)
        want = layers.layer_norm(x, w, w, r, 1e-5, 0.3, 4)
        n = rows * cols
        store = [torch.full((n + 96,), 7.0, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
        y, h = (s[47:47 + n] for s in store)
        stats = torch.full((2, rows + 8), 7.0, device=DEV)
        nat.check(lib.tg_layer_norm(0, 1, 1, x.data_ptr(), cols, r.data_ptr(), cols, w.data_ptr(), w.data_ptr(), 1e-5, 0.3,
                                    4, None, 0, y.data_ptr(), h.data_ptr(), stats[0].data_ptr(), stats[1].data_ptr(), rows,
                                    cols, torch.cuda.current_stream().cuda_stream))
        torch.cuda.synchronize()
        assert torch.equal(y.view(rows, cols), want[0]) and torch.equal(h.view(rows, cols), want[1])
        assert all((s[:47] == 7).all() and (s[47 + n:] == 7).all() for s in store) and (stats[:, rows:] == 7).all()
