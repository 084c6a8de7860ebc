"""Nothing is written before or behind an output or a workspace: the C entry points
of the 8-bit floating point layer, of layer norm's backward pass and of dropout with
outputs at odd elements and workspaces of exactly the size that is asked for, all
between patterns; the results as the Python functions give them."""
import pytest
import torch

from tropical_gemm import _native as nat
from tropical_gemm import fp8, layers

pytestmark = pytest.mark.gpu

DEV = "cuda"
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
TYPES = [torch.bfloat16, torch.float16, torch.float32]
IDS = {torch.bfloat16: "bf16", torch.float16: "f16", torch.float32: "f32"}
KIND = {torch.float32: nat.FLOAT["f32"], torch.bfloat16: nat.FLOAT["bf16"], torch.float16: nat.FLOAT["f16"]}
BEFORE, BEHIND = 63, 97  # an odd number of elements


class Guarded:
    """n elements between patterns."""

    def __init__(self, n, dtype, before=BEFORE):
        self.n, self.before = n, before
        self.store = torch.full((before + n + BEHIND,), 7, dtype=dtype, device=DEV)
        self.view = self.store[before:before + n]

    def ptr(self):
        return self.view.data_ptr()

    def whole(self):
        return bool((self.store[:self.before] == 7).all() and (self.store[self.before + self.n:] == 7).all())


def _workspace(need):
    return Guarded(need, torch.uint8, 512)  # its alignment kept


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _randn(seed, *shape):
    g = torch.Generator()
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g)


def _bytes(t):
    return t.contiguous().view(torch.uint8)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("br", [1, 128])
@pytest.mark.parametrize("rows,cols", [(3, 5), (130, 77), (17, 513), (5, 520), (129, 1031), (4, 4099), (2, 9001), (300, 8)])
def test_quantize(dtype, br, rows, cols):
    print("[case]", dtype, br, rows, cols, flush=True)
    lib = nat.load()
    x = _randn(cols, rows, cols).to(dtype).to(DEV)
    want_q, want_s = fp8.quantize(x, br)
    rb, cb = (rows if br == 1 else -(-rows // 128)), -(-cols // 128)
    q, s = Guarded(rows * cols, torch.uint8), Guarded(rb * cb, torch.uint8)
    nat.check(lib.tg_f8_quantize(0, KIND[dtype], x.data_ptr(), cols, br, q.ptr(), s.ptr(), rows, cols, _stream()))
    torch.cuda.synchronize()
    assert q.whole() and s.whole()
    assert torch.equal(q.view.view(rows, cols), _bytes(want_q)) and torch.equal(s.view.view(cb, rb), _bytes(want_s.t()))
    y = Guarded(rows * cols, dtype)
    nat.check(lib.tg_f8_dequantize(0, KIND[dtype], q.ptr(), cols, s.ptr(), 1, rb, br, y.ptr(), rows, cols, _stream()))
    torch.cuda.synchronize()
    assert y.whole() and torch.equal(y.view.view(rows, cols), fp8.dequantize(want_q, want_s, dtype))


def _operand(seed, rows, k, scale_rows):
    q = (_randn(seed, rows, k) * 100).clamp(-448, 448).to(E4M3).to(DEV)
    s = (torch.randint(118, 126, (-(-k // 128), scale_rows), generator=torch.Generator().manual_seed(seed))
         .to(torch.uint8).to(DEV).view(E8M0).t())
    return q, s


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("m,n,k", [(3, 5, 77), (40, 33, 128), (70, 75, 131), (300, 261, 260), (129, 1031, 1040), (700, 77, 5)])
def test_products_and_gradients(dtype, m, n, k):
    lib, kind = nat.load(), KIND[dtype]
    (a, sa), (b, sb) = _operand(m, m, k, m), _operand(n + 1000, n, k, -(-n // 128))
    g = _randn(k, m, n).to(dtype).to(DEV)
    plan = lib.tg_f8_backward_plan
    print("[case]", dtype, lib.tg_f8_gemm_plan(kind, a.data_ptr(), k, b.data_ptr(), k, m, n, k).decode(),
          *(plan(kind, w, g.data_ptr(), n, m, n, k).decode() for w in (1, 0)), flush=True)

    ws = _workspace(lib.tg_f8_gemm_workspace_size(kind, a.data_ptr(), k, b.data_ptr(), k, m, n, k))
    c = Guarded(m * n, dtype)
    nat.check(lib.tg_f8_gemm(0, kind, a.data_ptr(), k, sa.data_ptr(), *sa.stride(), b.data_ptr(), k, sb.data_ptr(),
                             *sb.stride(), None, c.ptr(), m, n, k, ws.ptr(), ws.n, _stream()))
    torch.cuda.synchronize()
    assert c.whole() and ws.whole() and torch.equal(c.view.view(m, n), fp8.matmul(a, sa, b, sb, dtype=dtype))

    ws = _workspace(lib.tg_f8_backward_a_workspace_size(kind, g.data_ptr(), n, m, n, k))
    ga = Guarded(m * k, dtype)
    nat.check(lib.tg_f8_backward_a(0, kind, g.data_ptr(), n, b.data_ptr(), k, sb.data_ptr(), *sb.stride(), ga.ptr(), m, n,
                                   k, ws.ptr(), ws.n, _stream()))
    torch.cuda.synchronize()
    assert ga.whole() and ws.whole() and torch.equal(ga.view.view(m, k), fp8.backward_a(g, b, sb))

    ws = _workspace(lib.tg_f8_backward_b_workspace_size(kind, g.data_ptr(), n, m, n, k))
    gb = Guarded(n * k, dtype)
    nat.check(lib.tg_f8_backward_b(0, kind, g.data_ptr(), n, a.data_ptr(), k, sa.data_ptr(), *sa.stride(), gb.ptr(), m, n,
                                   k, ws.ptr(), ws.n, _stream()))
    torch.cuda.synchronize()
    assert gb.whole() and ws.whole() and torch.equal(gb.view.view(n, k), fp8.backward_b(g, a, sa))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("rows,cols", [(3, 5), (70, 77), (9, 1031), (4, 4099), (2, 9001), (1, 1), (5, 8)])
def test_dropout(dtype, rows, cols):
    x, r = (_randn(s, rows, cols).to(dtype).to(DEV) for s in (1, 2))
    for res in (None, r):
        y = Guarded(rows * cols, dtype)
        nat.check(nat.load().tg_dropout(0, KIND[dtype], x.data_ptr(), cols, None if res is None else res.data_ptr(), cols, 0.3,
                                        11, None, 5, y.ptr(), rows, cols, _stream()))
        torch.cuda.synchronize()
        assert y.whole() and torch.equal(y.view.view(rows, cols), layers.dropout(x, 0.3, 11, 5, res))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 5), (70, 77), (600, 77), (9, 1031), (4, 4099), (3, 8191), (3, 8199),
                                       (300, 9001), (2, 16390)])
def test_layer_norm_backward(dtype, rows, cols):
    print("[case]", dtype, rows, cols, flush=True)
    lib, kind = nat.load(), KIND[dtype]
    h, g, gh = (_randn(s, rows, cols).to(dtype).to(DEV) for s in (1, 2, 3))
    w = _randn(4, cols).to(dtype).to(DEV)
    _, _, mean, rstd = layers.layer_norm(h, w)
    need = lib.tg_layer_norm_backward_workspace_size(rows, cols)
    for p, other in ((0.0, None), (0.3, gh)):
        want = layers.layer_norm_backward(g, h, mean, rstd, w, other, p, 5, 2)
        ws, outs = _workspace(need), [Guarded(rows * cols, dtype), Guarded(rows * cols, dtype), Guarded(cols, dtype),
                                      Guarded(cols, dtype)]
        nat.check(lib.tg_layer_norm_backward(
            0, kind, kind, g.data_ptr(), cols, h.data_ptr(), cols, mean.data_ptr(), rstd.data_ptr(), w.data_ptr(),
            None if other is None else other.data_ptr(), cols, p, 5, None, 2, outs[0].ptr() if p else None, outs[1].ptr(),
            outs[2].ptr(), outs[3].ptr(), rows, cols, ws.ptr(), need, _stream()))
        torch.cuda.synchronize()
        assert ws.whole() and all(o.whole() for o in outs)
        for i, (o, t) in enumerate(zip(outs, want)):
            assert i == 0 and not p or torch.equal(o.view.view(t.shape), t), i
