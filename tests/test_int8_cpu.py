"""The 8-bit layer's entry points refuse bad arguments before they touch a
device, size their workspaces, and the Python layer refuses host tensors."""
import ctypes

import pytest

from tropical_gemm import _native as nat

P = 4096  # stands for a device pointer; never dereferenced


def _call(name, **kw):
    """Calls entry point `name` with its default (valid) arguments but kw."""
    defaults = {
        "tg_i8_quantize": dict(device=0, type=1, x=P, ldx=8, q=P, scale=P, rows=4, cols=8, stream=None),
        "tg_i8_dequantize": dict(device=0, type=1, q=P, ldq=8, scale=P, y=P, rows=4, cols=8, stream=None),
        "tg_i8_rms_norm": dict(device=0, type=1, weight_type=1, x=P, ldx=8, residual=P, ldr=8, weight=P,
                               eps=1e-6, q=P, scale=P, h=P, rows=4, cols=8, stream=None),
        "tg_i8_rms_norm_backward": dict(device=0, type=1, weight_type=1, grad_y=P, ldg=8, h=P, ldh=8, weight=P,
                                        eps=1e-6, grad_h=P, ldgh=8, grad_x=P, grad_weight=P, rows=4, cols=8,
                                        ws=P, ws_bytes=1 << 20, stream=None),
        "tg_i8_gemm": dict(device=0, type=1, a=P, lda=16, a_scale=P, b=P, ldb=16, b_scale=P, bias=None, c=P,
                           m=4, n=8, k=16, ws=P, ws_bytes=1 << 24, stream=None),
        "tg_i8_backward_a": dict(device=0, type=1, grad_c=P, ldg=8, b=P, ldb=16, b_scale=P, grad_a=P, m=4, n=8,
                                 k=16, ws=P, ws_bytes=1 << 24, stream=None),
        "tg_i8_backward_b": dict(device=0, type=1, grad_c=P, ldg=8, a=P, lda=16, a_scale=P, grad_b=P, m=4, n=8,
                                 k=16, ws=P, ws_bytes=1 << 24, stream=None),
    }
    args = dict(defaults[name])
    assert set(kw) <= set(args)
    args.update(kw)
    return getattr(nat.load(), name)(*args.values())


ALL = ["tg_i8_quantize", "tg_i8_dequantize", "tg_i8_rms_norm", "tg_i8_rms_norm_backward", "tg_i8_gemm",
       "tg_i8_backward_a", "tg_i8_backward_b"]
ROWS = ALL[:4]
PRODUCTS = ALL[4:]


@pytest.mark.parametrize("name", ALL)
def test_unknown_type(name):
    assert _call(name, type=3) == nat.TG_ERR_INVALID_ARGUMENT
    assert "unknown type 3" in nat.last_error()


@pytest.mark.parametrize("name", ALL)
@pytest.mark.parametrize("value,needle", [(-1, "negative dimension"), (1 << 31, "2^31-1")])
def test_dimensions(name, value, needle):
    for dim in (("rows", "cols") if name in ROWS else ("m", "n", "k")):
        assert _call(name, **{dim: value}) == nat.TG_ERR_DIMENSION_MISMATCH
        assert needle in nat.last_error()


@pytest.mark.parametrize("name,kw,needle", [
    ("tg_i8_quantize", dict(ldx=7), "row stride of x"),
    ("tg_i8_dequantize", dict(ldq=7), "row stride of q"),
    ("tg_i8_rms_norm", dict(ldx=7), "row stride of x"),
    ("tg_i8_rms_norm", dict(ldr=7), "row stride of residual"),
    ("tg_i8_rms_norm_backward", dict(ldg=7), "row stride of grad_y"),
    ("tg_i8_rms_norm_backward", dict(ldh=-8), "row stride of h"),
    ("tg_i8_rms_norm_backward", dict(ldgh=0), "row stride of grad_h"),
    ("tg_i8_rms_norm_backward", dict(cols=(1 << 24) + 1, ldg=1 << 25, ldh=1 << 25, ldgh=1 << 25), "at most 2^24"),
    ("tg_i8_gemm", dict(lda=15), "row stride of a"),
    ("tg_i8_gemm", dict(ldb=15), "row stride of b"),
    ("tg_i8_gemm", dict(k=1 << 17, lda=1 << 17, ldb=1 << 17), "exact up to k = 131071"),
    ("tg_i8_backward_a", dict(ldg=7), "row stride of grad_c"),
    ("tg_i8_backward_a", dict(ldb=15), "row stride of b"),
    ("tg_i8_backward_b", dict(ldg=7), "row stride of grad_c"),
    ("tg_i8_backward_b", dict(lda=15), "row stride of a"),
])
def test_sizes_and_strides(name, kw, needle):
    assert _call(name, **kw) == nat.TG_ERR_DIMENSION_MISMATCH
    assert needle in nat.last_error()


@pytest.mark.parametrize("name,pointers", [
    ("tg_i8_quantize", ["x", "q", "scale"]),
    ("tg_i8_dequantize", ["q", "scale", "y"]),
    ("tg_i8_rms_norm", ["x", "weight", "q", "scale", "h"]),
    ("tg_i8_rms_norm_backward", ["grad_y", "h", "weight", "grad_x", "grad_weight"]),
    ("tg_i8_gemm", ["a", "a_scale", "b", "b_scale", "c"]),
    ("tg_i8_backward_a", ["grad_c", "b", "b_scale", "grad_a"]),
    ("tg_i8_backward_b", ["grad_c", "a", "a_scale", "grad_b"]),
])
def test_null_pointers(name, pointers):
    for p in pointers:
        assert _call(name, **{p: None}) == nat.TG_ERR_INVALID_ARGUMENT
        assert f"{p} is NULL" in nat.last_error()


@pytest.mark.parametrize("name", ["tg_i8_rms_norm", "tg_i8_rms_norm_backward"])
@pytest.mark.parametrize("eps", [-1e-6, float("nan"), float("inf")])
def test_eps(name, eps):
    assert _call(name, eps=eps) == nat.TG_ERR_INVALID_ARGUMENT
    assert "eps" in nat.last_error()


@pytest.mark.parametrize("name", ["tg_i8_rms_norm", "tg_i8_rms_norm_backward"])
def test_weight_type(name):
    assert _call(name, type=1, weight_type=2) == nat.TG_ERR_INVALID_ARGUMENT
    assert "weight's type" in nat.last_error()


def test_workspaces():
    lib = nat.load()
    need = lib.tg_i8_rms_norm_backward_workspace_size(4, 8)
    assert need >= 4 * 8 * 4
    assert lib.tg_i8_rms_norm_backward_workspace_size(-1, 8) == ctypes.c_size_t(-1).value
    assert _call("tg_i8_rms_norm_backward", ws_bytes=need - 1) == nat.TG_ERR_INVALID_ARGUMENT
    assert "workspace too small" in nat.last_error()
    assert _call("tg_i8_rms_norm_backward", ws=None) == nat.TG_ERR_INVALID_ARGUMENT
    assert _call("tg_i8_rms_norm_backward", ws=P + 16) == nat.TG_ERR_INVALID_ARGUMENT
    assert "256-byte aligned" in nat.last_error()
    assert lib.tg_i8_gemm_workspace_size(P, 16, P, 16, 4, 8, 1 << 17) == ctypes.c_size_t(-1).value
    assert lib.tg_i8_backward_a_workspace_size(1, P, 8, -1, 8, 16) == ctypes.c_size_t(-1).value
    assert lib.tg_i8_backward_b_workspace_size(1, P, 8, 4, 8, -16) == ctypes.c_size_t(-1).value


def test_python_layer_refuses_host_tensors():
    torch = pytest.importorskip("torch")
    from tropical_gemm import int8

    x = torch.zeros(2, 8)
    q, s, w = torch.zeros(2, 8, dtype=torch.int8), torch.ones(2), torch.ones(8)
    for call in (lambda: int8.quantize(x), lambda: int8.dequantize(q, s), lambda: int8.rms_norm(x, w),
                 lambda: int8.rms_norm_backward(x, x, w), lambda: int8.matmul(q, s, q, s),
                 lambda: int8.backward_a(x[:, :2], q, s), lambda: int8.backward_b(x, q, s)):
        with pytest.raises(ValueError, match="need device tensors"):
            call()


def _gemm_plan(m, n, k, lda=None, ldb=None, a=P, b=P):
    return nat.load().tg_i8_gemm_plan(a, lda or k, b, ldb or k, m, n, k).decode()


def _grad_plan(kind, want_a, m, n, k, ldg=None, g=P):
    return nat.load().tg_i8_backward_plan(nat.FLOAT[kind], want_a, g, ldg or n, m, n, k).decode()


@pytest.mark.parametrize("args,plan", [
    ((1, 8192, 8192), "stream rows 16 words"),
    ((13, 5003, 4099), "stream rows 16"),
    ((16, 28672, 8192), "stream rows 16 words"),
    ((17, 28672, 8192), "tiles 32x64 per_cu 3"),
    ((17, 28672, 8191), "stream rows 32"),
    ((32, 4096, 4100), "stream rows 32 words"),
    ((33, 4096, 4095), "stream rows 48"),
    ((64, 4096, 4095), "stream rows 64"),
    ((64, 16384, 4095), "any"),
    ((8192, 8192, 8192), "tiles 256x256"),
    ((512, 4096, 4096), "tiles 64x128 per_cu 2"),
    ((2048, 2048, 2048), "tiles 128x128"),
    ((2048, 4096, 2048), "tiles 128x128 per_cu 2"),
    ((1024, 1024, 1024), "tiles 64x64 per_cu 2"),
    ((64, 4096, 512), "tiles 32x64 per_cu 3"),
    ((64, 256, 16384), "tiles 32x64 per_cu 3 slices 32"),
    ((300, 500, 701), "any"),
    ((8191, 8191, 8191), "tiles 256x256 pack a pack b"),
    ((0, 8, 16), "none"),
    ((8, 8, 0), "bias"),
    ((8, 8, -1), "invalid"),
    ((8, 8, 1 << 17), "invalid"),
])
def test_gemm_plans(args, plan):
    assert _gemm_plan(*args) == plan


def test_gemm_plans_of_strides():
    assert _gemm_plan(8192, 8192, 8192, lda=8200) == "tiles 256x256 pack a"
    assert _gemm_plan(8192, 8192, 8192, b=P + 8) == "tiles 256x256 pack b"
    assert _gemm_plan(8192, 8192, 8192, ldb=1 << 23) == "tiles 256x256 pack b"
    assert _gemm_plan(8, 8, 16, lda=15) == "invalid"


@pytest.mark.parametrize("kind,want_a,args,plan", [
    ("bf16", 1, (8192, 4096, 4096), "tiles 256x256"),
    ("bf16", 0, (8192, 4096, 4096), "tiles 256x256 pack grad_c"),
    ("f16", 1, (8192, 4095, 4096), "tiles 256x256 pack grad_c"),
    ("f32", 1, (8192, 4096, 4096), "tiles 256x256 pack grad_c"),
    ("f32", 1, (301, 1031, 2049), "tiles 32x64 per_cu 2 planes 3 pack grad_c"),
    ("f32", 0, (1024, 2048, 2048), "tiles 64x128 planes 3 pack grad_c"),
    ("bf16", 0, (8192, 64, 64), "tiles 32x64 per_cu 3 slices 32 pack grad_c"),
    ("bf16", 1, (64, 256, 256), "turn"),
    ("f16", 0, (513, 1024, 1024), "turn"),
    ("f32", 0, (64, 301, 1031), "turn"),
    ("bf16", 0, (64, 256, 7), "tiles 32x64 per_cu 3 pack grad_c"),
    ("bf16", 1, (8, 0, 16), "zero"),
    ("bf16", 1, (0, 8, 16), "none"),
    ("bf16", 0, ((1 << 20) + 1, 8, 16), "invalid"),
])
def test_gradient_plans(kind, want_a, args, plan):
    assert _grad_plan(kind, want_a, *args) == plan
