"""The entry points of the layer in 8-bit floating point, of layer norm and of
dropout refuse bad arguments before they touch a device, size their workspaces
and name their plans; the Python layer refuses host tensors."""
import ctypes

import pytest
import torch

from tropical_gemm import _native as nat
from tropical_gemm import fp8, layers

P = 4096  # stands for a device pointer; never dereferenced
NONE = ctypes.c_size_t(-1).value

DEFAULTS = {
    "tg_f8_quantize": dict(device=0, type=1, x=P, ldx=8, block_rows=1, q=P, scale=P, rows=4, cols=8, stream=None),
    "tg_f8_dequantize": dict(device=0, type=1, q=P, ldq=8, scale=P, scale_row=1, scale_col=4, block_rows=1, y=P, rows=4,
                             cols=8, stream=None),
    "tg_f8_gemm": dict(device=0, type=1, a=P, lda=16, a_scale=P, a_scale_row=1, a_scale_col=4, b=P, ldb=16, b_scale=P,
                       b_scale_row=1, b_scale_col=1, bias=None, c=P, m=4, n=8, k=16, ws=P, ws_bytes=1 << 24, stream=None),
    "tg_f8_backward_a": dict(device=0, type=1, grad_c=P, ldg=8, b=P, ldb=16, b_scale=P, b_scale_row=1, b_scale_col=1,
                             grad_a=P, m=4, n=8, k=16, ws=P, ws_bytes=1 << 24, stream=None),
    "tg_f8_backward_b": dict(device=0, type=1, grad_c=P, ldg=8, a=P, lda=16, a_scale=P, a_scale_row=1, a_scale_col=4,
                             grad_b=P, m=4, n=8, k=16, ws=P, ws_bytes=1 << 24, stream=None),
    "tg_dropout": dict(device=0, type=1, x=P, ldx=8, residual=P, ldr=8, p=0.5, seed=1, seed_at=None, offset=0, y=P, rows=4,
                       cols=8, stream=None),
    "tg_layer_norm": dict(device=0, type=1, weight_type=1, x=P, ldx=8, residual=P, ldr=8, weight=P, bias=P, eps=1e-5, p=0.5,
                          seed=1, seed_at=None, offset=0, y=P, h=P, mean=P, rstd=P, rows=4, cols=8, stream=None),
    "tg_layer_norm_backward": dict(device=0, type=1, weight_type=1, grad_y=P, ldg=8, h=P, ldh=8, mean=P, rstd=P, weight=P,
                                   grad_h=P, ldgh=8, p=0.5, seed=1, seed_at=None, offset=0, grad_x=P, grad_residual=P,
                                   grad_weight=P, grad_bias=P, rows=4, cols=8, ws=P, ws_bytes=1 << 20, stream=None),
}
ALL = list(DEFAULTS)
PRODUCTS = ["tg_f8_gemm", "tg_f8_backward_a", "tg_f8_backward_b"]


def _call(name, **kw):
    """Calls entry point `name` with its default (valid) arguments but kw."""
    args = dict(DEFAULTS[name])
    assert set(kw) <= set(args)
    args.update(kw)
    return getattr(nat.load(), name)(*args.values())


@pytest.mark.parametrize("name", ALL)
def test_unknown_type(name):
    assert _call(name, type=3) == nat.TG_ERR_INVALID_ARGUMENT
    assert "unknown type 3" in nat.last_error()


@pytest.mark.parametrize("name", ALL)
@pytest.mark.parametrize("value,needle", [(-1, "negative dimension"), (1 << 31, "2^31-1")])
def test_dimensions(name, value, needle):
    for dim in (("m", "n", "k") if name in PRODUCTS else ("rows", "cols")):
        assert _call(name, **{dim: value}) == nat.TG_ERR_DIMENSION_MISMATCH
        assert needle in nat.last_error()


BIG = 1 << 32


@pytest.mark.parametrize("name,kw,needle", [
    ("tg_f8_quantize", dict(ldx=7), "row stride of x"),
    ("tg_f8_quantize", dict(cols=(1 << 30) + 1, ldx=BIG), "at most 2^30"),
    ("tg_f8_dequantize", dict(ldq=7), "row stride of q"),
    ("tg_f8_dequantize", dict(scale_row=-1), "strides of scale"),
    ("tg_f8_dequantize", dict(scale_col=1 << 41), "strides of scale"),
    ("tg_f8_gemm", dict(lda=15), "row stride of a"),
    ("tg_f8_gemm", dict(ldb=15), "row stride of b"),
    ("tg_f8_gemm", dict(k=(1 << 20) + 1, lda=BIG, ldb=BIG), "at most 2^20"),
    ("tg_f8_gemm", dict(a_scale_row=(1 << 22) + 1), "strides of a_scale"),
    ("tg_f8_gemm", dict(b_scale_col=-1), "strides of b_scale"),
    ("tg_f8_backward_a", dict(ldg=7), "row stride of grad_c"),
    ("tg_f8_backward_a", dict(ldb=15), "row stride of b"),
    ("tg_f8_backward_a", dict(b_scale_row=-1), "strides of b_scale"),
    ("tg_f8_backward_a", dict(n=(1 << 20) + 1, ldg=BIG), "at most 2^20"),
    ("tg_f8_backward_b", dict(ldg=7), "row stride of grad_c"),
    ("tg_f8_backward_b", dict(lda=15), "row stride of a"),
    ("tg_f8_backward_b", dict(a_scale_row=-1), "strides of a_scale"),
    ("tg_f8_backward_b", dict(m=(1 << 20) + 1), "at most 2^20"),
    ("tg_dropout", dict(ldx=7), "row stride of x"),
    ("tg_dropout", dict(ldr=7), "row stride of residual"),
    ("tg_layer_norm", dict(ldx=7), "row stride of x"),
    ("tg_layer_norm", dict(ldr=7), "row stride of residual"),
    ("tg_layer_norm", dict(cols=(1 << 24) + 1, ldx=BIG, ldr=BIG), "at most 2^24"),
    ("tg_layer_norm_backward", dict(ldg=7), "row stride of grad_y"),
    ("tg_layer_norm_backward", dict(ldh=-8), "row stride of h"),
    ("tg_layer_norm_backward", dict(ldgh=0), "row stride of grad_h"),
    ("tg_layer_norm_backward", dict(cols=(1 << 24) + 1, ldg=BIG, ldh=BIG, ldgh=BIG), "at most 2^24"),
])
def test_sizes(name, kw, needle):
    assert _call(name, **kw) == nat.TG_ERR_DIMENSION_MISMATCH
    assert needle in nat.last_error()


@pytest.mark.parametrize("name,pointers", [
    ("tg_f8_quantize", ["x", "q", "scale"]),
    ("tg_f8_dequantize", ["q", "scale", "y"]),
    ("tg_f8_gemm", ["a", "a_scale", "b", "b_scale", "c"]),
    ("tg_f8_backward_a", ["grad_c", "b", "b_scale", "grad_a"]),
    ("tg_f8_backward_b", ["grad_c", "a", "a_scale", "grad_b"]),
    ("tg_dropout", ["x", "y"]),
    ("tg_layer_norm", ["x", "weight", "y", "h", "mean", "rstd"]),
    ("tg_layer_norm_backward", ["grad_y", "h", "mean", "rstd", "weight", "grad_x", "grad_residual", "grad_weight",
                                "grad_bias"]),
])
def test_null_pointers(name, pointers):
    for p in pointers:
        assert _call(name, **{p: None}) == nat.TG_ERR_INVALID_ARGUMENT
        assert f"{p} is NULL" in nat.last_error()


@pytest.mark.parametrize("name", ["tg_f8_quantize", "tg_f8_dequantize"])
@pytest.mark.parametrize("value", [0, 2, 64, 256, -1])
def test_block_rows(name, value):
    assert _call(name, block_rows=value) == nat.TG_ERR_INVALID_ARGUMENT
    assert "1 or 128" in nat.last_error()


@pytest.mark.parametrize("name", ["tg_dropout", "tg_layer_norm", "tg_layer_norm_backward"])
@pytest.mark.parametrize("p", [-0.1, 1.0001, float("nan"), float("inf")])
def test_probability(name, p):
    assert _call(name, p=p) == nat.TG_ERR_INVALID_ARGUMENT
    assert "between 0 and 1" in nat.last_error()


@pytest.mark.parametrize("eps", [-1e-5, float("nan"), float("inf")])
def test_eps(eps):
    assert _call("tg_layer_norm", eps=eps) == nat.TG_ERR_INVALID_ARGUMENT
    assert "eps" in nat.last_error()


@pytest.mark.parametrize("name", ["tg_layer_norm", "tg_layer_norm_backward"])
def test_weight_type(name):
    assert _call(name, weight_type=2) == nat.TG_ERR_INVALID_ARGUMENT
    assert "weight's type" in nat.last_error()


def test_workspaces():
    lib = nat.load()
    need = lib.tg_layer_norm_backward_workspace_size(4, 8)
    assert need == 2 * 8 * 4 and lib.tg_layer_norm_backward_workspace_size(-1, 8) == NONE
    assert _call("tg_layer_norm_backward", ws_bytes=need - 1) == nat.TG_ERR_INVALID_ARGUMENT
    assert "workspace too small" in nat.last_error()
    assert _call("tg_layer_norm_backward", ws=P + 16) == nat.TG_ERR_INVALID_ARGUMENT
    assert "256-byte aligned" in nat.last_error()
    # Few rows need none, unaligned rows of many do.
    assert lib.tg_f8_gemm_workspace_size(1, P, 8192, P, 8192, 1, 8192, 8192) == 0
    assert lib.tg_f8_gemm_workspace_size(1, P + 1, 8192, P, 8192, 1000, 1000, 8192) >= 1000 * 8192
    assert lib.tg_f8_gemm_workspace_size(1, P, 8192, P, 8192, -1, 1, 1) == NONE
    assert lib.tg_f8_gemm_workspace_size(1, P, BIG, P, BIG, 1, 1, (1 << 20) + 1) == NONE
    kw = dict(m=1000, n=1000, k=999, lda=999, ldb=999)
    need = lib.tg_f8_gemm_workspace_size(1, P, 999, P, 999, 1000, 1000, 999)
    assert need > 0 and _call("tg_f8_gemm", **kw, ws_bytes=need - 1) == nat.TG_ERR_INVALID_ARGUMENT
    need = lib.tg_f8_backward_a_workspace_size(0, P, 999, 1000, 999, 1000)
    assert need >= 1000 * 1024 * 2 * 3
    assert _call("tg_f8_backward_a", type=0, m=1000, n=999, k=1000, ldg=999, ldb=1000,
                 ws_bytes=need - 1) == nat.TG_ERR_INVALID_ARGUMENT
    assert lib.tg_f8_backward_b_workspace_size(1, P, 8, -1, 1, 1) == NONE


def test_sizes_of_refused_calls():
    """What a call would refuse has no workspace size: SIZE_MAX, without a sum that overflows."""
    lib = nat.load()
    most = 2 ** 31 - 1
    for m, n, k in [(most + 1, 4, 8), (4, 2 ** 62, 8), (4, 4, 2 ** 20 + 1), (2 ** 62, 2 ** 62, 8)]:
        assert lib.tg_f8_gemm_workspace_size(1, P, k, P, k, m, n, k) == NONE
    assert lib.tg_f8_gemm_workspace_size(7, P, 8, P, 8, 4, 4, 8) == NONE
    for size in (lib.tg_f8_backward_a_workspace_size, lib.tg_f8_backward_b_workspace_size):
        assert size(7, P, 8, 4, 8, 8) == NONE and size(1, P, 8, 2 ** 62, 2 ** 62, 8) == NONE
    assert lib.tg_f8_backward_a_workspace_size(1, P, 2 ** 21, 4, 2 ** 21, 8) == NONE
    assert lib.tg_f8_backward_b_workspace_size(1, P, 8, 2 ** 21, 8, 8) == NONE
    assert lib.tg_layer_norm_backward_workspace_size(2 ** 62, 8) == NONE
    assert lib.tg_layer_norm_backward_workspace_size(4, 2 ** 24 + 1) == NONE


def test_plans():
    lib = nat.load()
    plan = lambda kind, a, lda, b, ldb, m, n, k: lib.tg_f8_gemm_plan(kind, a, lda, b, ldb, m, n, k).decode()
    assert plan(1, P, 8192, P, 8192, 1, 8192, 8192) == "stream rows 16 words"
    assert plan(1, P + 1, 8192, P, 8192, 5, 8192, 8192) == "stream rows 16"
    assert plan(1, P, 8192, P, 8192, 8192, 8192, 8192) == "tiles 256x256"
    assert plan(0, P, 8192, P, 8192, 8192, 8192, 8192).startswith("wide tiles")
    assert plan(1, P, 8192, P, 8192, 0, 8192, 8192) == "none" and plan(1, P, 0, P, 0, 3, 8192, 0) == "bias"
    assert plan(1, P, 8, P, 8192, 3, 8192, 8192) == "invalid" and plan(7, P, 8, P, 8, 3, 8, 8) == "invalid"
    assert lib.tg_f8_backward_plan(1, 1, P, 8, 4, 8, 0).decode() == "none"
    assert lib.tg_f8_backward_plan(1, 1, P, 0, 4, 0, 8).decode() == "zero"
    assert lib.tg_f8_backward_plan(1, 1, P, 7, 4, 8, 8).decode() == "invalid"


@pytest.mark.parametrize("kind,m,n,k,expected", [
    (1, 32, 4096, 8192, "stream rows 32 words"), (1, 32, 8192, 8192, "tiles"),
    (1, 48, 8192, 4096, "stream rows 48 words"), (2, 49, 4096, 4096, "stream rows 64 words"),
    (1, 64, 4096, 4112, "tiles"), (1, 48, 16384, 4095, "stream rows 48"), (1, 64, 8192, 8191, "stream rows 64"),
    (1, 64, 8193, 8191, "tiles"), (0, 64, 16384, 8192, "stream rows 64 words"), (0, 65, 16384, 8192, "wide tiles")])
def test_few_rows_read_the_weights_once(kind, m, n, k, expected):
    plan = nat.load().tg_f8_gemm_plan(kind, P, k, P, k, m, n, k).decode()
    assert plan == expected if "rows" in expected else plan.startswith(expected)


E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def test_host_tensors():
    x = torch.zeros(4, 8)
    q, s = torch.zeros(4, 8).to(E4M3), torch.zeros(4, 1, dtype=torch.uint8).view(E8M0)
    w = torch.ones(8)
    for call in (lambda: fp8.quantize(x), lambda: fp8.dequantize(q, s), lambda: fp8.matmul(q, s, q, s[:1]),
                 lambda: fp8.backward_a(x, q, s[:1]), lambda: fp8.backward_b(x, q, s), lambda: layers.dropout(x, 0.5, 1),
                 lambda: layers.layer_norm(x, w), lambda: layers.layer_norm_backward(x, x, w[:4], w[:4], w)):
        with pytest.raises(ValueError, match="device tensors"):
            call()
