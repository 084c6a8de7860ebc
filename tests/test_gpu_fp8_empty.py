"""The layer in 8-bit floating point where a dimension is zero: an empty sum gives
the bias or zeros, empty outputs their shapes, in each type, eagerly, with
gradients and from a captured graph."""
import pytest
import torch

from tropical_gemm import fp8
from tropical_gemm import pytorch as tgt

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16, torch.float32]
IDS = {torch.bfloat16: "bf16", torch.float16: "f16", torch.float32: "f32"}
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _blocks(n):
    return -(-n // 128)


def _operand(rows, k, scale_rows):
    return (torch.full((rows, k), 0x38, dtype=torch.uint8, device=DEV).view(E4M3),
            torch.full((scale_rows, _blocks(k)), 127, dtype=torch.uint8, device=DEV).view(E8M0))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("m", [0, 3, 65, 300])
@pytest.mark.parametrize("n", [0, 5, 200])
@pytest.mark.parametrize("k", [0, 8])
def test_matmul(dtype, m, n, k):
    a, b = _operand(m, k, m), _operand(n, k, _blocks(n))
    for bias in (None, torch.arange(n, device=DEV).to(dtype)):
        c = fp8.matmul(*a, *b, bias, dtype)
        want = torch.full((m, n), float(k), device=DEV) + (0 if bias is None else bias.float())
        assert c.dtype is dtype and torch.equal(c, want.to(dtype))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
@pytest.mark.parametrize("m,n,k", [(100, 70, 0), (0, 70, 130), (100, 0, 130), (0, 70, 0), (100, 0, 0)])
def test_linear(dtype, m, n, k):
    """Quantize, product and both gradients of a layer without features, tokens or
    outputs."""
    x = torch.ones(m, k, device=DEV, dtype=dtype).requires_grad_()
    w = torch.ones(n, k, device=DEV, dtype=dtype).requires_grad_()
    y = tgt.fp8_linear_gpu(x, w)
    assert torch.equal(y, torch.full((m, n), float(k), device=DEV, dtype=dtype))
    y.backward(torch.ones_like(y))
    assert torch.equal(x.grad, torch.full((m, k), float(n), device=DEV, dtype=dtype))
    assert torch.equal(w.grad, torch.full((n, k), float(m), device=DEV, dtype=dtype))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS.get)
def test_graph(dtype):
    a, b = _operand(100, 0, 100), _operand(70, 0, 1)
    bias = torch.zeros(70, device=DEV, dtype=dtype)
    fp8.matmul(*a, *b, bias, dtype)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c = fp8.matmul(*a, *b, bias, dtype)
    for turn in range(3):
        bias.fill_(turn + 1)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(c, bias.expand(100, 70))
