"""The 8-bit layer's operators at the limits of their definitions: ties, ranges,
rows in several workgroups, scales far from each other.  Expected values come
from integers, 64-bit sums or bits that have to be equal."""
import pytest
import torch

from tropical_gemm import int8

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
