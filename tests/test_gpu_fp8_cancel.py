"""Products in 8-bit floating point whose large terms cancel.

A row holds 448, -448 at one distance from it, and multiples of 2^-9 elsewhere;
a column is one number c throughout, so the result is c times the sum of the
small ones.  Products and all their partial sums are multiples of 2^-9 c below
2^11 c, which f32 holds: f32 outputs have to be equal to the last bit.  For 16
bits each group of eight products may be cut to multiples of 2^-13 of its largest
one's power of two: 2^-10 of the magnitudes' sum, and the output's rounding.

The power of two is that of the operands' exponents, where e4m3's numbers below 2^-6
count as 2^-6 and zeros not at all: the magnitudes are summed with operands so
taken.
"""
import pytest
import torch

from tropical_gemm import _native as nat
from tropical_gemm import fp8

pytestmark = pytest.mark.gpu

DEV = "cuda"
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
U = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
IDS = {torch.bfloat16: "bf16", torch.float16: "f16", torch.float32: "f32"}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=IDS.get)
@pytest.mark.parametrize("k", [128, 256, 144, 131])
@pytest.mark.parametrize("rows", [16, 64, 127])
def test_cancelling_products(dtype, k, rows):
    g = torch.Generator()
    g.manual_seed(k)
    a = torch.randint(-15, 16, (127, k), generator=g).float() * 2.0 ** -9
    at, apart = torch.arange(127) % (k - 127 + 1), torch.arange(127) + 1
    a[torch.arange(127), at] = 448.0
    a[torch.arange(127), at + apart.clamp(max=k - 1 - at.max().item())] = -448.0
    a = a[torch.randperm(127, generator=g)[:rows]]
    c = torch.tensor([0.5, 1.0, -1.0, 2.0, 0.25]).repeat(20)
    b = c[:, None].expand(100, k).contiguous()
    qa, qb = a.to(E4M3), b.to(E4M3)
    assert torch.equal(qa.float(), a) and torch.equal(qb.float(), b)
    sa = torch.full((rows, -(-k // 128)), 127, dtype=torch.uint8, device=DEV).view(E8M0)
    sb = torch.full((1, -(-k // 128)), 127, dtype=torch.uint8, device=DEV).view(E8M0)
    print("[case]", dtype, rows, k, nat.load().tg_f8_gemm_plan(1, 256, k, 256, k, rows, 100, k).decode(), flush=True)
    got = fp8.matmul(qa.to(DEV), sa, qb.to(DEV), sb, dtype=dtype).cpu().double()
    want, size = a.double() @ b.double().t(), a.double().abs() @ b.double().abs().t()
    if dtype is torch.float32:
        assert torch.equal(got, want)
    else:
        bound = 2.0 ** -10 * size
        assert ((got - want).abs() <= bound + U[dtype] * (want.abs() + bound) + 2.0 ** -24).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=IDS.get)
@pytest.mark.parametrize("m,n,k", [(16, 300, 4), (60, 300, 8), (300, 300, 3), (400, 500, 8), (300, 200, 64), (33, 300, 200)])
def test_numbers_below_the_normal_ones(dtype, m, n, k):
    """Large operands against the smallest ones, whose products are small and count as
    large, beside ordinary products and zeros."""
    g = torch.Generator()
    g.manual_seed(m + n + k)

    def operand(rows):
        kind = torch.randint(0, 4, (rows, k), generator=g)
        small = torch.randint(0, 8, (rows, k), generator=g).float() * 2.0 ** -9
        large = torch.exp2(torch.randint(6, 9, (rows, k), generator=g).float())
        plain = torch.randn(rows, k, generator=g).to(E4M3).float()
        sign = torch.randint(0, 2, (rows, k), generator=g).float() * 2 - 1
        return torch.where(kind == 0, small, torch.where(kind == 1, large, plain)) * sign

    a, b = operand(m), operand(n)
    qa, qb = a.to(E4M3), b.to(E4M3)
    assert torch.equal(qa.float(), a) and torch.equal(qb.float(), b)
    sa = torch.full((m, -(-k // 128)), 127 - 4, dtype=torch.uint8, device=DEV).view(E8M0)
    sb = torch.full((-(-n // 128), -(-k // 128)), 127 - 3, dtype=torch.uint8, device=DEV).view(E8M0)
    got = fp8.matmul(qa.to(DEV), sa, qb.to(DEV), sb, dtype=dtype).cpu().double() * 2.0 ** 7
    a64, b64 = a.double(), b.double()
    taken = [torch.where(t == 0, 0.0, t.abs().clamp(min=2.0 ** -6)) for t in (a64, b64)]
    want, size = a64 @ b64.t(), taken[0] @ taken[1].t()
    if dtype is torch.float32:
        # Sums of r exact products in f32.
        assert ((got - want).abs() <= k * 2.0 ** -23 * (a64.abs() @ b64.abs().t())).all()
    else:
        bound = (k * 2.0 ** -23 + 2.0 ** -10) * size
        assert ((got - want).abs() <= bound + U[dtype] * (want.abs() + bound) + 2.0 ** -17).all()
