"""GPU tests of the 8-bit product's tiles over rows that are long enough for their steady loops (eight rounds of the 128 and 256
wide tiles, four of the 64 wide one), with ragged edges, every type of result, bias and scales.

Exact: factors of at most 3 (one of 127 in a row that is quantized), powers of two as scales and whole numbers as bias give sums
below 2^24, which fp32 holds, so what is left is one rounding to the result's type - the reference's as well."""
import pytest
import torch

from tests.test_gpu_dense_ops import TYPES, gen

pytestmark = pytest.mark.gpu

# 16 x 16 (of 8 waves), 64 x 64, 128 x 128 and 256 x 256 tiles, by the rule in gemm_i8.hip
SIZES = [(40, 200, 2048), (200, 130, 4700), (515, 300, 2500), (700, 500, 2048), (690, 500, 4600), (2100, 700, 512), (2050, 770, 1090),
         (2100, 700, 2111), (8100, 1500, 512), (8100, 1500, 575), (8000, 1537, 1088), (8100, 1500, 2111), (16400, 1030, 4096)]


@pytest.fixture(scope="module")
def ops():
    from scarches_amd import ops as m
    return m


def small(rows, k, seed, pitch):
    """Whole numbers from -3 to 3 in rows of a pitch, other ones behind their ends."""
    v = torch.full((rows, pitch), 100, dtype=torch.int8, device="cuda")[:, :k]
    return v.random_(-3, 4, generator=gen(seed))


def powers(n, seed):
    return torch.exp2(torch.randint(-2, 3, (n,), device="cuda", generator=gen(seed)).float())


@pytest.mark.parametrize("m,n,k", SIZES)
def test_product(ops, m, n, k):
    whole = -(-k // 128) * 128
    sx, sw = powers(m, 3), powers(n, 4)
    bias = torch.randint(-9, 10, (n,), device="cuda", generator=gen(5)).float()
    for px, pw in ((whole, whole), (k, k), (k + 5, whole)):         # aligned rows, packed ones, an odd pitch
        xq, wq = small(m, k, 1, px), small(n, k, 2, pw)
        sums = xq.float() @ wq.float().t().contiguous()
        assert sums.abs().max() < 2 ** 18
        want = sums * sx[:, None] * sw
        assert torch.equal(ops.int8_matmul(xq, sx, wq, sw), want), (px, pw)
        for out in TYPES:
            assert torch.equal(ops.int8_matmul(xq, sx, wq, sw, bias.to(out), out), (want + bias).to(out)), (px, pw, out)
        assert torch.equal(ops.int8_matmul(xq, sx, wq, sw, bias, torch.bfloat16), (want + bias).bfloat16()), (px, pw)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m,n,k", SIZES + [(1, 300, 4100), (2, 300, 8064), (2, 300, 9000), (600, 2100, 777), (900, 333, 20001)])
def test_linear(ops, m, n, k, dtype):
    """Rows quantized on the way (scale 1), weights as they come: in padded rows, packed, from an odd address, transposed."""
    x = small(m, k, 1, k).to(dtype)
    x[:, k // 2] = 127
    wq = small(n, k, 2, -(-k // 128) * 128)
    sw = powers(n, 4)
    want = (x.float() @ wq.float().t().contiguous()) * sw
    buf = torch.full((n * (k + 7) + 1,), -128, dtype=torch.int8, device="cuda")
    for w in (wq, wq.contiguous(), torch.as_strided(buf, (n, k), (k + 7, 1), 1).copy_(wq), wq.t().contiguous().t()):
        assert torch.equal(ops.int8_linear(x, w, sw), want.to(dtype)), w.stride()
