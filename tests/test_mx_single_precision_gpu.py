"""The product of e4m3 activations with results in f32: as exact as the sums in fp32 allow, whatever lies beside an element."""
import pytest
import torch

from mx_reference import E8M0, FP4, FP8, blocks, operands, values
from vecops_amd import capi

pytestmark = pytest.mark.gpu
# each kernel that sizes choose, with shares of k and without, odd ends of every extent
SIZES = [(4, 33, 544), (2, 100, 9000), (13, 17, 90), (50, 30, 70), (40, 17, 2208), (260, 17, 32), (1030, 90, 70), (1030, 19, 5200), (4100, 207, 1536),
         (4100, 113, 14560), (4100, 453, 32), (4100, 210, 10176), (2050, 4100, 224), (2050, 1083, 15712), (1, 4096, 4096), (16, 4096, 1024), (33, 100, 4096)]


def in_64_bits(device, a, sa, b, sb):
    """(the product, the sum of its terms' sizes)."""
    x, w = values(a, sa).to(device), values(b, sb).to(device)
    return x @ w.t(), x.abs() @ w.abs().t()


def within_fp32(c, want, size, k):
    """Two instructions for each 128 k, each of six additions that lose up to 2^-23 of the terms' sizes; eight wavefronts' and two shares'
    sums; products and scales are exact."""
    bound = (12 * blocks(k, 128) + 12) * 2.0 ** -23 * size
    worst = ((c.double() - want).abs() / bound).nan_to_num(0.0).max()
    assert float(worst) <= 1, f"{float(worst)} times the bound"


@pytest.mark.parametrize("m,n,k", SIZES)
def test_every_element_counts(device, m, n, k):
    a, sa = operands(m, k, FP8, seed=21, low=125, high=130)
    b, sb = operands(n, k, FP4, seed=22, low=125, high=130)
    c = torch.empty((m, n), device=device)
    capi.matmul_mx(*(t.to(device) for t in (a, sa, b, sb)), c)
    within_fp32(c, *in_64_bits(device, a, sa, b, sb), k)


@pytest.mark.parametrize("m,n,k", SIZES)
def test_the_smallest_beside_the_largest(device, m, n, k):
    """Of every eight elements one of 448, one of -448 that takes it away again, and numbers down to 2^-9: what is left is theirs, to the last bit."""
    g = torch.Generator().manual_seed(k)
    a = torch.randint(1, 16, (m, k), generator=g).to(torch.uint8)   # 2^-9 .. 15 * 2^-9
    whole = k // 8 * 8
    a[:, 0:whole:8], a[:, 5:whole:8] = 0x7e, 0xfe
    codes = torch.randint(0, 16, (n, k), generator=g)
    codes[:, 5:whole:8] = codes[:, 0:whole:8]
    b = (codes[:, 0::2] | codes[:, 1::2] << 4).to(torch.uint8).view(FP4)
    sa, sb = (torch.full((rows, blocks(k)), 127, dtype=torch.uint8).view(E8M0) for rows in (m, n))
    a = a.view(FP8)
    c = torch.empty((m, n), device=device)
    capi.matmul_mx(*(t.to(device) for t in (a, sa, b, sb)), c)
    want, _ = in_64_bits(device, a, sa, b, sb)
    assert torch.equal(c.double(), want)   # (units of 2^-10, of which even the largest sum has fewer than 2^24: 15 * 12 * 15712)


def test_elements_that_are_not_numbers(device):
    """e4m3's NaN makes its row NaN, and no other."""
    for m in (3, 16, 40, 300):
        a, sa = operands(m, 640, FP8, seed=5)
        b, sb = operands(70, 640, FP4, seed=6)
        a.view(torch.uint8)[1, 100], a.view(torch.uint8)[2, 639] = 0x7f, 0xff
        c = torch.empty((m, 70), device=device)
        capi.matmul_mx(*(t.to(device) for t in (a, sa, b, sb)), c)
        odd = torch.isnan(c)
        assert bool(odd[1:3].all()) and not bool(odd[0].any()) and not bool(odd[3:].any())
