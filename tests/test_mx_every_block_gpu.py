"""Products of small whole numbers, whose sums fp32 holds to the last bit in any order: a block left out, taken twice or scaled by another's power of
two shows in every kernel, however small a part of a result it is."""
import pytest
import torch

from conftest import launched_kernels
from mx_reference import E8M0, FP4, FP8, blocks, values
from test_mx_gpu import REAL, ROWS, SIZES, TILE
from vecops_amd import capi

pytestmark = pytest.mark.gpu


def whole_numbers(rows, k, dtype, seed):
    """Elements (e2m1: all of them; e4m3: -8 .. 8) and scales of 1 and 2."""
    g = torch.Generator().manual_seed(seed + rows * 31 + k)
    scales = torch.randint(127, 129, (rows, blocks(k)), generator=g).to(torch.uint8).view(E8M0)
    if dtype == FP8:
        return torch.randint(-8, 9, (rows, k), generator=g).float().to(FP8), scales
    return torch.randint(0, 256, (rows, k // 2), generator=g).to(torch.uint8).view(FP4), scales


def exact(device, m, n, k, form):
    """(operands there, their product).  Terms are multiples of 1/4 up to 6 * 6 * 4 (e4m3: of 1/2 up to 8 * 6 * 4): 576 units, so that any sum of 29127 of
    them lies below 2^24 units."""
    assert 576 * k < 2 ** 24
    a, sa = whole_numbers(m, k, form, 1)
    b, sb = whole_numbers(n, k, FP4, 2)
    x, w = values(a, sa).to(device), values(b, sb).to(device)
    if m * n <= 10 ** 4 and m * n * k >= 10 ** 4:   # (no block is nothing in all results)
        g = blocks(k)
        fill = lambda t: torch.nn.functional.pad(t, (0, 32 * g - k)).unflatten(1, (g, 32)).transpose(0, 1).contiguous()  # noqa: E731
        parts = torch.matmul(fill(x), fill(w).transpose(1, 2).contiguous())
        assert bool((parts != 0).flatten(1).any(dim=1).all())
    return [t.to(device) for t in (a, sa, b, sb)], x @ w.t()


@pytest.mark.parametrize("form", [FP4, FP8])
@pytest.mark.parametrize("m,n,k", [*SIZES, (2, 100, 9000), (3, 17, 2368), (4, 33, 14336), (14, 33, 96), (16, 4096, 14336), (32, 100, 14336)])
def test_sums_are_exact(device, m, n, k, form):
    there, want = exact(device, m, n, k, form)
    for dtype in REAL:
        c = torch.full((m, n), 7.0, dtype=dtype, device=device)
        capi.matmul_mx(*there, c)
        assert torch.equal(c, want.to(dtype)), dtype


@pytest.mark.parametrize("m,n,k,form,kernel", [
    (1, 17, 96, FP4, ROWS(16, 4, 0, 2, 1)), (4, 33, 544, FP8, ROWS(16, 4, 1, 2, 1)), (3, 17, 2368, FP4, ROWS(16, 4, 0, 4, 2)), (2, 100, 9000, FP8, ROWS(16, 4, 1, 4, 2)),
    (50, 30, 70, FP8, ROWS(16, 16, 1, 4, 1)), (17, 16, 32, FP4, ROWS(16, 16, 0, 4, 1)), (40, 100, 5000, FP4, ROWS(16, 16, 0, 4, 2)), (40, 17, 2208, FP8, ROWS(16, 16, 1, 8, 1)),
    (260, 17, 32, FP4, ROWS(32, 32, 0, 4, 1)), (260, 17, 32, FP8, ROWS(32, 32, 1, 4, 1)), (1030, 19, 4928, FP4, TILE(1, 2, 2, 2, 1, 0)), (1030, 19, 5200, FP8, TILE(1, 2, 2, 2, 1, 1)),
    (4100, 248, 2400, FP4, TILE(2, 1, 2, 2, 2, 0)), (4100, 113, 14560, FP8, TILE(2, 1, 2, 2, 2, 1)), (4100, 453, 32, FP4, TILE(2, 2, 1, 2, 2, 0)),
    (4100, 210, 10176, FP4, TILE(2, 2, 2, 2, 2, 0)), (4100, 210, 10176, FP8, TILE(2, 2, 2, 2, 2, 1)), (4100, 3257, 1312, FP4, TILE(2, 2, 1, 4, 4, 0)),
    (2050, 2041, 12288, FP4, TILE(2, 2, 1, 4, 4, 0)), (2050, 4100, 224, FP8, TILE(2, 2, 1, 4, 2, 1)), (2050, 1083, 15712, FP8, TILE(2, 2, 1, 4, 2, 1))])
def test_sums_of_every_kernel_are_exact(device, m, n, k, form, kernel):
    there, want = exact(device, m, n, k, form)
    for dtype in REAL:
        c = torch.full((m, n), 7.0, dtype=dtype, device=device)
        names = launched_kernels(lambda c=c: capi.matmul_mx(*there, c))
        assert any(name.startswith(kernel) for name in names), names
        assert torch.equal(c, want.to(dtype)), dtype


@pytest.mark.parametrize("m", [1, 4, 16, 40])
@pytest.mark.parametrize("k", [512, 544, 9000, 14336])
def test_one_element_of_each_block(device, m, k):
    """Activations with one number in a block, each at another place and of another size (e4m3), weights of 1 and scales that bring every block's term to
    a power of two of its own among 2^0 .. 2^7: the sum names the blocks."""
    g, n = blocks(k), 33
    at = torch.arange(g) * 32 + torch.arange(g) * 7 % torch.where(torch.arange(g) == g - 1, k - 32 * (g - 1), 32)
    a = torch.zeros(m, k)
    size = torch.exp2((torch.arange(g) % 15 - 6).float())
    a[:, at] = size
    power = torch.arange(g) % 8
    sa = (127 + power - torch.log2(size).long()).to(torch.uint8).repeat(m, 1).view(E8M0)
    b = torch.full((n, k // 2), 0x22, dtype=torch.uint8).view(FP4)
    sb = torch.full((n, g), 127, dtype=torch.uint8).view(E8M0)
    want = float(torch.exp2(power.float()).sum())
    for dtype in REAL:
        c = torch.empty((m, n), dtype=dtype, device=device)
        capi.matmul_mx(*(t.to(device) for t in (a.to(FP8), sa, b, sb)), c)
        assert bool((c == torch.tensor(want).to(dtype).to(device)).all()), (dtype, want)
