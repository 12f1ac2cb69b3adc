"""Products of 8-bit floats whose rows are as long, or lie as far apart, as the kernels' offsets reach."""
import pytest
import torch

from vecops_amd import capi

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


def some(shape, seed):
    """e4m3 numbers, none of them a NaN, on the CPU."""
    v = torch.randint(0, 256, shape, generator=torch.Generator().manual_seed(seed)).to(torch.uint8)
    v[(v & 0x7f) == 0x7f] = 0x30
    return v.view(FP8)


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n,k,apart", [(1, 21, 700, 2 ** 27), (16, 35, 128, 2 ** 27), (80, 70, 700, 2 ** 25)])
def test_rows_far_apart(device, m, n, k, apart, out):
    """Rows of weights up to 2 GiB apart within a tile, read where they lie: the same bits as from rows side by side."""
    a, b = some((m, k), 1).to(device), some((n, k), 2).to(device)
    sa, sb = torch.ones((m, -(-k // 128)), device=device), torch.ones((1, -(-k // 128)), device=device)
    store = torch.empty(((n - 1) * apart + k,), dtype=torch.uint8, device=device)
    wide = store.as_strided((n, k), (apart, 1))
    wide.copy_(b.view(torch.uint8))
    c, d = torch.full((m, n), float("nan"), dtype=out, device=device), torch.full((m, n), float("nan"), dtype=out, device=device)
    capi.matmul_fp8_block(a, sa, b, sb, c)
    capi.matmul_fp8_block(a, sa, wide.view(FP8), sb, d)
    assert bool(torch.isfinite(c).all()) and torch.equal(c, d)


@pytest.mark.parametrize("m,n", [(1, 16), (17, 64)])
@pytest.mark.parametrize("k", [2 ** 24, 2 ** 24 + 100])
def test_long_rows(device, m, n, k):
    """A result that is the sum of a few products, at the ends of K and where offsets pass powers of two: exact in fp32."""
    at = torch.tensor([0, 1, 127, 128, 2 ** 23 - 1, 2 ** 23, k - 129, k - 101, k - 100, k - 17, k - 16, k - 1])
    numbers = some((n, len(at)), 3)
    a, b = torch.zeros((m, k), dtype=torch.uint8, device=device), torch.zeros((n, k), dtype=torch.uint8, device=device)
    one = torch.ones((), dtype=torch.float32).to(FP8).view(torch.uint8)
    a[:, at.to(device)] = one.to(device)
    b[:, at.to(device)] = numbers.view(torch.uint8).to(device)
    groups = -(-k // 128)
    c = torch.full((m, n), float("nan"), device=device)
    capi.matmul_fp8_block(a.view(FP8), torch.ones((m, groups), device=device), b.view(FP8), torch.ones((1, groups), device=device), c)
    want = numbers.double().sum(dim=1)   # (of multiples of 2^-9 up to 448: every order gives it)
    assert torch.equal(c.cpu().double(), want.expand(m, n))
