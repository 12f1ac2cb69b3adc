"""Which kernel sizes choose where the rule has a step: the launch that the largest tiles need for rows of fewer than sixteen scales."""
import pytest
import torch

from conftest import launched_kernels
from mx_reference import FP4, FP8, blocks, operands, values
from test_mx_gpu import TILE
from vecops_amd import capi

pytestmark = pytest.mark.gpu
LARGEST = TILE(2, 2, 1, 4, 2, 1)


@pytest.mark.parametrize("m,n,k,kernels", [(1024, 4608, 512, [LARGEST]), (384, 12288, 512, [LARGEST]), (2304, 2048, 512, [LARGEST]),
                                           (2050, 4100, 480, ["mx_copies_kernel", LARGEST]), (2050, 4100, 490, ["mx_copies_kernel", LARGEST])])
def test_sixteen_scales_a_row_are_read_in_place(device, m, n, k, kernels):
    """Rows of sixteen scales (K of 512, or of 481 and more) need no launch that lays them out, and none is counted (1024 x 4608 x 512 10.2 us
    in the largest tiles, 14.0 in those of 64 x 64)."""
    a, sa = operands(m, k, FP8, seed=31, low=125, high=130)
    b, sb = operands(n, k, FP4, seed=32, low=125, high=130)
    there = [t.to(device) for t in (a, sa, b, sb)]
    c = torch.empty((m, n), dtype=torch.bfloat16, device=device)
    names = launched_kernels(lambda: capi.matmul_mx(*there, c))
    assert len(names) == len(kernels) and all(name.startswith(kernel) for name, kernel in zip(names, kernels)), names
    x, w = values(a, sa).to(device), values(b, sb).to(device)
    want, size = x @ w.t(), x.abs() @ w.abs().t()
    # of eight products seven may lose 2^-13 of the largest; six additions an instruction; the result's rounding
    bound = (7 * 2.0 ** -13 + (6 * blocks(k, 128) + 12) * 2.0 ** -23) * size
    assert bool(((c.double() - want).abs() <= bound + 2.0 ** -8 * (want.abs() + bound)).all())
