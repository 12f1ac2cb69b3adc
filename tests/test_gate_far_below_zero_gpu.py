"""The gated activation where a gate's exponential is near the end of fp32 and its result is not: blocks that hold nothing else."""
import pytest
import torch

from test_row_operators_gpu import FORMATS, check, gate64, gate_slack, results
from vecops_amd import capi

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("low,high,up", [(-84.0, -82.0, 1.0), (-88.6, -87.4, 1.0), (-92.0, -88.8, 1.0), (-92.0, -80.0, 3.0), (-104.0, -93.0, 2.0 ** 60), (-130.0, -105.0, 2.0 ** 120),
                                         (-84.0, -83.0, 2.0 ** 126)])
def test_results_that_fp32_holds(device, dtype, form, low, high, up):
    k, rows = 512, 7
    g = torch.linspace(low, high, k).repeat(rows, 1)
    u = up * (1 + torch.rand((rows, k), generator=torch.Generator().manual_seed(1)))
    x = torch.cat([g, u], dim=1).to(dtype)
    q, scales = results((rows,), k, form)
    capi.silu_mul_quantize(x.to(device), q, scales)
    y = gate64(x)
    # at least half the smallest normal number: there the last product, of which fp32 then holds multiples of 2^-149, is off by up to 2^-23 of itself, two of the
    # eight units of gate_slack (of which the exponential and the reciprocal take two each, two products one each, and the sum, of which 1 is no part, none)
    assert bool((y.abs() > 2.0 ** -127).all())
    check(q, scales, y, form, gate_slack(x))
    if form in ("fp8", "fp4"):   # what the elements stand for: nothing is lost but their rounding
        out = torch.empty((rows, k), device=device)
        capi.dequantize_mx(q, scales, out)
        assert bool((out < 0).all())
