"""Rows without elements: the row operators and quantisers write nothing, as their header says, scales of int8 rows included."""
import pytest
import torch

from test_row_operators_gpu import FORMATS, results
from vecops_amd import capi

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("lead", [(5,), (2, 3)])
def test_nothing_is_written(device, form, lead):
    x = torch.empty((*lead, 0), dtype=torch.bfloat16, device=device)
    q, _ = results(lead, 0, form if form != "int8" else "fp8")
    scales = torch.full((*lead, 1), -1.0, device=device) if form == "int8" else results(lead, 0, form)[1]
    if form == "int8":
        q = torch.empty((*lead, 0), dtype=torch.int8, device=device)
    before = scales.view(torch.uint8).clone()
    out, summed = torch.empty_like(x), torch.empty_like(x)
    assert capi.rms_norm(x, torch.empty(0, device=device), q=q, scales=scales, out=out, residual=x.clone(), summed=summed) == (q, scales, out)
    capi.silu_mul_quantize(x, q, scales)
    if form in ("fp8", "fp4"):
        capi.quantize_mx(x, q, scales)
        capi.dequantize_mx(q, scales, out)
    torch.cuda.synchronize()
    assert torch.equal(scales.view(torch.uint8), before)
