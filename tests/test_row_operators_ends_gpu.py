"""Rows without elements, of which the row operators and quantisers write nothing, scales of int8 rows included, and rows whose squares fp32 does not hold."""
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


@pytest.mark.parametrize("form", FORMATS)
def test_squares_past_fp32(device, form):
    """A sum of squares that fp32 does not hold: its row becomes zeros, as the header says, and the rows beside it stay."""
    x = torch.randn((3, 640), generator=torch.Generator().manual_seed(1)).to(device)
    x[1, 77] = 1e20
    weight = torch.ones(640, device=device)
    found = []
    for rows in (x, x[0::2].contiguous()):
        q, scales = results(rows.shape[:1], 640, form)
        out = torch.empty_like(rows)
        capi.rms_norm(rows, weight, q=q, scales=scales, out=out)
        found.append((out, q.view(torch.uint8), scales.view(torch.uint8)))
    assert bool((found[0][0][1] == 0).all()) and bool(torch.isfinite(found[0][0]).all())
    for some, others in zip(*found):
        assert torch.equal(some[0::2], others)
