"""More rows than one launch has workgroups for (2^20 of them): those that a workgroup comes to on its second way round the loop, and the rows beside."""
import pytest
import torch

from mx_reference import E8M0, FP4, FP8, blocks, elements, quantized, values
from test_row_operators_gpu import FORMATS, check, gate64, gate_slack, norm64, norm_slack, results
from vecops_amd import capi

pytestmark = pytest.mark.gpu


def picked(rows, first):
    """Rows at the start, around the one where the second way round begins, at the end, and between."""
    g = torch.Generator().manual_seed(rows)
    return torch.cat([torch.arange(40), torch.arange(first - 40, min(first + 40, rows)), torch.arange(rows - 40, rows), torch.randint(0, rows, (200,), generator=g),
                      torch.randint(first, rows, (60,), generator=g)]).unique()


def rows_of(t, at):
    return t.view(torch.uint8)[at.to(t.device)].cpu().view(t.dtype) if t.element_size() == 1 else t[at.to(t.device)].cpu()


# 64 threads a row, four rows a workgroup; 128 threads a row, whose wavefronts meet
LAYOUTS = [(4 * 2 ** 20 + 1003, 72, 4 * 2 ** 20), (2 ** 20 + 300, 2056, 2 ** 20)]


def need(bytes_):
    if torch.cuda.mem_get_info()[0] < bytes_:
        pytest.skip(f"needs {bytes_ >> 30} GiB of device memory")


@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("rows,k,first", LAYOUTS)
def test_norm(device, rows, k, first, form):
    """Rows that lie in one another, an element apart: each has a sum, a largest number and results of its own."""
    need(16 << 30)
    g = torch.Generator(device=device).manual_seed(3)
    line = torch.randn(rows + k, generator=g, device=device) * torch.exp(torch.randn(rows + k, generator=g, device=device))
    x = line.bfloat16().as_strided((rows, k), (1, 1))
    weight = torch.randn(k)
    q, scales = results((rows,), k, form)
    capi.rms_norm(x, weight.to(device), q=q, scales=scales, eps=1e-5)
    at = picked(rows, first)
    _, y = norm64(x[at.to(device)].cpu(), None, weight, 1e-5)
    check(rows_of(q, at), rows_of(scales, at), y, form, norm_slack(k))


def test_norm_with_the_residual(device):
    """The sum is written once a row, also by rows of a second way round."""
    rows, k, first = LAYOUTS[1]
    need(24 << 30)
    g = torch.Generator(device=device).manual_seed(4)
    x = torch.randn(rows + k, generator=g, device=device).bfloat16().as_strided((rows, k), (1, 1))
    residual = torch.randn(rows + k, generator=g, device=device).bfloat16().as_strided((rows, k), (1, 1))
    weight = torch.randn(k)
    summed, out = (torch.full((rows, k), 9.0, dtype=torch.bfloat16, device=device) for _ in range(2))
    q, scales = results((rows,), k, "int8")
    capi.rms_norm(x, weight.to(device), q=q, scales=scales, out=out, residual=residual, summed=summed, eps=1e-5)
    at = picked(rows, first)
    h, y = norm64(x[at.to(device)].cpu(), residual[at.to(device)].cpu(), weight, 1e-5)
    assert torch.equal(rows_of(summed, at).double(), h)
    slack = norm_slack(k)
    assert bool(((rows_of(out, at).double() - y).abs() <= (2.0 ** -8 + slack) * y.abs() * 1.01).all())
    check(rows_of(q, at), rows_of(scales, at), y, "int8", slack)


@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("rows,k,first", LAYOUTS)
def test_gate(device, rows, k, first, form):
    need(16 << 30)
    g = torch.Generator(device=device).manual_seed(5)
    x = (torch.randn(rows + 2 * k, generator=g, device=device) * 3).half().as_strided((rows, 2 * k), (1, 1))
    q, scales = results((rows,), k, form)
    capi.silu_mul_quantize(x, q, scales)
    at = picked(rows, first)
    some = x[at.to(device)].cpu()
    check(rows_of(q, at), rows_of(scales, at), gate64(some), form, gate_slack(some))


@pytest.mark.parametrize("form", [FP4, FP8])
def test_quantise_and_back(device, form):
    """2^30 pieces of eight elements are one way round: 2^20 rows of 8224."""
    need(60 << 30)
    rows, k, first = 2 ** 20, 8224, 2 ** 30 // (blocks(8224) * 4)
    g = torch.Generator(device=device).manual_seed(6)
    x = torch.randn(rows + k, generator=g, device=device).bfloat16().as_strided((rows, k), (1, 1))
    q = torch.full((rows, k // 2 if form == FP4 else k), 0xA5, dtype=torch.uint8, device=device).view(form)
    scales = torch.full((rows, blocks(k)), 0x7B, dtype=torch.uint8, device=device).view(E8M0)
    capi.quantize_mx(x, q, scales)
    at = picked(rows, first)
    want_q, want_s = quantized(x[at.to(device)].cpu(), form)
    assert torch.equal(rows_of(scales, at).view(torch.uint8), want_s) and torch.equal(elements(rows_of(q, at)), want_q)
    out = torch.full((rows, k), 9.0, dtype=torch.bfloat16, device=device)
    capi.dequantize_mx(q, scales, out)
    assert torch.equal(rows_of(out, at), values(rows_of(q, at), rows_of(scales, at)).float().bfloat16())
