"""Microscaled and row operators on operands whose rows and batches lie further apart than 32 bits of bytes or elements reach."""
import pytest
import torch

from mx_reference import E8M0, FP4, FP8, operands, quantized, room
from vecops_amd import capi

pytestmark = pytest.mark.gpu
FAR = (1 << 31) + 64    # elements, of three rows: past 2^32 bytes whatever they are


@pytest.fixture(scope="module")
def far(device):
    """far(place, shape, dtype, apart): a tensor of uninitialised memory whose rows (or batches) are `apart` elements from one another."""
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GiB of device memory")
    memory = torch.empty(18 << 30, dtype=torch.uint8, device=device)

    def at(place, shape, dtype, apart=FAR):
        inner = [1]
        for extent in reversed(shape[2:] if len(shape) == 3 else []):
            inner.insert(0, inner[0] * extent)
        strides = [apart] + inner
        held = torch.uint8 if dtype in (FP4, E8M0, FP8) else dtype
        return memory[place << 16:].view(held).as_strided(shape, strides).view(dtype)

    yield at
    del memory
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_far_apart(device, far, dtype):
    m, k = 3, 500
    x, r, w = torch.randn(m, k).to(dtype), torch.randn(m, k).to(dtype), torch.randn(k)
    for form, scale in ((FP8, E8M0), (FP4, E8M0)):
        near_q, near_s = room((m,), k, form)
        near_out, near_summed = torch.empty(m, k, dtype=dtype, device=device), torch.empty(m, k, dtype=dtype, device=device)
        capi.rms_norm(x.to(device), w.to(device), near_q, near_s, near_out, r.to(device), near_summed)
        fx, fr, fo, fs = (far(p, (m, k), dtype) for p in (0, 1, 2, 3))
        fx.copy_(x)
        fr.copy_(r)
        fq, fsc = far(4, near_q.shape, form), far(5, near_s.shape, scale)
        capi.rms_norm(fx, w.to(device), fq, fsc, fo, fr, fs)
        same = lambda a, b: torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))  # noqa: E731
        assert torch.equal(fo, near_out) and torch.equal(fs, near_summed)
        assert same(fq.view(torch.uint8), near_q.view(torch.uint8)) and same(fsc.view(torch.uint8), near_s.view(torch.uint8))
        capi.quantize_mx(fx, fq, fsc)
        want_q, want_s = room((m,), k, form)
        capi.quantize_mx(x.to(device), want_q, want_s)
        assert same(fq.view(torch.uint8), want_q.view(torch.uint8)) and same(fsc.view(torch.uint8), want_s.view(torch.uint8))
        assert torch.equal(fsc.view(torch.uint8).cpu(), quantized(x, form)[1])
        back = torch.empty(m, k, dtype=dtype, device=device)
        capi.dequantize_mx(want_q, want_s, back)
        capi.dequantize_mx(fq, fsc, fo)
        assert torch.equal(fo, back)
        gate_q, gate_s = room((m,), k // 2, form)
        capi.silu_mul_quantize(x.to(device), gate_q, gate_s)
        gq, gs = far(6, gate_q.shape, form), far(7, gate_s.shape, scale)
        capi.silu_mul_quantize(fx, gq, gs)
        assert same(gq.view(torch.uint8), gate_q.view(torch.uint8)) and same(gs.view(torch.uint8), gate_s.view(torch.uint8))


@pytest.mark.parametrize("form", [FP4, FP8])
def test_product_of_rows_and_batches_far_apart(device, far, form):
    m, n, k = 3, 40, 1024
    a, sa = operands(m, k, form)
    b, sb = operands(n, k, FP4, seed=1)
    there = [t.to(device) for t in (a, sa, b, sb)]
    near = capi.matmul_mx(*there, torch.empty(m, n, device=device))
    fa, fsa = far(0, a.shape, form), far(1, sa.shape, E8M0)
    fa.view(torch.uint8).copy_(a.view(torch.uint8))
    fsa.view(torch.uint8).copy_(sa.view(torch.uint8))
    c = far(2, (m, n), torch.float32)
    capi.matmul_mx(fa, fsa, there[2], there[3], c)
    assert torch.equal(c, near)
    # batches: a row each
    fb, fsb = far(3, (3, n, k // 2), torch.uint8), far(5, (3, n, k // 32), torch.uint8)
    for i in range(3):
        fb[i].copy_(there[2].view(torch.uint8))
        fsb[i].copy_(there[3].view(torch.uint8))
    one = lambda t, of: t.view(torch.uint8).as_strided((3, 1, t.shape[1]), (t.stride(0), t.shape[1], 1)).view(of)  # noqa: E731
    c = far(8, (3, 1, n), torch.float32)
    capi.matmul_mx(one(fa, form), one(fsa, E8M0), fb.view(FP4), fsb.view(E8M0), c)
    assert torch.equal(c[:, 0], capi.matmul_mx(*there, torch.empty(m, n, device=device)))
