"""8-bit floats with a scale for each block of 128: the quantiser bit for bit, the product against 64-bit sums."""
import numpy as np
import pytest
import torch

from vecops_amd import capi

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


def blocks(extent):
    return -(-extent // 128)


def quantized(x, rows):
    """The definition, on the CPU: the quotients are correctly rounded (a 64-bit quotient of fp32 numbers rounds to fp32
    without harm), then to the nearest e4m3 by torch's CPU conversion."""
    x = x.double().cpu()
    m, k = x.shape[-2:]
    scales = torch.empty((*x.shape[:-2], -(-m // rows), blocks(k)), dtype=torch.float32)
    q = torch.empty(x.shape, dtype=FP8)
    for i in range(scales.shape[-2]):
        for g in range(scales.shape[-1]):
            at = (..., slice(i * rows, (i + 1) * rows), slice(g * 128, (g + 1) * 128))
            part = x[at]
            s = (part.abs().amax(dim=(-1, -2)) / 448).float().clamp(min=2.0 ** -126)
            scales[..., i, g] = s
            q[at] = (part / s.double()[..., None, None]).float().to(FP8)
    return q, scales


def same_quantized(got_q, got_s, want_q, want_s):
    assert np.array_equal(got_s.cpu().numpy(), want_s.numpy(), equal_nan=True)
    got, want = got_q.cpu().view(torch.uint8), want_q.view(torch.uint8)
    nan = (want & 0x7f) == 0x7f
    assert torch.equal((got & 0x7f) == 0x7f, nan)
    assert torch.equal(got[~nan], want[~nan])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape,rows", [((1, 128), 1), ((1, 1), 1), ((5, 300), 1), ((33, 1000), 1), ((3, 7, 129), 1), ((260, 4096), 1),
                                        ((1, 1), 128), ((128, 128), 128), ((129, 257), 128), ((2, 200, 300), 128), ((300, 4001), 128)])
def test_quantize(device, dtype, shape, rows):
    torch.manual_seed(hash((shape, rows)) % 1000)
    x = (torch.randn(shape) * torch.exp(torch.randn(shape[-1]) * 3)).to(dtype)
    want_q, want_s = quantized(x, rows)
    q = torch.empty(shape, dtype=FP8, device=device)
    scales = torch.empty(want_s.shape, device=device)
    capi.quantize_fp8_block(x.to(device), q, scales, block_rows=rows)
    same_quantized(q, scales, want_q, want_s)


@pytest.mark.parametrize("rows", [1, 128])
def test_quantize_numbers_at_the_edges(device, rows):
    """Zeros, one number alone, the smallest and largest fp32 numbers, halves between neighbouring e4m3 numbers, infinities
    and NaN in one block of many."""
    line = torch.zeros(14, 128)
    line[1, 5] = -3.0
    line[2] = torch.arange(128) * 2.0 ** -149
    line[3] = torch.arange(1, 129) * 2.0 ** -133
    line[4] = torch.finfo(torch.float32).max * torch.linspace(-1, 1, 128)
    line[5] = torch.linspace(-448, 448, 128)                          # the scale is 1
    line[6] = 2.0 ** -10 * torch.arange(128)
    line[6, 0] = 448.0                                                # ties among the subnormal numbers
    line[7] = (torch.arange(128) + 0.5) * 2.0
    line[7, 0] = 448.0                                                # ties among the normal ones
    line[8] = torch.randn(128)
    line[8, 77] = float("inf")
    line[9, 3] = float("-inf")
    line[10] = torch.randn(128)
    line[10, 127] = float("nan")
    line[11] = 2.0 ** -126 * torch.linspace(0, 500, 128)
    line[12] = torch.exp(torch.linspace(-87, 0, 128)) * 1e30
    line[13] = torch.randn(128) * 1e-30
    x = line if rows == 1 else line.repeat_interleave(128, dim=0)[:, torch.randperm(128)]
    want_q, want_s = quantized(x, rows)
    q, scales = torch.empty(x.shape, dtype=FP8, device=device), torch.empty(want_s.shape, device=device)
    capi.quantize_fp8_block(x.to(device), q, scales, block_rows=rows)
    same_quantized(q, scales, want_q, want_s)


@pytest.mark.parametrize("rows", [1, 128])
def test_quantize_strides(device, rows):
    """Padded rows, a transposed source, a transposed result, scales stored the other way round; nothing else is written."""
    torch.manual_seed(3)
    m, k = 150, 333
    x = torch.randn(m, k)
    want_q, want_s = quantized(x, rows)
    for source in ("padded", "transposed"):
        if source == "padded":
            xs = torch.full((m, k + 7), float("nan"), device=device)
            xs[:, 3:3 + k] = x.to(device)
            xv = xs[:, 3:3 + k]
        else:
            xv = x.t().contiguous().to(device).t()
        q_store = torch.full((k + 2, m + 5), 77, dtype=torch.uint8, device=device)
        s_store = torch.full((want_s.shape[1] + 1, want_s.shape[0] + 2), -1.0, device=device)
        q, scales = q_store.view(FP8)[1:1 + k, 2:2 + m].t(), s_store[:-1, 1:-1].t()
        capi.quantize_fp8_block(xv, q, scales, block_rows=rows)
        same_quantized(q.contiguous(), scales, want_q, want_s)
        q_store[1:1 + k, 2:2 + m] = 77
        s_store[:-1, 1:-1] = -1.0
        assert bool((q_store == 77).all()) and bool((s_store == -1.0).all())


def operands(m, n, k, batch=(), seed=0):
    """e4m3 operands and scales on the CPU: all finite numbers of the type, scales over six powers of ten."""
    g = torch.Generator().manual_seed(seed + m * 31 + n * 7 + k)
    def bytes_(*shape):
        v = torch.randint(0, 256, shape, generator=g, dtype=torch.int64).to(torch.uint8)
        v[(v & 0x7f) == 0x7f] = 0x38
        return v.view(FP8)
    a, b = bytes_(*batch, m, k), bytes_(*batch, n, k)
    sa = torch.exp(torch.randn((*batch, m, blocks(k)), generator=g) * 2)
    sb = torch.exp(torch.randn((*batch, blocks(n), blocks(k)), generator=g) * 2)
    return a, sa, b, sb


def dequantized(q, scales, rows):
    m, k = q.shape[-2:]
    wide = scales.double().repeat_interleave(rows, dim=-2)[..., :m, :].repeat_interleave(128, dim=-1)[..., :k]
    return q.double() * wide


def check(c, a, sa, b, sb):
    """|error| <= (terms of the inner sum + roundings of the scales and of the outer sum) 2^-24 times the sum of the terms'
    sizes, and the rounding of the result.  16-bit results come from the 8-bit matrix instruction: of
    eight products along k the seven smaller ones may each lose 2^-13 of the largest's power of two."""
    x, w = dequantized(a, sa, 1), dequantized(b, sb, 128)
    want, size = x @ w.transpose(-1, -2), x.abs() @ w.abs().transpose(-1, -2)
    k = a.shape[-1]
    bound = (min(k, 128) + 3 + blocks(k)) * 2.0 ** -24 * size
    if c.dtype != torch.float32:
        bound = bound + 7 * 2.0 ** -13 * size
    unit = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[c.dtype]
    bound = bound + unit * (want.abs() + bound) + (2.0 ** -25 if c.dtype == torch.float16 else 0.0)
    got = c.double().cpu()
    if c.dtype == torch.float16:   # past the largest number the rounding gives infinity
        far = want.abs() - bound > 65519
        assert bool(torch.isinf(got[far]).all())
        near = want.abs() + bound < 65519
        got, want, bound = got[near], want[near], bound[near]
    assert bool(((got - want).abs() <= bound).all()), f"{((got - want).abs() / bound).max()} times the bound"


SIZES = [(1, 16, 128), (1, 1, 1), (1, 4096, 4096), (3, 100, 127), (16, 256, 1024), (7, 513, 16 * 1024 + 40), (17, 200, 300), (32, 128, 640),
         (33, 1000, 513), (64, 512, 17000), (65, 130, 256), (100, 257, 1000), (128, 384, 129), (130, 640, 16), (200, 300, 2049),
         (777, 500, 130), (1100, 4400, 384), (4096, 4100, 200), (9, 40, 5), (90, 300, 7), (70, 200, 15), (66, 129, 17), (5, 33, 31), (257, 513, 143),
         (3000, 6000, 128), (2900, 6001, 4097), (64, 1000, 14336), (100, 513, 4109), (300, 700, 2304), (128, 2000, 8192),
         (500, 5000, 1000), (900, 3000, 700), (2049, 2049, 257)]


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16, torch.float16])
def test_matmul(device, m, n, k, out):
    a, sa, b, sb = operands(m, n, k)
    c = torch.full((m, n), float("nan"), dtype=out, device=device)
    capi.matmul_fp8_block(a.to(device), sa.to(device), b.to(device), sb.to(device), c)
    check(c, a, sa, b, sb)


@pytest.mark.parametrize("m,n,k", [(5, 150, 300), (40, 150, 300), (150, 330, 300), (300, 200, 1000)])
def test_matmul_strides(device, m, n, k):
    """Operands inside larger ones whose other bytes are NaN, rows at odd addresses; k that is not contiguous on either side;
    scales and results stored the other way round."""
    a, sa, b, sb = operands(m, n, k)

    def inside(t, offset):
        store = torch.full((t.shape[0] + 2, t.shape[1] + 9), 0x7f, dtype=torch.uint8, device=device)
        view = store[1:-1, offset:offset + t.shape[1]]
        view.copy_(t.view(torch.uint8).to(device))
        return view.view(FP8)

    def turned(t):
        return t.view(torch.uint8).t().contiguous().to(device).t().view(FP8)

    for make_a, make_b in ((lambda t: inside(t, 3), lambda t: inside(t, 5)), (turned, lambda t: inside(t, 1)), (lambda t: inside(t, 0), turned),
                           (turned, turned)):
        store = torch.full((n + 1, m + 3), -5.0, device=device)
        c = store[:-1, 2:-1].t()
        capi.matmul_fp8_block(make_a(a), sa.t().contiguous().to(device).t(), make_b(b), sb.t().contiguous().to(device).t(), c)
        check(c, a, sa, b, sb)
        store[:-1, 2:-1] = -5.0
        assert bool((store == -5.0).all())


@pytest.mark.parametrize("m", [2, 20, 70])
def test_matmul_batches(device, m):
    """Rank 3, weights shared by all batches, and activations shared."""
    a, sa, b, sb = operands(m, 140, 260, batch=(3,))
    dev = [t.to(device) for t in (a, sa, b, sb)]
    c = torch.full((3, m, 140), float("nan"), device=device)
    capi.matmul_fp8_block(*dev, c)
    check(c, a, sa, b, sb)
    shared = [t[:1].expand(3, *t.shape[1:]) for t in (b, sb)]
    capi.matmul_fp8_block(dev[0], dev[1], dev[2][:1].expand(3, -1, -1), dev[3][:1].expand(3, -1, -1), c)
    check(c, a, sa, *shared)
    turned = dev[0].view(torch.uint8)[0].t().contiguous().t().view(FP8)[None].expand(3, -1, -1)
    capi.matmul_fp8_block(turned, dev[1][:1].expand(3, -1, -1), dev[2], dev[3], c)
    check(c, a[:1].expand(3, -1, -1), sa[:1].expand(3, -1, -1), b, sb)


@pytest.mark.parametrize("m", [0, 1, 20, 80])
def test_matmul_without_work(device, m):
    """No rows, no columns, no batches: nothing is written; no k: zeros."""
    f = lambda *s: torch.empty(s, dtype=FP8, device=device)  # noqa: E731
    z = lambda *s: torch.empty(s, device=device)  # noqa: E731
    c = torch.full((m, 50), 3.0, device=device)
    capi.matmul_fp8_block(f(m, 0), z(m, 0), f(50, 0), z(1, 0), c)
    assert bool((c == 0).all())
    capi.matmul_fp8_block(f(m, 64), z(m, 1), f(0, 64), z(0, 1), torch.empty((m, 0), device=device))
    capi.matmul_fp8_block(f(0, m, 64), z(0, m, 1), f(0, 50, 64), z(0, 1, 1), torch.empty((0, m, 50), device=device))
    capi.quantize_fp8_block(torch.empty((m, 0), device=device), f(m, 0), z(m, 0))


@pytest.mark.parametrize("m,n,k", [(4, 200, 512), (100, 300, 512), (300, 40000, 256)])
def test_matmul_not_finite(device, m, n, k):
    """A NaN element, and an infinite scale, reach the results of their row (their 128 columns) and no others."""
    a, sa, b, sb = operands(m, n, k)
    a, b = a.float().clamp(-16, 16).to(FP8), b.float().clamp(-16, 16).to(FP8)
    a.view(torch.uint8)[1, 7] = 0x7f
    b.view(torch.uint8)[130, k - 1] = 0xff
    sb[0, 1] = float("inf")
    sa[2, 0] = float("nan")
    c = torch.zeros((m, n), device=device)
    capi.matmul_fp8_block(a.to(device), sa.to(device), b.to(device), sb.to(device), c)
    bad = torch.zeros((m, n), dtype=torch.bool)
    bad[1], bad[2], bad[:, 130], bad[:, :128] = True, True, True, True
    assert torch.equal(~torch.isfinite(c.cpu()), bad)


def test_matmul_the_same_every_time_and_on_another_stream(device):
    for m in (3, 50, 300):
        a, sa, b, sb = (t.to(device) for t in operands(m, 1000, 2000))
        c = torch.empty((m, 1000), device=device)
        capi.matmul_fp8_block(a, sa, b, sb, c)
        torch.cuda.synchronize()
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(3):
                again = torch.empty_like(c)
                capi.matmul_fp8_block(a, sa, b, sb, again)
        stream.synchronize()
        assert torch.equal(again, c)


@pytest.mark.parametrize("out,unit", [(torch.bfloat16, 2.0 ** -8 / 3 ** 0.5), (torch.float16, 2.0 ** -11 / 3 ** 0.5), (torch.float32, 2.0 ** -20)])
@pytest.mark.parametrize("m,n,k", [(8, 300, 2048), (200, 256, 2048), (2100, 8300, 640)])
def test_matmul_as_a_whole(device, m, n, k, out, unit):
    """Normally distributed operands: the error's 2-norm stays below that of the result's rounding (evenly distributed up
    to a half of its last place), and for 16-bit results 2^-14 besides (of eight products seven lose up to 2^-13 of the largest, to either side of a product: less
    than a fourth of that by root mean square over a sum's terms, which are of the largest's size on the whole)."""
    g = torch.Generator(device=device).manual_seed(1)
    x, w = torch.randn((m, k), generator=g, device=device), torch.randn((n, k), generator=g, device=device)
    a, sa = torch.empty((m, k), dtype=FP8, device=device), torch.empty((m, blocks(k)), device=device)
    b, sb = torch.empty((n, k), dtype=FP8, device=device), torch.empty((blocks(n), blocks(k)), device=device)
    capi.quantize_fp8_block(x, a, sa)
    capi.quantize_fp8_block(w, b, sb, block_rows=128)
    c = torch.empty((m, n), dtype=out, device=device)
    capi.matmul_fp8_block(a, sa, b, sb, c)
    want = dequantized(a, sa, 1) @ dequantized(b, sb, 128).t()
    more = 2.0 ** -14 if out != torch.float32 else 0.0
    assert float((c.double() - want).norm() / want.norm()) < unit + more


def test_quantize_then_multiply(device):
    """The two together, as a layer uses them: within what rounding both sides to e4m3 (a half of 2^-3 of each number) gives."""
    torch.manual_seed(0)
    m, n, k = 48, 384, 1024
    x, w = torch.randn(m, k), torch.randn(n, k) * k ** -0.5
    a, sa = torch.empty((m, k), dtype=FP8, device=device), torch.empty((m, blocks(k)), device=device)
    b, sb = torch.empty((n, k), dtype=FP8, device=device), torch.empty((blocks(n), blocks(k)), device=device)
    capi.quantize_fp8_block(x.bfloat16().to(device), a, sa)
    capi.quantize_fp8_block(w.bfloat16().to(device), b, sb, block_rows=128)
    c = torch.empty((m, n), dtype=torch.bfloat16, device=device)
    capi.matmul_fp8_block(a, sa, b, sb, c)
    off = (c.double().cpu() - x.double() @ w.double().t())
    assert float(off.abs().max()) < 6 * 2 ** 0.5 * 2 ** -4
    check(c, a.cpu(), sa.cpu(), b.cpu(), sb.cpu())
