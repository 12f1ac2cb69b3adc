"""Microscaled floats: the quantiser bit for bit and its way back, the product against 64-bit sums."""
import numpy as np
import pytest
import torch

from conftest import launched_kernels
from mx_reference import E8M0, FP4, FP8, blocks, elements, operands, quantized, room, values, width
from vecops_amd import capi

pytestmark = pytest.mark.gpu
REAL = [torch.bfloat16, torch.float16, torch.float32]


def same(q, scales, want_q, want_bytes):
    assert torch.equal(scales.cpu().contiguous().view(torch.uint8), want_bytes)
    got = elements(q.cpu().contiguous())
    assert torch.equal(got, want_q)
    assert torch.equal(torch.signbit(got), torch.signbit(want_q))


@pytest.mark.parametrize("dtype", REAL)
@pytest.mark.parametrize("form", [FP4, FP8])
@pytest.mark.parametrize("shape", [(1, 32), (1, 2), (5, 30), (33, 1000), (3, 7, 130), (260, 4096), (1, 34), (4, 6), (2, 1, 62)])
def test_quantize(device, dtype, form, shape):
    torch.manual_seed(sum(shape))
    x = (torch.randn(shape) * torch.exp(torch.randn(shape[-1]) * 3)).to(dtype)
    q, scales = room(shape[:-1], shape[-1], form)
    assert capi.quantize_mx(x.to(device), q, scales) == (q, scales)
    same(q, scales, *quantized(x, form))


def test_quantize_odd_rows_of_eight_bits(device):
    x = torch.randn(3, 45)
    q, scales = room((3,), 45, FP8)
    capi.quantize_mx(x.to(device), q, scales)
    same(q, scales, *quantized(x, FP8))


@pytest.mark.parametrize("form", [FP4, FP8])
def test_quantize_numbers_at_the_edges(device, form):
    """Zeros, the smallest and largest fp32 numbers, numbers halfway between neighbours, past the largest, infinities and NaN."""
    line = torch.zeros(16, 32)
    line[1, 5] = -3.0
    line[2] = torch.arange(32) * 2.0 ** -149
    line[3] = torch.arange(1, 33) * 2.0 ** -133
    line[4] = torch.finfo(torch.float32).max * torch.linspace(-1, 1, 32)
    line[5] = torch.arange(32) * 0.25                                 # every number of e2m1, and between
    line[6] = -torch.arange(32) * 0.25
    line[7] = torch.linspace(4.0, 7.999, 32)                          # past 6
    line[8] = torch.linspace(256, 511, 32)                            # past 448
    line[9] = 2.0 ** -10 * torch.arange(32)
    line[9, 0] = 256.0                                                # ties among e4m3's subnormal numbers
    line[10] = (torch.arange(32) + 0.5) * 2.0
    line[10, 0] = 256.0
    line[11] = torch.randn(32)
    line[11, 7] = float("inf")
    line[12, 3] = float("-inf")
    line[13] = torch.randn(32)
    line[13, 31] = float("nan")
    line[14] = 2.0 ** -126 * torch.linspace(0, 7, 32)
    line[15] = torch.exp(torch.linspace(-87, 0, 32)) * 1e30
    q, scales = room((16,), 32, form)
    capi.quantize_mx(line.to(device), q, scales)
    want_q, want = quantized(line, form)
    same(q, scales, want_q, want)
    out = torch.empty(16, 32, device=device)
    capi.dequantize_mx(q, scales, out)
    assert torch.equal(torch.isnan(out).any(dim=1).cpu(), want[:, 0] == 255)


@pytest.mark.parametrize("form", [FP4, FP8])
def test_quantize_strides(device, form):
    """Padded rows, a transposed source, a transposed result, scales stored the other way round; nothing else is written."""
    torch.manual_seed(3)
    m, k = 50, 334
    w = width(form, k)
    x = torch.randn(m, k)
    want = quantized(x, form)
    for source in ("padded", "transposed"):
        if source == "padded":
            xs = torch.full((m, k + 7), float("nan"), device=device)
            xs[:, 3:3 + k] = x.to(device)
            xv = xs[:, 3:3 + k]
        else:
            xv = x.t().contiguous().to(device).t()
        q_store = torch.full((w + 2, m + 5), 77, dtype=torch.uint8, device=device)
        s_store = torch.full((blocks(k) + 1, m + 2), 99, dtype=torch.uint8, device=device)
        q, scales = q_store.view(form)[1:1 + w, 2:2 + m].t(), s_store.view(E8M0)[:-1, 1:-1].t()
        capi.quantize_mx(xv, q, scales)
        same(q_store[1:1 + w, 2:2 + m].t().contiguous().view(form), s_store[:-1, 1:-1].t().contiguous().view(E8M0), *want)
        out = torch.full((k + 1, m + 3), -5.0, device=device)
        capi.dequantize_mx(q, scales, out[:-1, 2:-1].t())
        assert torch.equal(out[:-1, 2:-1].t().double().cpu(), values(q_store[1:1 + w, 2:2 + m].t().contiguous().view(form),
                                                                     s_store[:-1, 1:-1].t().contiguous().view(E8M0)))
        out[:-1, 2:-1] = -5.0
        q_store[1:1 + w, 2:2 + m] = 77
        s_store[:-1, 1:-1] = 99
        assert bool((q_store == 77).all()) and bool((s_store == 99).all()) and bool((out == -5.0).all())


@pytest.mark.parametrize("dtype", REAL)
@pytest.mark.parametrize("form", [FP4, FP8])
def test_dequantize_every_element_and_scale(device, dtype, form):
    """Every byte with every scale: one rounding of the product, NaN where the scale or the element is."""
    q = torch.arange(256, dtype=torch.int64).to(torch.uint8).view(1, 256).repeat(256, 1)
    bytes_ = torch.arange(256, dtype=torch.int64).to(torch.uint8).view(256, 1).repeat(1, blocks(256 if form == FP8 else 512))
    out = torch.empty((256, 256 if form == FP8 else 512), dtype=dtype, device=device)
    capi.dequantize_mx(q.view(form).to(device), bytes_.view(E8M0).to(device), out)
    want = values(q.view(form), bytes_.view(E8M0)).float()   # (fp32 holds the products but for e4m3 under 2^-149, which no type here has)
    want = want.to(dtype)
    assert np.array_equal(out.cpu().float().numpy(), want.float().numpy(), equal_nan=True)


def check(c, a, sa, b, sb):
    """|error| <= what the additions can lose, times the sum of the terms' sizes, and the rounding of the result.  An instruction adds
    four blocks' sums to the accumulator, or twice two: each of the five or six may lose a unit of the sum's last place in fp32, 2^-23 of the sizes;
    then up to eight wavefronts' and two shares of k are added.  With e4m3 operands, of eight products along k the seven smaller ones may each lose
    2^-13 of the largest's power of two."""
    x, w = values(a, sa), values(b, sb)
    want, size = x @ w.transpose(-1, -2), x.abs() @ w.abs().transpose(-1, -2)
    bound = (6 * blocks(x.shape[-1], 128) + 12) * 2.0 ** -23 * size
    if a.dtype == FP8:
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


def only(t, rows):
    return t.view(torch.uint8)[rows].view(t.dtype)


SIZES = [(1, 16, 128), (1, 1, 2), (1, 4096, 4096), (3, 100, 126), (16, 256, 1024), (7, 513, 16 * 1024 + 40), (17, 200, 300), (32, 128, 640),
         (33, 1000, 514), (64, 512, 17024), (65, 130, 256), (100, 257, 1000), (128, 384, 160), (130, 640, 16), (200, 300, 2050),
         (777, 500, 130), (1100, 4400, 384), (2050, 4100, 224), (9, 40, 6), (90, 300, 8), (70, 200, 32), (66, 129, 64), (5, 33, 96), (257, 513, 144),
         (3000, 6000, 128), (1500, 3001, 4128), (64, 1000, 14336), (100, 513, 4110), (300, 700, 2304), (128, 2000, 8192),
         (16, 15, 288), (2, 17, 544), (512, 512, 512), (300, 300, 288)]


@pytest.mark.parametrize("form", [FP4, FP8])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_matmul(device, m, n, k, form):
    a, sa = operands(m, k, form)
    b, sb = operands(n, k, FP4, seed=1)
    there = [t.to(device) for t in (a, sa, b, sb)]
    for dtype in (torch.float32, torch.bfloat16) if m * n > 10 ** 6 else REAL:
        store = torch.full((m + 1, n + 3), 7.0, dtype=dtype, device=device)
        c = store[:m, :n]
        assert capi.matmul_mx(*there, c) is c
        check(c, a, sa, b, sb)
        c.fill_(7.0)
        assert bool((store == 7.0).all())


ROWS = lambda *of: f"mx_slim_kernel<{','.join(map(str, of))}>"  # noqa: E731  (weight rows, activation rows, e4m3, wavefronts, places)
TILE = lambda *of: f"mx_tile_kernel<{','.join(map(str, of))}"  # noqa: E731  (wavefronts, blocks of 32 a wavefront, e4m3)


@pytest.mark.parametrize("m,n,k,form,kernel,shares", [
    (1, 17, 96, FP4, ROWS(16, 4, 0, 2, 1), 0), (4, 33, 544, FP8, ROWS(16, 4, 1, 2, 1), 0), (3, 17, 2368, FP4, ROWS(16, 4, 0, 4, 2), 0),
    (2, 100, 9000, FP8, ROWS(16, 4, 1, 4, 2), 0), (14, 33, 96, FP4, ROWS(16, 4, 0, 2, 1), 0), (13, 17, 90, FP8, ROWS(16, 4, 1, 2, 1), 0),
    (17, 16, 32, FP4, ROWS(16, 16, 0, 4, 1), 0), (50, 30, 70, FP8, ROWS(16, 16, 1, 4, 1), 0), (40, 100, 5000, FP4, ROWS(16, 16, 0, 4, 2), 0),
    (40, 17, 2208, FP8, ROWS(16, 16, 1, 8, 1), 0), (260, 17, 32, FP4, ROWS(32, 32, 0, 4, 1), 0), (260, 17, 32, FP8, ROWS(32, 32, 1, 4, 1), 0),
    (1030, 18, 32, FP4, TILE(1, 2, 2, 2, 1, 0), 0), (1030, 90, 70, FP8, TILE(1, 2, 2, 2, 1, 1), 0), (1030, 19, 4928, FP4, TILE(1, 2, 2, 2, 1, 0), 2),
    (1030, 19, 5200, FP8, TILE(1, 2, 2, 2, 1, 1), 2), (4100, 453, 32, FP4, TILE(2, 2, 1, 2, 2, 0), 0), (4100, 248, 2400, FP4, TILE(2, 1, 2, 2, 2, 0), 0), (4100, 207, 1536, FP8, TILE(2, 1, 2, 2, 2, 1), 0),
    (4100, 113, 14560, FP8, TILE(2, 1, 2, 2, 2, 1), 2),
    (4100, 550, 3488, FP4, TILE(2, 2, 2, 2, 2, 0), 0), (4100, 210, 10176, FP4, TILE(2, 2, 2, 2, 2, 0), 2), (4100, 453, 32, FP8, TILE(2, 2, 2, 2, 2, 1), 0),
    (4100, 210, 10176, FP8, TILE(2, 2, 2, 2, 2, 1), 2), (4100, 3257, 1312, FP4, TILE(2, 2, 1, 4, 4, 0), 0), (2050, 2041, 12288, FP4, TILE(2, 2, 1, 4, 4, 0), 2),
    (2050, 4100, 224, FP8, TILE(2, 2, 1, 4, 2, 1), 0), (2050, 1083, 15712, FP8, TILE(2, 2, 1, 4, 2, 1), 2)])
def test_every_kernel_of_the_product(device, m, n, k, form, kernel, shares):
    """Each variant that sizes choose, with shares of k and without, up to odd ends of every extent."""
    a, sa = operands(m, k, form, seed=11)
    b, sb = operands(n, k, FP4, seed=12)
    there = [t.to(device) for t in (a, sa, b, sb)]
    rows = torch.arange(m) if m <= 300 else torch.cat([torch.arange(70), torch.arange(m - 70, m), torch.randint(0, m, (60,), generator=torch.Generator().manual_seed(m))])
    for dtype in REAL:
        c = torch.full((m, n), 7.0, dtype=dtype, device=device)
        names = launched_kernels(lambda c=c: capi.matmul_mx(*there, c))
        assert any(name.startswith(kernel) for name in names), names
        assert ("join_shares_kernel" in "".join(names)) == (shares > 0), names
        check(c[rows.to(device)], only(a, rows), only(sa, rows), b, sb)


@pytest.mark.parametrize("form", [FP4, FP8])
@pytest.mark.parametrize("m", [5, 40, 300])
def test_matmul_strides_and_batches(device, m, form):
    """Padded and transposed operands, scales and results, an operand that every batch shares, rows at odd addresses."""
    n, k, batch = 70, 352, 3
    a, sa = operands(m, k, form, (batch,))
    b, sb = operands(n, k, FP4, (1,), seed=5)
    wa, wb, g = width(form, k), k // 2, blocks(k)
    pad_a = torch.full((batch, m, wa + 13), 0xFF, dtype=torch.uint8, device=device)
    pad_a[..., 5:5 + wa] = a.view(torch.uint8).to(device)
    pad_sa = torch.full((batch, m, g + 3), 0xFF, dtype=torch.uint8, device=device)
    pad_sa[..., 2:2 + g] = sa.view(torch.uint8).to(device)
    turned = lambda t: t.view(torch.uint8).to(device).transpose(-1, -2).contiguous().transpose(-1, -2)  # noqa: E731
    b_all, sb_all = b.expand(batch, -1, -1), sb.expand(batch, -1, -1)
    share = lambda t, of: t.as_strided((batch, *t.shape[1:]), (0, *t.stride()[1:])).view(of)  # noqa: E731
    for at, (xa, xsa, xb, xsb) in enumerate([
            (pad_a[..., 5:5 + wa].view(form), pad_sa[..., 2:2 + g].view(E8M0), share(b.view(torch.uint8).to(device), FP4), share(sb.view(torch.uint8).to(device), E8M0)),
            (turned(a).view(form), turned(sa).view(E8M0), share(turned(b), FP4), share(turned(sb), E8M0))]):
        store = torch.full((batch, n, m + 2), 3.0, device=device)
        c = store[..., 1:-1].transpose(1, 2)
        capi.matmul_mx(xa, xsa, xb, xsb, c)
        check(c, a, sa, b_all, sb_all)
        c.fill_(3.0)
        assert bool((store == 3.0).all()), at


@pytest.mark.parametrize("m", [1, 3, 40, 300])
def test_matmul_rows_that_overlap(device, m):
    """Rows that lie in one another, that are all the same one, and a single row with a stride that says nothing."""
    n, k = 90, 640
    a, sa = operands(m, k, FP8)
    line, scales = operands(1, 8 * k, FP4, seed=9)
    line, scales = line.view(torch.uint8).flatten(), scales.view(torch.uint8).flatten()
    for apart, scales_apart in ((16, 1), (0, 0)):
        b = line.to(device).as_strided((n, k // 2), (apart, 1)).view(FP4)
        sb = scales.to(device).as_strided((n, k // 32), (scales_apart, 1)).view(E8M0)
        there_a, there_sa = a.to(device), sa.to(device)
        if m == 1:
            there_a, there_sa = (t.view(torch.uint8).as_strided((1, t.shape[1]), (1 << 40, 1)).view(t.dtype) for t in (there_a, there_sa))
        c = torch.empty(m, n, device=device)
        capi.matmul_mx(there_a, there_sa, b, sb, c)
        check(c, a, sa, b.view(torch.uint8).cpu().contiguous().view(FP4), sb.view(torch.uint8).cpu().contiguous().view(E8M0))


def test_matmul_in_a_workspace_of_its_caller(device):
    """Copies and shares of k in memory that held other things; one that is too small is left alone."""
    for m, n, k in ((7, 33, 300), (1030, 19, 4928), (65, 40, 90)):
        a, sa = operands(m, k, FP4)
        b, sb = operands(n, k, FP4, seed=4)
        c = torch.empty(m, n, device=device)
        there = [t.to(device) for t in (a, sa, b, sb)]
        room_for_it = torch.full((1 << 21,), 0xFF, dtype=torch.uint8, device=device)
        capi.matmul_mx(*there, c, workspace=room_for_it)
        check(c, a, sa, b, sb)
        room_for_it.fill_(0xFF)
        capi.matmul_mx(*there, c.fill_(7.0), workspace=room_for_it[:256])
        check(c, a, sa, b, sb)
        assert bool((room_for_it == 0xFF).all())


@pytest.mark.parametrize("form", [FP4, FP8])
@pytest.mark.parametrize("m", [3, 50, 200, 1000])
def test_matmul_scales_that_are_not_numbers(device, m, form):
    """A NaN scale makes its row or column NaN, and nothing else: neither the rows beside it nor blocks past a row's end."""
    n, k = 300, 32 * 13   # (rows of thirteen scales: a load of four bytes would pass the end)
    a, sa = operands(m, k, form)
    b, sb = operands(n, k, FP4, seed=2)
    sa.view(torch.uint8)[1, 0] = 255
    sb.view(torch.uint8)[7, 12] = 255
    sb.view(torch.uint8)[250, 3] = 255
    c = torch.empty(m, n, device=device)
    capi.matmul_mx(a.to(device), sa.to(device), b.to(device), sb.to(device), c)
    rows, columns = torch.arange(m) != 1, torch.ones(n, dtype=torch.bool)
    columns[[7, 250]] = False
    assert bool(torch.isnan(c[1]).all()) and bool(torch.isnan(c[:, ~columns.to(device)]).all())
    check(c[rows.to(device)][:, columns.to(device)], only(a, rows), only(sa, rows), only(b, columns), only(sb, columns))


def test_matmul_elements_that_are_not_numbers(device):
    """e4m3 has a NaN: it makes its row NaN, and no other row's partial block."""
    for m, k in ((4, 96), (40, 96), (40, 70)):
        a, sa = operands(m, k, FP8)
        b, sb = operands(200, k, FP4, seed=2)
        a.view(torch.uint8)[2, 0] = 0x7f
        c = torch.empty(m, 200, device=device)
        capi.matmul_mx(a.to(device), sa.to(device), b.to(device), sb.to(device), c)
        assert bool(torch.isnan(c[2]).all())
        keep = torch.arange(m) != 2
        check(c[keep.to(device)], only(a, keep), only(sa, keep), b, sb)


@pytest.mark.parametrize("form", [FP4, FP8])
def test_matmul_extreme_scales(device, form):
    """The smallest and the largest powers of two: results that only both together bring into range, and infinities."""
    m, n, k = 20, 40, 64
    a, sa = operands(m, k, form, low=0, high=4)
    b, sb = operands(n, k, FP4, seed=3, low=245, high=254)
    c = torch.empty(m, n, device=device)
    capi.matmul_mx(a.to(device), sa.to(device), b.to(device), sb.to(device), c)
    check(c, a, sa, b, sb)
    high = torch.full_like(sa.view(torch.uint8), 254).view(E8M0)
    capi.matmul_mx(a.to(device), high.to(device), b.to(device), sb.to(device), c)
    assert bool(torch.isinf(c).any()) and not bool(((c.abs() < 1e30) & (c != 0)).any())


def test_matmul_nothing_to_sum(device):
    empty = torch.empty((5, 0), dtype=torch.uint8, device=device)
    wide = torch.empty((9, 0), dtype=torch.uint8, device=device)
    c = torch.full((5, 9), 4.0, device=device)
    capi.matmul_mx(empty.view(FP4), empty.view(E8M0), wide.view(FP4), wide.view(E8M0), c)
    assert bool((c == 0).all())
    a, sa = room((0,), 64, FP4)
    b, sb = room((9,), 64, FP4)
    capi.matmul_mx(a, sa, b, sb, torch.empty((0, 9), device=device))
    capi.quantize_mx(torch.empty((0, 64), device=device), a, sa)


@pytest.mark.parametrize("m,n,k", [(64, 512, 8000), (1030, 19, 4928), (100, 64, 300)])
def test_matmul_replayed_in_a_graph(device, m, n, k):
    """Captured, also with a workspace for shares of k or for copies; replayed among eager work, on new operands."""
    g = torch.Generator(device=device).manual_seed(1)
    x = torch.randn((m, k), generator=g, device=device)
    w = torch.randn((n, k), generator=g, device=device)
    qa, sa = room((m,), k, FP4)
    qb, sb = room((n,), k, FP4)
    capi.quantize_mx(w, qb, sb)
    c, eager = torch.empty((m, n), device=device), torch.empty((m, n), device=device)

    def step(to):
        capi.quantize_mx(x, qa, sa)
        capi.matmul_mx(qa, sa, qb, sb, to)

    step(c)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(c)
    for _ in range(4):
        x.copy_(torch.randn((m, k), generator=g, device=device))
        graph.replay()
        step(eager)
        torch.cuda.synchronize()
        assert torch.equal(c, eager)
        check(c, qa, sa, qb, sb)


def test_python_and_native_calls_agree(device, monkeypatch):
    """The entry points' two ways in, with tensors that the one leaves to the other."""
    x = torch.randn(40, 320, device=device).bfloat16()
    w, sw = operands(96, 320, FP4)
    w, sw = w.to(device), sw.to(device)
    results = []
    for native in (True, False):
        if not native:
            monkeypatch.setattr(capi, "_calls", capi._NoNativeCalls())
        q, s = room((40,), 320, FP4)
        c, out = torch.empty(40, 96, device=device), torch.empty(40, 320, device=device)
        capi.quantize_mx(x, q, s)
        capi.matmul_mx(q, s, w, sw, c)
        capi.dequantize_mx(q, s, out)
        results.append((q.view(torch.uint8), s.view(torch.uint8), c, out))
    for one, other in zip(*results):
        assert torch.equal(one, other)


def test_two_streams_and_two_graphs(device):
    """Calls with copies and shares of k at once on two streams, named and current ones, and two graphs replayed in turn: none has another's scratch."""
    cases = []
    for m, n, k in ((1030, 19, 4928), (300, 200, 300)):
        a, sa = operands(m, k, FP4)
        b, sb = operands(n, k, FP4, seed=6)
        there = [t.to(device) for t in (a, sa, b, sb)]
        cases.append((there, capi.matmul_mx(*there, torch.empty(m, n, device=device)), torch.zeros(m, n, device=device)))
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for turn in range(20):
        for stream, (there, _, c) in zip(streams, cases):
            if turn % 2:
                capi.matmul_mx(*there, c, stream=stream)
            else:
                with torch.cuda.stream(stream):
                    capi.matmul_mx(*there, c)
    torch.cuda.synchronize()
    graphs = []
    for there, want, c in cases:
        assert torch.equal(c, want)
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            capi.matmul_mx(*there, c)
    for _ in range(3):
        for (_, _, c), stream in zip(cases, streams):
            c.zero_()
            stream.wait_stream(torch.cuda.current_stream())
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, want, c in cases:
            assert torch.equal(c, want)
