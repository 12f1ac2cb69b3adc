"""The norm with the residual's addition and the gated activation, results quantised in each format, against 64 bits."""
import pytest
import torch

from mx_reference import E8M0, FP4, FP8, block_most, blocks, elements, nearest, room, scale_bytes, spread, width
from vecops_amd import capi

pytestmark = pytest.mark.gpu
REAL = [torch.bfloat16, torch.float16, torch.float32]
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
FORMATS = {"int8": (torch.int8, torch.float32, None), "fp8_128": (FP8, torch.float32, 128), "fp8": (FP8, E8M0, 32), "fp4": (FP4, E8M0, 32)}


def results(lead, k, form):
    dtype, scale, block = FORMATS[form]
    return room(lead, k, dtype, scale, block or k)


def check(q, scales, y, form, slack):
    """q and scales hold y (64 bits): a scale is off by no more than `slack` of it, an element is as near to y / scale as the nearest
    number of its type, but for what `slack` of y allows (in fp32, whose results y is the 64-bit value of)."""
    dtype, _, block = FORMATS[form]
    k = y.shape[-1]
    most = block_most(y, block or k)
    if dtype == torch.int8 or block == 128:
        want = (most / (127 if dtype == torch.int8 else 448)).clamp(min=2.0 ** -126)
        assert bool(((scales.cpu().double() - want).abs() <= (slack + 2.0 ** -23) * want).all())
    else:
        got = scales.cpu().view(torch.uint8)
        low, high = (scale_bytes(most * (1 + by), dtype) for by in (-slack, slack))
        assert bool(((got >= low) & (got <= high)).all())
    wide = spread(scales, k, block or k)
    v = y / wide
    if dtype == torch.int8:
        ideal, top = torch.round(v).clamp(-127, 127), 127
    else:
        ideal, top = nearest(v, dtype), {FP4: 6.0, FP8: 448.0}[dtype]
    off = (elements(q) - v).abs()
    assert bool((off <= (ideal - v).abs() + 2 * (slack + 2.0 ** -23) * v.abs().clamp(max=2 * top)).all()), float((off - (ideal - v).abs()).max())


def norm64(x, residual, weight, eps):
    h = x.double().cpu()
    if residual is not None:
        h = (x.float().cpu() + residual.float().cpu()).to(x.dtype).double()
    return h, h / torch.sqrt((h * h).mean(dim=-1, keepdim=True) + eps) * weight.double().cpu()


def norm_slack(k):
    """Roundings between the sum of squares and the result, in units of 2^-24: a thread adds up to 32 squares a span (of at least 2048
    elements), lanes six times, wavefronts sixteen; the sum's error counts half (the root); a dozen other operations."""
    return (16 * blocks(k, 2048) + 11 + 12) * 2.0 ** -24


SHAPES = [(1, 1), (1, 2), (5, 8), (3, 62), (7, 128), (64, 130), (33, 512), (4, 1000), (2, 3, 2048), (300, 4096), (1, 4096), (9, 5002), (2, 8192), (1, 16384),
          (3, 33000), (1, 70002), (2000, 64)]


@pytest.mark.parametrize("dtype", REAL)
@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("shape", SHAPES)
def test_norm(device, dtype, form, shape):
    k = shape[-1]
    if form == "fp4" and k % 2:
        pytest.skip("an odd row has no e2m1 form (refused)")
    torch.manual_seed(k)
    x, r = torch.randn(shape).mul_(3).to(dtype), torch.randn(shape).to(dtype)
    weight = torch.randn(k)
    for residual, w in ((None, weight), (r, weight.to(dtype))):
        q, scales = results(shape[:-1], k, form)
        out, summed = (torch.full(shape, 9.0, dtype=dtype, device=device) for _ in range(2))
        held = None if residual is None else residual.to(device)
        got = capi.rms_norm(x.to(device), w.to(device), q=q, scales=scales, out=out, residual=held, summed=None if held is None else summed, eps=1e-5)
        assert got == (q, scales, out)
        h, y = norm64(x, residual, w, 1e-5)
        if residual is not None:
            assert torch.equal(summed.cpu().double(), h) and torch.equal(held.cpu(), residual)
        slack = norm_slack(k)
        assert bool(((out.cpu().double() - y).abs() <= (UNIT[dtype] + slack) * y.abs() * 1.01 + 2.0 ** -24 * (dtype == torch.float16)).all())
        check(q, scales, y, form, slack)


def test_norm_alone_and_in_place(device):
    """Without a quantised result; the sum in the residual's place, the result in x's; the same bits as apart."""
    for shape in ((7, 4096), (3, 40000)):
        x, r = torch.randn(shape, device=device).bfloat16(), torch.randn(shape, device=device).bfloat16()
        w = torch.randn(shape[-1], device=device)
        out, summed = torch.empty_like(x), torch.empty_like(x)
        assert capi.rms_norm(x, w, out=out, residual=r, summed=summed) is out
        q, scales = results(shape[:-1], shape[-1], "fp8_128")
        assert capi.rms_norm(x, w, q=q, scales=scales, residual=r.clone()) == (q, scales)
        x2, r2 = x.clone(), r.clone()
        capi.rms_norm(x2, w, out=x2, residual=r2)
        assert torch.equal(x2, out) and torch.equal(r2, summed)
        x3 = x.clone()
        capi.rms_norm(x3, w, q=q, scales=scales, residual=r, summed=x3)
        assert torch.equal(x3, summed)
        q2, scales2 = results(shape[:-1], shape[-1], "fp8_128")
        capi.quantize_fp8_block((h := summed.double()).div((h * h).mean(-1, keepdim=True).add(1e-6).sqrt()).mul(w.double()).float(), q2, scales2)
        assert bool(((scales - scales2).abs() <= 2 * norm_slack(shape[-1]) * scales2).all())


@pytest.mark.parametrize("form", FORMATS)
def test_norm_of_numbers_at_the_edges(device, form):
    """Rows of zeros, with an infinity, with a NaN, of the largest numbers and the smallest; the rows beside them stay."""
    x = torch.randn(8, 512)
    x[1] = 0
    x[2, 100] = float("inf")
    x[3, 200] = float("nan")
    x[4] *= 2.0 ** -140
    x[5] *= 2.0 ** 50
    w = torch.ones(512)
    q, scales = results((8,), 512, form)
    out = torch.empty(8, 512, device=device)
    capi.rms_norm(x.to(device), w.to(device), q=q, scales=scales, out=out, eps=1e-5)
    fine = torch.tensor([0, 1, 4, 5, 6, 7])
    _, y = norm64(x[fine], None, w, 1e-5)
    take = lambda t: t.view(torch.uint8).cpu()[fine].view(t.dtype) if t.dtype != torch.float32 else t.cpu()[fine]  # noqa: E731
    check(take(q), take(scales), y, form, norm_slack(512) + 2.0 ** -20)
    assert bool((out[1] == 0).all()) and bool(torch.isnan(out[3]).all()) and bool(torch.isnan(out[2, 100]))
    s = scales.cpu().double()
    assert bool(torch.isnan(s[3]).all()) and bool(torch.isnan(s[2]).any())


@pytest.mark.parametrize("form", FORMATS)
def test_norm_strides(device, form):
    """Rows and batches apart, at odd addresses, scales the other way round; nothing else is written."""
    b, m, k = 2, 5, 200
    x, r, w = torch.randn(b, m, k).half(), torch.randn(b, m, k).half(), torch.randn(k).half()
    lay = lambda t: torch.full((m, b, k + 9), 5.0, dtype=t.dtype, device=device)  # noqa: E731
    view = lambda t: t.transpose(0, 1)[..., 3:3 + k]  # noqa: E731
    xs, rs, hs, os = (lay(x) for _ in range(4))
    view(xs).copy_(x)
    view(rs).copy_(r)
    dtype, scale_dtype, block = FORMATS[form]
    wq, g = width(dtype, k), blocks(k, block or k)
    q_store = torch.full((m, b, wq + 3), 77, dtype=torch.uint8, device=device)
    s_store = torch.full((b, g + 1, m), 1.5, device=device) if scale_dtype == torch.float32 else torch.full((b, g + 1, m), 99, dtype=torch.uint8, device=device)
    q, scales = q_store.view(dtype).transpose(0, 1)[..., 1:1 + wq], s_store.view(scale_dtype)[:, :g].transpose(1, 2)
    capi.rms_norm(view(xs), w.to(device), q=q, scales=scales, out=view(os), residual=view(rs), summed=view(hs))
    h, y = norm64(x, r, w, 1e-6)
    assert torch.equal(view(hs).cpu().double(), h) and torch.equal(view(xs).cpu(), x) and torch.equal(view(rs).cpu(), r)
    check(q.view(torch.uint8).contiguous().view(dtype), s_store[:, :g].transpose(1, 2).contiguous().view(scale_dtype), y, form, norm_slack(k))
    for store, seen in ((hs, view(hs)), (os, view(os))):
        seen.fill_(5.0)
        assert bool((store == 5.0).all())
    q_store.transpose(0, 1)[..., 1:1 + wq] = 77
    s_store[:, :g] = s_store[0, -1, 0]
    assert bool((q_store == 77).all()) and bool((s_store == s_store[0, -1, 0]).all())


def gate64(x):
    g, u = x.double().cpu().chunk(2, dim=-1)
    return g / (1 + torch.exp(-g)) * u


def gate_slack(x):
    """log2 e as an fp32 number and its product with g are off by 2^-26 and 2^-24 of |g|, and e^-g, so the result, by as much of itself;
    the exponential, the sum, its reciprocal and two products add a rounding each, the two functions' up to a unit of the last place."""
    g = x.double().cpu().chunk(2, dim=-1)[0].abs()
    return (1.25 * float(g[torch.isfinite(g)].max()) + 8) * 2.0 ** -24


@pytest.mark.parametrize("dtype", REAL)
@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("shape", SHAPES)
def test_gate(device, dtype, form, shape):
    k = shape[-1]
    if form == "fp4" and k % 2:
        pytest.skip("an odd row has no e2m1 form (refused)")
    torch.manual_seed(k + 1)
    x = torch.randn(*shape[:-1], 2 * k).mul_(4).to(dtype)
    q, scales = results(shape[:-1], k, form)
    assert capi.silu_mul_quantize(x.to(device), q, scales) == (q, scales)
    check(q, scales, gate64(x), form, gate_slack(x))


@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("shape", [(5000, 1030), (2100, 4100), (130, 70002)])
def test_many_rows(device, form, shape):
    """So many that a thread takes several pieces of a row, and rows that are read again."""
    torch.manual_seed(shape[0])
    k = shape[-1]
    x = torch.randn(shape[0], 2 * k).bfloat16()
    q, scales = results(shape[:-1], k, form)
    capi.silu_mul_quantize(x.to(device), q, scales)
    check(q, scales, gate64(x), form, gate_slack(x))
    x, weight = x[:, :k], torch.randn(k)
    capi.rms_norm(x.to(device), weight.to(device), q=q, scales=scales, eps=1e-5)
    check(q, scales, norm64(x, None, weight, 1e-5)[1], form, norm_slack(k))


@pytest.mark.parametrize("form", FORMATS)
def test_gate_of_numbers_at_the_edges(device, form):
    """Gates far from zero on both sides, infinities, NaN: what silu gives, and the rows beside."""
    x = torch.randn(6, 512)
    x[1, :256] = torch.linspace(-200, 200, 256)
    x[2, :256] = torch.linspace(-80, -60, 256)
    x[3, 3] = float("inf")
    x[4, 300] = float("nan")
    q, scales = results((6,), 256, form)
    capi.silu_mul_quantize(x.to(device), q, scales)
    fine = torch.tensor([0, 1, 2, 5])
    take = lambda t: t.view(torch.uint8).cpu()[fine].view(t.dtype) if t.dtype != torch.float32 else t.cpu()[fine]  # noqa: E731
    check(take(q), take(scales), gate64(x[fine]), form, gate_slack(x[fine]))
    s = scales.cpu().double()
    for row, at in ((3, 3), (4, 44)):
        group = at // (FORMATS[form][2] or 256)
        assert not bool(torch.isfinite(s[row, group])) and bool(torch.isfinite(s[row]).sum() == s.shape[1] - 1)


def test_feed_forward_as_a_program_runs_it(device):
    """Norm, product, gated activation, product, in 4 bits and with 8-bit activations; captured, replayed among eager work."""
    t, h, i = 24, 512, 704
    g = torch.Generator(device=device).manual_seed(0)
    n = lambda *s: torch.randn(s, generator=g, device=device)  # noqa: E731
    gate_up, gate_up_scales = capi.quantize_mx(n(2 * i, h) * h ** -0.5, *room((2 * i,), h, FP4))
    down, down_scales = capi.quantize_mx(n(h, i) * i ** -0.5, *room((h,), i, FP4))
    weight = n(h).bfloat16()
    for form in (FP4, FP8):
        x, residual = n(t, h).bfloat16(), n(t, h).bfloat16()
        both, out, summed = (torch.empty((t, w), dtype=torch.bfloat16, device=device) for w in (2 * i, h, h))
        q, s = room((t,), h, form)
        inner, inner_s = room((t,), i, form)

        def step():
            capi.rms_norm(x, weight, q=q, scales=s, residual=residual, summed=summed)
            capi.matmul_mx(q, s, gate_up, gate_up_scales, both)
            capi.silu_mul_quantize(both, inner, inner_s)
            return capi.matmul_mx(inner, inner_s, down, down_scales, out)

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        for _ in range(3):
            x.copy_(n(t, h))
            graph.replay()
            replayed = [v.view(torch.uint8).clone() for v in (out, summed, inner, inner_s)]
            torch.cuda.synchronize()
            step()
            assert all(torch.equal(a, b.view(torch.uint8)) for a, b in zip(replayed, (out, summed, inner, inner_s)))
        # each operator from what the one before has left, in 64 bits
        _, y = norm64(x, residual, weight, 1e-6)
        check(q, s, y, "fp4" if form == FP4 else "fp8", norm_slack(h))
        value = lambda e, sc: elements(e) * spread(sc, elements(e).shape[-1])  # noqa: E731
        want = value(q, s) @ value(gate_up, gate_up_scales).t()
        assert float((both.cpu().double() - want).norm() / want.norm()) < 2.0 ** -8
        check(inner, inner_s, gate64(both), "fp4" if form == FP4 else "fp8", gate_slack(both))
        want = value(inner, inner_s) @ value(down, down_scales).t()
        assert float((out.cpu().double() - want).norm() / want.norm()) < 2.0 ** -8


def test_norm_feeds_the_other_products(device):
    """int8 with row scales into the dequantising product, e4m3 with blocks of 128 into the 8-bit one."""
    m, k, n = 20, 640, 300
    x, w = torch.randn(m, k, device=device).bfloat16(), torch.randn(k, device=device)
    _, y = norm64(x, None, w, 1e-6)
    weights = torch.randn(n, k, device=device) * k ** -0.5
    q, s = results((m,), k, "int8")
    capi.rms_norm(x, w, q=q, scales=s)
    column = (weights.abs().amax(dim=1) / 127).contiguous()
    c = torch.empty(m, n, device=device)
    capi.matmul_i8_dequant(q, torch.round(weights / column[:, None]).to(torch.int8), s.view(-1), column, c)
    want = y @ weights.double().cpu().t()
    assert float((c.cpu().double() - want).norm() / want.norm()) < 0.03   # (two roundings of up to 1/254 of a row's largest number, three deviations or so)
    q, s = results((m,), k, "fp8_128")
    capi.rms_norm(x, w, q=q, scales=s)
    wq, ws = torch.empty((n, k), dtype=FP8, device=device), torch.empty((blocks(n, 128), blocks(k, 128)), device=device)
    capi.quantize_fp8_block(weights, wq, ws, block_rows=128)
    capi.matmul_fp8_block(q, s, wq, ws, c)
    assert float((c.cpu().double() - want).norm() / want.norm()) < 0.06   # (two roundings of up to 2^-4 each)
