"""Mixture-of-experts layers for a few tokens against the definition in 64 bits."""
import pytest
import torch

from vecops_amd import capi

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


def blocks(extent):
    return -(-extent // 128)


def case(t, e, top, h, i, weights, seed=0, sigma=1.0):
    """Operands on the CPU: (x, gate_up, its scales, down, its scales)."""
    g = torch.Generator().manual_seed(seed + 1000 * t + 100 * e + 10 * top + h + i)
    n = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    dtype = torch.float16 if "f16" in weights.split("_") else torch.bfloat16
    x = (n(t, h) * sigma).to(dtype)
    if weights.startswith("fp8"):
        def quantized(*shape):
            v = torch.randint(0, 256, shape, generator=g).to(torch.uint8)
            v[(v & 0x7f) >= 0x70] = 0x30
            s = torch.rand((shape[0], blocks(shape[1]), blocks(shape[2])), generator=g) + 0.5
            return v.view(FP8), s * 0.05 * shape[2] ** -0.5
        return x, *quantized(e, 2 * i, h), *quantized(e, h, i)
    return x, (n(e, 2 * i, h) * h ** -0.5).to(dtype), None, (n(e, h, i) * i ** -0.5).to(dtype), None


def wide(w, scales):
    w = w.double()
    if scales is None:
        return w
    s = scales.double().repeat_interleave(128, dim=1)[:, :w.shape[1]].repeat_interleave(128, dim=2)[:, :, :w.shape[2]]
    return w * s


def experts64(x, ids, weights, gate_up, gs, down, ds):
    """(out, a bound of the fp32 work's error): sums of n terms are off by at most (n + a few) 2^-24 of the terms' sizes, the inner
    values, a pair of bf16 each, by 2^-16 of theirs besides; the exponential and the quotient by 8 units of 2^-24 (the
    activation's slope is at most 1.1, and 1.1 (|g| + 1) bounds it)."""
    t, h = x.shape
    e, i = gate_up.shape[0], down.shape[2]
    out, bound = torch.zeros(t, h, dtype=torch.float64), torch.zeros(t, h, dtype=torch.float64)
    u = 2.0 ** -24
    for token in range(t):
        terms = 0
        size = torch.zeros(h, dtype=torch.float64)
        for r in range(ids.shape[1]):
            expert = int(ids[token, r])
            if not 0 <= expert < e:
                continue
            w13, w2 = wide(gate_up[expert:expert + 1], None if gs is None else gs[expert:expert + 1])[0], \
                wide(down[expert:expert + 1], None if ds is None else ds[expert:expert + 1])[0]
            row, weight = x[token].double(), float(weights[token, r])
            both, sizes = w13 @ row, w13.abs() @ row.abs()
            off = (h + 8) * u * sizes
            gate, up = both[:i], both[i:]
            act = gate * torch.sigmoid(gate)
            act_off = 1.1 * off[:i] + 8 * u * (act.abs() + gate.abs())
            inner = act * up * weight
            inner_off = abs(weight) * (act_off * (up.abs() + off[i:]) + act.abs() * off[i:]) + (4 * u + 2.0 ** -16) * inner.abs()
            out[token] += w2 @ inner
            size += w2.abs() @ (inner.abs() + inner_off)
            bound[token] += w2.abs() @ inner_off
            terms += i
        bound[token] += (terms + 8 * 3 + 8) * u * size + 2.0 ** -16 * size * (gate_up.dtype == torch.float16)
    return out, bound


def check(out, want, bound):
    unit = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[out.dtype]
    bound = bound + unit * (want.abs() + bound) + (2.0 ** -25 if out.dtype == torch.float16 else 1e-37)
    off = (out.double().cpu() - want).abs()
    assert bool((off <= bound).all()), f"{float((off / bound).max())} times the bound"


def choices(t, e, top, seed=1):
    g = torch.Generator().manual_seed(seed)
    ids = torch.rand((t, e), generator=g).argsort(dim=1)[:, :top].to(torch.int32).contiguous()
    return ids, torch.rand((t, top), generator=g) + 0.1


def to(device, *tensors):
    return [None if v is None else v.to(device) for v in tensors]


SIZES = [(1, 8, 2, 256, 128), (1, 64, 6, 512, 352), (2, 3, 3, 64, 16), (5, 60, 4, 333, 141), (16, 8, 2, 384, 256), (17, 4, 1, 130, 40),
         (33, 16, 3, 256, 272), (64, 40, 8, 128, 96), (70, 2, 1, 200, 64), (128, 3, 2, 144, 130), (128, 256, 8, 64, 32), (1, 1, 1, 1, 1),
         (3, 512, 16, 32, 16), (128, 20, 16, 32, 24)]


@pytest.mark.parametrize("weights", ["bf16", "f16", "fp8_bf16", "fp8_f16"])
@pytest.mark.parametrize("t,e,top,h,i", SIZES)
def test_experts(device, t, e, top, h, i, weights):
    x, gate_up, gs, down, ds = case(t, e, top, h, i, weights)
    ids, w = choices(t, e, top)
    want, bound = experts64(x, ids, w, gate_up, gs, down, ds)
    dx, dids, dw, dg, dgs, dd, dds = to(device, x, ids, w, gate_up, gs, down, ds)
    for dtype in (x.dtype, torch.float32):
        out = torch.full((t, h), float("nan"), dtype=dtype, device=device)
        capi.moe_experts(dx, dids, dw, dg, dd, out, gate_up_scales=dgs, down_scales=dds)
        check(out, want, bound)


@pytest.mark.parametrize("weights", ["bf16", "fp8_bf16"])
def test_experts_elsewhere_twice_and_none(device, weights):
    """Ids that name no expert here, an expert named twice by a token, tokens that name none, all of them; all on one expert."""
    t, e, top, h, i = 20, 6, 4, 160, 96
    x, gate_up, gs, down, ds = case(t, e, top, h, i, weights)
    ids, w = choices(t, e, top)
    ids[0] = torch.tensor([-1, 6, 2 ** 31 - 1, -2 ** 31])
    ids[1] = torch.tensor([3, 3, 3, 3])
    ids[2] = torch.tensor([5, -1, 5, 2])
    ids[3] = -1
    dev = to(device, x, gate_up, gs, down, ds, w)
    for chosen in (ids, torch.full_like(ids, -7), torch.full_like(ids, 2)):
        want, bound = experts64(x, chosen, w, gate_up, gs, down, ds)
        out = torch.full((t, h), float("nan"), device=device)
        capi.moe_experts(dev[0], chosen.to(device), dev[5], dev[1], dev[3], out, gate_up_scales=dev[2], down_scales=dev[4])
        check(out, want, bound)
        assert bool((out[3] == 0).all()) or int(chosen[3, 0]) == 2


@pytest.mark.parametrize("weights", ["bf16", "f16", "fp8_bf16"])
@pytest.mark.parametrize("t", [3, 40])
def test_experts_strides(device, t, weights):
    """Everything inside larger tensors whose other numbers are NaN, at odd places; a transposed result, ids and weights."""
    e, top, h, i = 5, 2, 203, 75
    x, gate_up, gs, down, ds = case(t, e, top, h, i, weights)
    ids, w = choices(t, e, top)
    want, bound = experts64(x, ids, w, gate_up, gs, down, ds)

    def inside(v):
        if v is None:
            return None
        store = torch.full([n + 3 for n in v.shape], 0x7f, dtype=torch.uint8, device=device).view(FP8) if v.dtype == FP8 else \
            torch.full([n + 3 for n in v.shape], float("nan"), dtype=v.dtype, device=device)
        view = store[tuple(slice(1, 1 + n) for n in v.shape)]
        view.view(torch.uint8).copy_(v.view(torch.uint8)) if v.dtype == FP8 else view.copy_(v)
        return view

    store = torch.full((h + 1, t + 2), -3.0, device=device)
    out = store[:-1, 1:-1].t()
    capi.moe_experts(inside(x), ids.t().contiguous().to(device).t(), w.t().contiguous().to(device).t(), inside(gate_up), inside(down), out,
                     gate_up_scales=inside(gs), down_scales=inside(ds))
    check(out, want, bound)
    store[:-1, 1:-1] = -3.0
    assert bool((store == -3.0).all())


def test_experts_not_finite(device):
    """A NaN in a token's row, or in weights of an expert that it names, reaches that token alone."""
    t, e, top, h, i = 6, 4, 1, 96, 64
    x, gate_up, _, down, _ = case(t, e, top, h, i, "bf16")
    ids = torch.tensor([[0], [1], [2], [3], [2], [-1]], dtype=torch.int32)
    x[0, 5], gate_up[1, 3, 7], down[3, 8, 60], x[5, 0] = float("nan"), float("nan"), float("inf"), float("nan")
    out = torch.zeros((t, h), device=device)
    capi.moe_experts(*to(device, x, ids, torch.ones(t, 1), gate_up, down), out)
    ok = torch.isfinite(out.cpu())
    assert not bool(ok[0].any()) and not bool(ok[1].any()) and bool(ok[2].all()) and bool(ok[4].all()) and bool(ok[5].all())
    assert not bool(ok[3, 8]) and int((~ok[3]).sum()) == 1


@pytest.mark.parametrize("weights", ["bf16", "f16"])
@pytest.mark.parametrize("at", [1, 2, 9, 30])
def test_experts_infinite_weights(device, weights, at):
    """An infinite weight gives the infinity that the formula gives, and touches nothing else; rows end inside a load."""
    t, e, top, h, i = 3, 3, 1, 99, 43
    x, gate_up, _, down, _ = case(t, e, top, h, i, weights)
    ids, w = torch.tensor([[0], [1], [2]], dtype=torch.int32), torch.ones(t, 1)
    plain, bound = experts64(x, ids, w, gate_up, None, down, None)
    gate_up[0, i + 5, h - at], down[1, 8, i - at] = float("inf"), float("inf")
    want, _ = experts64(x, ids, w, gate_up, None, down, None)
    assert bool(torch.isinf(want[0]).all()) and bool(torch.isinf(want[1, 8]))
    out = torch.zeros((t, h), device=device)
    capi.moe_experts(*to(device, x, ids, w, gate_up, down), out)
    got = out.cpu().double()
    assert torch.equal(got[0], want[0]) and got[1, 8] == want[1, 8]
    got[0], got[1, 8] = plain[0], plain[1, 8]
    assert bool(((got - plain).abs() <= bound).all())


def test_experts_large_values_of_half_precision(device):
    """Inner values past the largest f16 number (they are held in bf16 pairs)."""
    t, e, top, h, i = 2, 2, 1, 64, 32
    x, gate_up, _, down, _ = case(t, e, top, h, i, "f16", sigma=400.0)
    down = (down.float() * 1e-3).half()
    ids, w = choices(t, e, top)
    want, bound = experts64(x, ids, w, gate_up, None, down, None)
    both = (gate_up.double()[ids[0, 0]] @ x[0].double())
    assert float((both[:i] * both[i:]).abs().max()) > 65504
    out = torch.empty((t, h), dtype=torch.float16, device=device)
    capi.moe_experts(*to(device, x, ids, w, gate_up, down), out)
    check(out, want, bound)


def test_experts_without_work(device):
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(s, dtype=dtype, device=device)  # noqa: E731
    i32 = torch.int32
    for t, e, top, h, i in ((0, 4, 2, 64, 32), (3, 4, 0, 64, 32), (3, 0, 2, 64, 32), (3, 4, 2, 64, 0), (3, 4, 2, 0, 32)):
        out = torch.full((t, h), 7.0, dtype=torch.bfloat16, device=device)
        capi.moe_experts(z(t, h), z(t, top, dtype=i32), z(t, top, dtype=torch.float32), z(e, 2 * i, h), z(e, h, i), out)
        assert bool((out == 0).all())


def route64(x, router, top, scoring, renormalize, scale, bias):
    logits = x.double() @ router.double().t()
    score = torch.softmax(logits, dim=1) if scoring == "softmax" else torch.sigmoid(logits)
    key = logits if bias is None else score + bias.double()
    order = key.sort(dim=1, descending=True, stable=True)
    weights = score.gather(1, order.indices[:, :top])
    if renormalize:
        weights = weights / weights.sum(dim=1, keepdim=True)
    gaps = (order.values[:, :-1] - order.values[:, 1:])[:, :top]
    return order.indices[:, :top].to(torch.int32), weights * scale, float(gaps.min()) if gaps.numel() else 1.0


@pytest.mark.parametrize("t,e,top,h", [(1, 8, 2, 256), (1, 64, 6, 2048), (1, 1, 1, 33), (5, 60, 4, 1001), (16, 128, 8, 512), (33, 256, 8, 700),
                                       (128, 512, 16, 64), (64, 100, 16, 130)])
@pytest.mark.parametrize("scoring,renormalize,biased,router_dtype", [("softmax", True, False, None), ("softmax", False, False, torch.float32),
                                                                     ("sigmoid", True, True, None), ("sigmoid", False, True, torch.float32),
                                                                     ("softmax", True, True, None), ("sigmoid", True, False, torch.float32)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_layer(device, t, e, top, h, scoring, renormalize, biased, router_dtype, dtype):
    """The choice and its weights, and the experts on them.  The inputs are such that neighbouring keys lie further apart than
    fp32 sums err: otherwise the choice would not be one."""
    i = 16
    x, gate_up, _, down, _ = case(t, e, top, h, i, "f16" if dtype == torch.float16 else "bf16")
    for seed in range(200):
        g = torch.Generator().manual_seed(seed)
        router = (torch.randn((e, h), generator=g) * 2 * h ** -0.5).to(router_dtype or dtype)
        bias = torch.randn((e,), generator=g) * 0.1 if biased else None
        ids, weights, gap = route64(x, router, top, scoring, renormalize, 1.5, bias)
        if gap > (1e-7 if scoring == "softmax" and biased else 2e-7) * 4:
            break
    dx, dr, dg, dd, db = to(device, x, router, gate_up, down, bias)
    got_ids = torch.full((t, top), -9, dtype=torch.int32, device=device)
    got_w = torch.full((t, top), float("nan"), device=device)
    out = torch.full((t, h), float("nan"), device=device)
    capi.moe_layer(dx, dr, dg, dd, got_ids, got_w, out, scoring=scoring, renormalize=renormalize, scale=1.5, bias=db)
    same = got_ids.cpu() == ids
    assert bool(same.all()), f"{int((~same).sum())} of {same.numel()} ids differ (gap {gap})"
    # a logit is off by (h + 8) 2^-24 of its terms' sizes, a score by that much of itself
    sizes = float((x.double().abs() @ router.double().abs().t()).max())
    assert float(((got_w.double().cpu() - weights) / weights).abs().max()) < 2 * (h + 8) * 2.0 ** -24 * sizes + (e + 16) * 2.0 ** -24
    want, bound = experts64(x, ids, got_w.cpu(), gate_up, None, down, None)
    check(out, want, bound)


def test_layer_ties_and_infinities(device):
    """Equal scores go to the lower index; an expert with a bias of -infinity comes last, one with NaN first."""
    t, e, top, h, i = 3, 70, 5, 64, 16
    x, gate_up, _, down, _ = case(t, e, top, h, i, "bf16")
    dx, dg, dd = to(device, x, gate_up, down)
    router = torch.zeros((e, h), dtype=torch.bfloat16, device=device)
    ids, w, out = torch.empty((t, top), dtype=torch.int32, device=device), torch.empty((t, top), device=device), torch.empty((t, h), device=device)
    capi.moe_layer(dx, router, dg, dd, ids, w, out)
    assert ids.tolist() == [[0, 1, 2, 3, 4]] * t and bool(((w - 0.2).abs() < 1e-6).all())
    bias = torch.full((e,), float("-inf"), device=device)
    bias[[3, 66]] = torch.tensor([-2.0, 1.0], device=device)
    capi.moe_layer(dx, router, dg, dd, ids, w, out, scoring="sigmoid", bias=bias)
    assert ids.tolist() == [[66, 3, 0, 1, 2]] * t
    bias[69] = float("nan")
    capi.moe_layer(dx, router, dg, dd, ids, w, out, scoring="sigmoid", bias=bias)
    assert ids.tolist() == [[69, 66, 3, 0, 1]] * t


def test_layer_the_same_every_time_and_on_another_stream(device):
    for t, weights in ((1, "bf16"), (24, "fp8_bf16"), (100, "f16")):
        x, gate_up, gs, down, ds = to(device, *case(t, 32, 4, 512, 272, weights))
        router = torch.randn((32, 512), device=device).to(x.dtype)
        ids, w, out = torch.empty((t, 4), dtype=torch.int32, device=device), torch.empty((t, 4), device=device), torch.empty((t, 512), device=device)
        capi.moe_layer(x, router, gate_up, down, ids, w, out, gate_up_scales=gs, down_scales=ds)
        torch.cuda.synchronize()
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(4):
                again = [torch.empty_like(v) for v in (ids, w, out)]
                capi.moe_layer(x, router, gate_up, down, *again, gate_up_scales=gs, down_scales=ds)
                stream.synchronize()
                assert all(torch.equal(a, b) for a, b in zip(again, (ids, w, out)))


def test_layer_in_a_graph(device):
    """Captured once, replayed on other inputs in the same places."""
    t, e, top, h, i = 4, 16, 2, 256, 128
    x, gate_up, _, down, _ = to(device, *case(t, e, top, h, i, "bf16"))
    router = torch.randn((e, h), device=device).bfloat16()
    results = [torch.empty((t, top), dtype=torch.int32, device=device), torch.empty((t, top), device=device), torch.empty((t, h), device=device)]
    capi.moe_layer(x, router, gate_up, down, *results)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        capi.moe_layer(x, router, gate_up, down, *results)
    for _ in range(3):
        x.copy_(torch.randn((t, h), device=device))
        graph.replay()
        torch.cuda.synchronize()
        eager = [torch.empty_like(v) for v in results]
        capi.moe_layer(x, router, gate_up, down, *eager)
        assert all(torch.equal(a, b) for a, b in zip(eager, results))
