"""Mixture-of-experts layers where the kernels take another way: up to four tokens through a layer of 8-bit floats (the choice is
made by the kernel that uses it), and an expert that many more tokens name than the average one."""
import pytest
import torch

from vecops_amd import capi

from test_moe_few_tokens_gpu import case, check, choices, experts64, route64, to

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("e,top,h,i", [(8, 2, 256, 128), (64, 6, 512, 352), (60, 4, 333, 141), (3, 3, 130, 40), (160, 8, 1001, 75), (512, 16, 64, 24),
                                       (1, 1, 16, 16)])
@pytest.mark.parametrize("weights", ["fp8_bf16", "fp8_f16", "bf16", "f16"])
@pytest.mark.parametrize("scoring,biased,wide_router", [("softmax", False, False), ("sigmoid", True, True)])
def test_single_tokens(device, t, e, top, h, i, weights, scoring, biased, wide_router):
    """The choice as its definition makes it (keys further apart than fp32 sums err), its weights, and the experts on them."""
    x, gate_up, gs, down, ds = case(t, e, top, h, i, weights)
    for seed in range(200):
        g = torch.Generator().manual_seed(seed)
        router = (torch.randn((e, h), generator=g) * 2 * h ** -0.5).to(torch.float32 if wide_router else x.dtype)
        bias = torch.randn((e,), generator=g) * 0.1 if biased else None
        ids, w, gap = route64(x, router, top, scoring, True, 1.5, bias)
        if gap > 2e-7 * 4:
            break
    assert gap > 2e-7 * 4
    dx, dr, dg, dgs, dd, dds, db = to(device, x, router, gate_up, gs, down, ds, bias)
    for dtype in (x.dtype, torch.float32):
        got_ids = torch.full((t, top), -9, dtype=torch.int32, device=device)
        got_w, out = torch.full((t, top), float("nan"), device=device), torch.full((t, h), float("nan"), dtype=dtype, device=device)
        capi.moe_layer(dx, dr, dg, dd, got_ids, got_w, out, scoring=scoring, scale=1.5, bias=db, gate_up_scales=dgs, down_scales=dds)
        assert torch.equal(got_ids.cpu(), ids)
        # a logit is off by (h + 8) 2^-24 of its terms' sizes, a score by that much of itself
        sizes = float((x.double().abs() @ router.double().abs().t()).max())
        assert float(((got_w.double().cpu() - w) / w).abs().max()) < 2 * (h + 8) * 2.0 ** -24 * sizes + (e + 16) * 2.0 ** -24
        want, bound = experts64(x, ids, got_w.cpu(), gate_up, gs, down, ds)
        check(out, want, bound)
        again = torch.full((t, h), float("nan"), dtype=dtype, device=device)
        capi.moe_experts(dx, got_ids, got_w, dg, dd, again, gate_up_scales=dgs, down_scales=dds)
        assert torch.equal(out, again)


@pytest.mark.parametrize("weights", ["bf16", "f16", "fp8_bf16", "fp8_f16"])
@pytest.mark.parametrize("t,e,top,hot", [(64, 64, 2, 64), (40, 48, 3, 17), (128, 256, 4, 100), (128, 64, 2, 128), (33, 512, 1, 33)])
def test_an_expert_that_many_tokens_name(device, t, e, top, hot, weights):
    """On average an expert has up to eight tokens, one has `hot`: its weights serve them sixteen (in down eight) at a time."""
    h, i = 272, 136
    x, gate_up, gs, down, ds = case(t, e, top, h, i, weights)
    ids, w = choices(t, e, top)
    assert t * top // e <= 8
    ids[ids == 5] = -1
    ids[:hot, top - 1] = 5
    want, bound = experts64(x, ids, w, gate_up, gs, down, ds)
    dx, dids, dw, dg, dgs, dd, dds = to(device, x, ids, w, gate_up, gs, down, ds)
    for dtype in (x.dtype, torch.float32):
        out = torch.full((t, h), float("nan"), dtype=dtype, device=device)
        capi.moe_experts(dx, dids, dw, dg, dd, out, gate_up_scales=dgs, down_scales=dds)
        check(out, want, bound)


@pytest.mark.parametrize("weights", ["bf16", "fp8_f16"])
@pytest.mark.parametrize("t,h", [(5, 200), (37, 512), (128, 256), (128, 1040)])
def test_shares_of_a_result_are_added_whole(device, t, h, weights):
    """Where few columns leave compute units idle, workgroups share a column block and the last one adds: from a workspace that
    holds NaN before each call, so that a number that was not there yet would show."""
    e, top, i = 12, 3, 272
    x, gate_up, gs, down, ds = case(t, e, top, h, i, weights)
    ids, w = choices(t, e, top)
    want, bound = experts64(x, ids, w, gate_up, gs, down, ds)
    dx, dids, dw, dg, dgs, dd, dds = to(device, x, ids, w, gate_up, gs, down, ds)
    workspace = torch.empty(64 << 20, dtype=torch.uint8, device=device)
    first = None
    for _ in range(12):
        workspace.fill_(0xff)
        out = torch.full((t, h), float("nan"), device=device)
        capi.moe_experts(dx, dids, dw, dg, dd, out, gate_up_scales=dgs, down_scales=dds, workspace=workspace)
        if first is None:
            first = out
            check(out, want, bound)
        assert torch.equal(out, first)
