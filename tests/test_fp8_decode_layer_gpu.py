"""The example of a decoder layer on 8-bit floats, and that both ways into an entry point are one."""
import importlib.util
import os

import pytest
import torch

from vecops_amd import capi

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


def example():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "fp8_decode_layer.py")
    spec = importlib.util.spec_from_file_location("fp8_decode_layer", at)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def wide(q, scales):
    s = scales.double().repeat_interleave(128, dim=-2)[..., :q.shape[-2], :].repeat_interleave(128, dim=-1)[..., :q.shape[-1]]
    return q.double() * s


def test_layer_step(device):
    """Against 64 bits on the operands as quantised.  The projection's bf16 result is taken from the step itself, so that what is
    compared is a sum of H products with scales (16-bit results: of eight products seven may lose 2^-13 of the largest) and its
    rounding; the layer's part by its own tests' order: inner values to 2^-16, the result's rounding 2^-8."""
    t, h, i, e, top = 5, 256, 136, 8, 2
    layer = example().Layer(t, h, i, e, top)
    attended = torch.randn((t, h), generator=torch.Generator().manual_seed(3)).bfloat16().to(device)
    out = layer.step(attended).double().cpu()
    q, x = layer.q.cpu(), layer.x.double().cpu()
    row_scales = layer.scales.double().cpu().repeat_interleave(128, dim=1)[:, :h]
    w = wide(layer.proj.cpu(), layer.proj_scales.cpu())
    dequantized = q.double() * row_scales
    want, size = dequantized @ w.T, dequantized.abs() @ w.abs().T
    bound = (7 * 2.0 ** -13 + (128 + 3 + h // 128) * 2.0 ** -24) * size
    assert bool(((x - want).abs() <= bound + 2.0 ** -8 * (want.abs() + bound)).all())
    # a block's scale is its largest number's over 448, and a quotient is off by half a unit of three bits, or of the smallest one
    amax = attended.double().cpu().abs().unflatten(1, (h // 128, 128)).amax(2).repeat_interleave(128, dim=1)
    off = (dequantized - attended.double().cpu()).abs()
    assert bool((off <= 2.0 ** -4 * attended.double().cpu().abs() * 1.001 + 2.0 ** -10 * amax / 448 * 1.001).all())
    # the experts on the step's own choice
    gate_up, down = wide(layer.gate_up.cpu(), layer.gate_up_scales.cpu()), wide(layer.down.cpu(), layer.down_scales.cpu())
    ids, weights = layer.ids.cpu(), layer.weights.double().cpu()
    scores = torch.softmax(x @ layer.router.double().cpu().T, dim=1)
    best, which = scores.topk(top, dim=1)
    assert torch.equal(ids.long(), which)
    assert torch.allclose(weights, best / best.sum(1, keepdim=True), rtol=1e-4, atol=0)
    for token in range(t):
        want, size = torch.zeros(h, dtype=torch.float64), torch.zeros(h, dtype=torch.float64)
        for r in range(top):
            n = int(ids[token, r])
            both = gate_up[n] @ x[token]
            sizes = gate_up[n].abs() @ x[token].abs()
            inner = both[:i] * torch.sigmoid(both[:i]) * both[i:] * weights[token, r]
            # (sums of h products; the activation's slope is at most 1.1, the exponential and the quotient 8 units of it)
            off = (h + 8) * 2.0 ** -24 * sizes
            inner_off = weights[token, r] * (1.1 * off[:i] * (both[i:].abs() + off[i:]) + both[:i].abs() * off[i:]) + (2.0 ** -16 + 20 * 2.0 ** -24) * (
                inner.abs() + weights[token, r] * both[:i].abs() * both[i:].abs())
            want += down[n] @ inner
            size += down[n].abs() @ (inner_off + (top * i + 32) * 2.0 ** -24 * inner.abs())
        assert bool(((out[token] - want).abs() <= size + 2.0 ** -8 * (want.abs() + size)).all())


@pytest.mark.parametrize("t", [1, 6, 40])
def test_stream_given_or_current(device, t):
    """A call on a stream of the caller's, which describes its operands in Python, and one on the current stream give the same
    bits."""
    g = torch.Generator().manual_seed(t)
    h, i, e, top = 200, 72, 6, 2
    x = torch.randn((t, h), generator=g).bfloat16().to(device)
    q, s = torch.empty((t, h), dtype=FP8, device=device), torch.empty((t, 2), device=device)
    w, ws = torch.empty((i, h), dtype=FP8, device=device), torch.empty((1, 2), device=device)
    c = torch.empty((t, i), dtype=torch.bfloat16, device=device)
    gate_up, down = (torch.randn((e, 2 * i, h), generator=g) * 0.1).bfloat16().to(device), (torch.randn((e, h, i), generator=g) * 0.1).bfloat16().to(device)
    router, ids, weights = torch.randn((e, h), generator=g).to(device), torch.empty((t, top), dtype=torch.int32, device=device), torch.empty((t, top), device=device)
    out, again = torch.empty((t, h), device=device), torch.empty((t, h), device=device)
    raw = torch.randn((i, h), generator=g).to(device)

    def everything(stream):
        for v in (q, w):
            v.view(torch.uint8).fill_(0x7f)
        for v in (s, ws, c, weights, out, again):
            v.fill_(float("nan"))
        torch.cuda.synchronize()
        capi.quantize_fp8_block(x, q, s, stream=stream)
        capi.quantize_fp8_block(raw, w, ws, 128, stream=stream)
        capi.matmul_fp8_block(q, s, w, ws, c, stream=stream)
        capi.moe_layer(x, router, gate_up, down, ids, weights, out, scoring="sigmoid", scale=2.0, stream=stream)
        capi.moe_experts(x, ids, weights, gate_up, down, again, stream=stream)
        torch.cuda.synchronize()
        return [v.view(torch.uint8).clone() for v in (q, s, w, ws, c, ids, weights, out, again)]

    current, other = everything(None), everything(torch.cuda.Stream())
    assert all(torch.equal(a, b) for a, b in zip(current, other))
    assert torch.equal(out, again) and bool(torch.isfinite(out).all())
