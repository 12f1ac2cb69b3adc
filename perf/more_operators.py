"""The calls that microscaled formats and the operators between a decoder layer's products are measured by: quantisation to
4-bit and 8-bit floats with a power of two for each 32 elements, the product of such operands, the root-mean-square norm with
the residual's addition and quantised results, the gated activation with quantised results, and the feed-forward half of a
layer made of them - from single tokens that are bound by launches and latency to prefill products bound by the matrix cores.

``listed()`` names twelve of them, ``draw(rng)`` gives another of the same kinds and ranges, ``prepare`` makes what a
program holds before the call, ``run`` is one call: of the framework's operators where ``own`` is true, else of their plain
form in elementary torch operations.  ``exact`` is the same in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

_TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}
_FP4, _FP8, _E8M0 = torch.float4_e2m1fn_x2, torch.float8_e4m3fn, torch.float8_e8m0fnu
# a quantised format: bytes an element, elements that share a scale, bytes of a scale
_FORMATS = {"fp4": (0.5, 32, 1), "fp8": (1, 32, 1), "fp8_128": (1, 128, 4)}
_EPS = 1e-5


def listed() -> list[dict]:
    return [
        # the activations of a few decoded tokens, to 4 bits and back (as a program looks what the format costs): latency
        {"name": "round_trip_decode", "kind": "round_trip", "m": 16, "k": 4096, "dtype": "bf16", "format": "fp4"},
        # a checkpoint's projection, to 4 bits and back
        {"name": "round_trip_weights", "kind": "round_trip", "m": 11008, "k": 4096, "dtype": "bf16", "format": "fp4"},
        # one token through a 4-bit projection: the weights' bytes once
        {"name": "product_m1", "kind": "product", "m": 1, "n": 14336, "k": 4096, "a": "fp4", "out": "bf16"},
        # sixteen sequences decoded together with 8-bit activations, long K
        {"name": "product_m16_a8", "kind": "product", "m": 16, "n": 4096, "k": 14336, "a": "fp8", "out": "bf16"},
        # a short prompt with 8-bit activations
        {"name": "product_m128_a8", "kind": "product", "m": 128, "n": 11008, "k": 4096, "a": "fp8", "out": "bf16"},
        # extents that line up with no tile, single-precision results
        {"name": "product_ragged", "kind": "product", "m": 777, "n": 1000, "k": 3008, "a": "fp4", "out": "f32"},
        # a feed-forward projection of a long prompt (the largest case)
        {"name": "product_prefill", "kind": "product", "m": 4096, "n": 11008, "k": 4096, "a": "fp4", "out": "bf16"},
        # the norm in front of a projection, a few decoded tokens: latency
        {"name": "norm_decode", "kind": "norm", "m": 4, "k": 4096, "dtype": "bf16", "format": "fp8_128", "residual": True},
        # the same of a long prompt, scales that are powers of two
        {"name": "norm_prefill", "kind": "norm", "m": 4096, "k": 8192, "dtype": "bf16", "format": "fp8", "residual": True},
        # the gated activation in front of a down projection whose width is no multiple of 128
        {"name": "gate_odd", "kind": "gate", "m": 1999, "k": 11000, "dtype": "f16", "format": "fp8_128"},
        # the feed-forward half of a layer in 4 bits, one token
        {"name": "feed_forward_t1", "kind": "feed_forward", "t": 1, "h": 4096, "i": 14336, "a": "fp4"},
        # the same with 8-bit activations, a prompt
        {"name": "feed_forward_t512_a8", "kind": "feed_forward", "t": 512, "h": 4096, "i": 11008, "a": "fp8"},
    ]


def _size(rng, low: int, high: int, steps=(1, 1, 8, 64, 128)) -> int:
    """An extent between low and high, even over the logarithm; a good part of them multiples of what kernels like."""
    value = math.exp(rng.uniform(math.log(low), math.log(high)))
    step = rng.choice(steps)
    return int(min(high, max(low, round(value / step) * step)))


def _cost(case: dict) -> float:
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def _drawn(rng) -> dict:
    kind = rng.choice(["round_trip", "product", "product", "product", "norm", "norm", "gate", "feed_forward"])
    if kind == "round_trip":
        return {"kind": kind, "m": _size(rng, 1, 16384, (1, 1, 16)), "k": _size(rng, 64, 16384, (2, 2, 32, 128)),
                "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "format": rng.choice(["fp4", "fp4", "fp8"])}
    if kind == "product":
        a = rng.choice(["fp4", "fp4", "fp8"])
        return {"kind": kind, "m": _size(rng, 1, 4096, (1, 1, 16)), "n": _size(rng, 256, 14336, (1, 16, 64, 128)),
                "k": _size(rng, 128, 14336, (2, 32, 32, 128, 256)), "a": a, "out": rng.choice(["bf16", "bf16", "f16", "f32"] if a == "fp4" else ["bf16", "f16"])}
    if kind == "feed_forward":
        return {"kind": kind, "t": _size(rng, 1, 1024, (1, 1, 16)), "h": _size(rng, 512, 5120, (32, 128)), "i": _size(rng, 512, 14336, (32, 128)),
                "a": rng.choice(["fp4", "fp8"])}
    case = {"kind": kind, "m": _size(rng, 1, 8192, (1, 1, 16)), "k": _size(rng, 64, 16384, (1, 1, 8, 32, 128)), "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]),
            "format": rng.choice(["fp8_128", "fp8"])}
    if kind == "norm":
        case["residual"] = rng.choice([True, True, False])
    return case


def draw(rng) -> dict:
    most = max(map(_cost, listed()))
    while True:
        case = _drawn(rng)
        if _cost(case) <= most:
            return case


def _blocks(extent: int, block: int = 32) -> int:
    return -(-extent // block)


def _blocked(x, block: int):
    """x [.., K] in fp32 as [.., blocks, block], zeros behind K."""
    k = x.shape[-1]
    return torch.nn.functional.pad(x.float(), (0, _blocks(k, block) * block - k)).unflatten(-1, (-1, block))


def _e2m1_codes(y):
    """The nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with y's sign, ties to the even code."""
    a = y.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    return code + 8 * torch.signbit(y).to(torch.uint8)


def _quantized(x, kind: str):
    """The plain form of the quantiser: x [.., K] -> (elements' bytes, scales).  Microscaled: the power of two that brings a
    block's largest number into the element type's highest binade; what is then past its largest number becomes that."""
    block, k = _FORMATS[kind][1], x.shape[-1]
    y = _blocked(x, block)
    most = y.abs().amax(dim=-1)
    if kind == "fp8_128":
        scales = (most / 448.0).clamp(min=2.0 ** -126)
        return (y / scales[..., None]).to(_FP8).flatten(-2)[..., :k].contiguous(), scales
    exponent = ((most.view(torch.int32) >> 23) - (2 if kind == "fp4" else 8)).clamp(min=0)
    y = y * ((254 - exponent) << 23).view(torch.float32)[..., None]
    scales = exponent.to(torch.uint8).view(_E8M0)
    if kind == "fp8":
        return y.clamp(-448.0, 448.0).to(_FP8).flatten(-2)[..., :k].contiguous(), scales
    codes = _e2m1_codes(y).flatten(-2)[..., :k]
    return (codes[..., 0::2] | codes[..., 1::2] << 4).contiguous().view(_FP4), scales


def _values(q, scales):
    """fp32 numbers that microscaled elements stand for."""
    if q.dtype == _FP4:
        table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=q.device)
        table = torch.cat([table, -table])
        pairs = q.view(torch.uint8).int()
        v = torch.stack([table[pairs & 15], table[pairs >> 4]], dim=-1).flatten(-2)
    else:
        v = q.float()
    return v * scales.float().repeat_interleave(32, dim=-1)[..., :v.shape[-1]]


class _Random:
    """Operands of one state, from its seed alone."""

    def __init__(self, seed: int):
        self.generator = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, shape, sigma=1.0, dtype=torch.float32):
        x = torch.randn(shape, generator=self.generator, device="cuda", dtype=torch.float32)
        return x.mul_(sigma).to(dtype)

    def activations(self, shape, dtype):
        """Normal values with some channels that are ten times the others, as hidden states have them."""
        channels = torch.rand(shape[-1], generator=self.generator, device="cuda") < 0.01
        return self.normal(shape).mul_(torch.where(channels, 10.0, 1.0)).to(dtype)

    def weights(self, n: int, k: int):
        """(4-bit weights, their scales), of the deviation that keeps a product's result near its input's."""
        return _quantized(self.normal((n, k), k ** -0.5), "fp4")


def _room(m: int, k: int, kind: str):
    """(elements, scales) for the results of a quantiser."""
    size, block, _ = _FORMATS[kind]
    q = torch.zeros((m, k // 2), dtype=torch.uint8, device="cuda").view(_FP4) if kind == "fp4" else torch.zeros((m, k), dtype=_FP8, device="cuda")
    return q, torch.ones((m, _blocks(k, block)), device="cuda").to(torch.float32 if kind == "fp8_128" else _E8M0)


def prepare(case: dict, seed: int) -> dict:
    """Operands, outputs and what a program keeps from call to call."""
    r, kind = _Random(seed), case["kind"]
    s = dict(case)
    if kind == "product":
        m, n, k = case["m"], case["n"], case["k"]
        s["a"], s["a_scales"] = _quantized(r.activations((m, k), torch.bfloat16), case["a"])
        s["b"], s["b_scales"] = r.weights(n, k)
        s["c"] = torch.empty((m, n), dtype=_TORCH[case["out"]], device="cuda")
        return s
    if kind == "feed_forward":
        t, h, i, a = (case[name] for name in ("t", "h", "i", "a"))
        s["x"], s["residual"] = r.normal((t, h), 0.5, torch.bfloat16), r.activations((t, h), torch.bfloat16)
        s["weight"] = (1 + r.normal((h,), 0.1)).bfloat16()
        s["gate_up"], s["gate_up_scales"] = r.weights(2 * i, h)
        s["down"], s["down_scales"] = r.weights(h, i)
        s["summed"], s["both"], s["out"] = (torch.empty((t, n), dtype=torch.bfloat16, device="cuda") for n in (h, 2 * i, h))
        s["q"], s["q_scales"] = _room(t, h, a)
        s["inner"], s["inner_scales"] = _room(t, i, a)
        return s
    m, k, dtype = case["m"], case["k"], _TORCH[case["dtype"]]
    s["q"], s["q_scales"] = _room(m, k, case["format"])
    if kind == "gate":
        s["gate_up"] = r.activations((m, 2 * k), dtype)
        return s
    s["x"] = r.activations((m, k), dtype)
    if kind == "round_trip":
        s["out"] = torch.empty_like(s["x"])
        return s
    s["weight"] = (1 + r.normal((k,), 0.1)).to(dtype)
    s["residual"] = r.normal((m, k), 2.0, dtype) if case["residual"] else None
    s["summed"] = torch.empty_like(s["x"]) if case["residual"] else None
    return s


def _plain_norm(x, residual, weight):
    """(the sum in x's type or None, its norm times the weight in fp32)."""
    summed = None if residual is None else (x.float() + residual.float()).to(x.dtype)
    h = (x if residual is None else summed).float()
    return summed, h * torch.rsqrt(h.square().mean(dim=-1, keepdim=True) + _EPS) * weight.float()


def _plain_gate(gate_up):
    gate, up = gate_up.float().chunk(2, dim=-1)
    return gate * torch.sigmoid(gate) * up


def _plain_product(a, a_scales, b, b_scales, dtype):
    return (_values(a, a_scales) @ _values(b, b_scales).t()).to(dtype)


def _own_run(s: dict):
    from vecops_amd import capi
    kind = s["kind"]
    if kind == "round_trip":
        capi.quantize_mx(s["x"], s["q"], s["q_scales"])
        return capi.dequantize_mx(s["q"], s["q_scales"], s["out"]), s["q_scales"]
    if kind == "product":
        return capi.matmul_mx(s["a"], s["a_scales"], s["b"], s["b_scales"], s["c"])
    if kind == "gate":
        return capi.silu_mul_quantize(s["gate_up"], s["q"], s["q_scales"])
    capi.rms_norm(s["x"], s["weight"], q=s["q"], scales=s["q_scales"], residual=s["residual"], summed=s["summed"], eps=_EPS)
    if kind == "norm":
        return s["q"], s["q_scales"], s["summed"]
    capi.matmul_mx(s["q"], s["q_scales"], s["gate_up"], s["gate_up_scales"], s["both"])
    capi.silu_mul_quantize(s["both"], s["inner"], s["inner_scales"])
    capi.matmul_mx(s["inner"], s["inner_scales"], s["down"], s["down_scales"], s["out"])
    return s["out"], s["summed"]


def run(s: dict):
    kind = s["kind"]
    if own:
        return _own_run(s)
    if kind == "round_trip":
        q, scales = _quantized(s["x"], s["format"])
        return _values(q, scales).to(s["x"].dtype), scales
    if kind == "product":
        return _plain_product(s["a"], s["a_scales"], s["b"], s["b_scales"], s["c"].dtype)
    if kind == "gate":
        return _quantized(_plain_gate(s["gate_up"]), s["format"])
    summed, y = _plain_norm(s["x"], s["residual"], s["weight"])
    if kind == "norm":
        return *_quantized(y, s["format"]), summed
    both = _plain_product(*_quantized(y, s["a"]), s["gate_up"], s["gate_up_scales"], torch.bfloat16)
    return _plain_product(*_quantized(_plain_gate(both), s["a"]), s["down"], s["down_scales"], torch.bfloat16), summed


def _held(m: int, k: int, kind: str) -> float:
    """Bytes of m x k quantised elements and their scales."""
    size, block, scale = _FORMATS[kind]
    return m * (k * size + _blocks(k, block) * scale)


def work(case: dict) -> dict:
    kind = case["kind"]
    if kind == "product":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": _held(m, k, case["a"]) + _held(n, k, "fp4") + m * n * _BYTES[case["out"]], "flops": 2 * m * n * k}
    if kind == "feed_forward":
        t, h, i = case["t"], case["h"], case["i"]
        return {"bytes": _held(2 * i, h, "fp4") + _held(h, i, "fp4") + 2 * h + 8 * t * h, "flops": 6 * t * h * i}
    m, k = case["m"], case["k"]
    size, q = _BYTES[case["dtype"]], _held(m, k, case["format"])
    if kind == "round_trip":   # two operators: what the first one writes the second one reads
        return {"bytes": 2 * m * k * size + 2 * q, "flops": 3 * m * k}
    if kind == "gate":
        return {"bytes": 2 * m * k * size + q, "flops": 8 * m * k}
    return {"bytes": m * k * size * (3 if case["residual"] else 1) + k * size + q, "flops": 8 * m * k}


def _nearest64(y, kind: str):
    """The element type's number nearest to y, ties to even: by the step between its numbers where y lies."""
    exponent = torch.frexp(y.abs()).exponent - 1
    low, bits, most = (0, 1, 6.0) if kind == "fp4" else (-6, 3, 448.0)
    step = torch.exp2((exponent.clamp(min=low) - bits).double())
    return (torch.round(y / step) * step).clamp(-most, most)


def _scaled64(x, kind: str):
    """(x over its scales before it is rounded, the scales spread over the elements, the scales)."""
    block, k = _FORMATS[kind][1], x.shape[-1]
    parts = [part.abs().amax(dim=-1) for part in x.split(block, dim=-1)]
    most = torch.stack(parts, dim=-1)
    if kind == "fp8_128":
        scales = torch.maximum(most / 448, torch.full_like(most, 2.0 ** -126))
    else:
        exponent = torch.where(most == 0, -200, torch.frexp(most).exponent - 1 - (2 if kind == "fp4" else 8))
        scales = torch.exp2(exponent.clamp(min=-127).double())
    wide = scales[..., torch.arange(k, device=x.device) // block]
    return x / wide, wide, scales


def _represented64(x, kind: str):
    """What a microscaled copy of x stands for."""
    y, wide, _ = _scaled64(x, kind)
    return _nearest64(y, kind) * wide


def _values64(q, scales):
    """The numbers of microscaled elements, by their bits."""
    bits = q.view(torch.uint8).int()
    if q.dtype == _FP4:
        bits = torch.stack([bits % 16, bits // 16], dim=-1).flatten(-2)
        sign, exponent, mantissa, bias, places = bits // 8, bits // 2 % 4, bits % 2, 1, 1
    else:
        sign, exponent, mantissa, bias, places = bits // 128, bits // 8 % 16, bits % 8, 7, 3
    fraction = mantissa.double() / 2 ** places + (exponent > 0)
    value = fraction * torch.exp2((exponent.clamp(min=1) - bias).double()) * (1 - 2 * sign)
    power = torch.exp2(scales.view(torch.uint8).double() - 127)
    return value * power[..., torch.arange(value.shape[-1], device=q.device) // 32]


def _bf16(x):
    return x.to(torch.bfloat16).double()


def _norm64(s: dict):
    """(the sum or None, the norm)."""
    x = s["x"].double()
    h = x if s["residual"] is None else x + s["residual"].double()
    held = h.to(s["x"].dtype).double()
    mean = torch.sum(held * held, dim=1) / held.shape[1]
    return (None if s["residual"] is None else h), held / torch.sqrt(mean + _EPS)[:, None] * s["weight"].double()


def _gate64(both):
    width = both.shape[1] // 2
    gate, up = both[:, :width].double(), both[:, width:].double()
    return gate / (1 + (-gate).exp()) * up


def exact(case: dict, seed: int):
    """The definition in 64 bits.  8-bit elements that are returned as they are held are given before they are rounded."""
    s, kind = prepare(case, seed), case["kind"]
    if kind == "round_trip":
        x = s["x"].double()
        return _represented64(x, case["format"]), _scaled64(x, case["format"])[2]
    if kind == "product":
        return torch.mm(_values64(s["a"], s["a_scales"]), _values64(s["b"], s["b_scales"]).t())
    if kind == "gate":
        y, _, scales = _scaled64(_gate64(s["gate_up"]), case["format"])
        return y, scales
    summed, y = _norm64(s)
    if kind == "norm":
        y, _, scales = _scaled64(y, case["format"])
        return y, scales, summed
    # (the 16-bit values between the products are part of the definition)
    both = _bf16(torch.mm(_represented64(y, case["a"]), _values64(s["gate_up"], s["gate_up_scales"]).t()))
    return torch.mm(_represented64(_gate64(both), case["a"]), _values64(s["down"], s["down_scales"]).t()), summed
