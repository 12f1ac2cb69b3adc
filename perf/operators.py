"""The calls that the low-precision and mixture-of-experts operators are measured by: quantisation to 8-bit floats with a
scale for each block of 128, the product of such operands, a mixture-of-experts layer for a few tokens and its experts
alone, from single tokens that are bound by launches and latency to prefill products bound by the matrix cores.

``listed()`` names twelve of them, ``draw(rng)`` gives another of the same kinds and ranges, ``prepare`` makes what a
program holds before the call, ``run`` is one call: of the framework's operators where ``own`` is true, else of their plain
form in elementary torch operations.  ``exact`` is the same in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

_TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4, "fp8": 1}
_BLOCK = 128


def listed() -> list[dict]:
    return [
        # the activations of a few decoded tokens in front of a product: latency
        {"name": "quantize_decode", "kind": "quantize", "m": 4, "k": 4096, "dtype": "bf16", "rows": 1},
        # the activations of a long prompt
        {"name": "quantize_prefill", "kind": "quantize", "m": 4096, "k": 14336, "dtype": "bf16", "rows": 1},
        # a checkpoint's weights, blocks of 128 x 128, extents that are no multiple of the block
        {"name": "quantize_weights_odd", "kind": "quantize", "m": 11000, "k": 4001, "dtype": "bf16", "rows": 128},
        # one token through a projection: the weights' bytes once
        {"name": "product_m1", "kind": "product", "m": 1, "n": 14336, "k": 4096, "out": "bf16"},
        # sixteen sequences decoded together, long K
        {"name": "product_m16", "kind": "product", "m": 16, "n": 4096, "k": 14336, "out": "bf16"},
        # a short prompt
        {"name": "product_m128", "kind": "product", "m": 128, "n": 11008, "k": 4096, "out": "bf16"},
        # extents that line up with nothing, single-precision results
        {"name": "product_ragged", "kind": "product", "m": 777, "n": 1000, "k": 3001, "out": "f32"},
        # a feed-forward projection of a long prompt (the largest case)
        {"name": "product_prefill", "kind": "product", "m": 4096, "n": 11008, "k": 4096, "out": "bf16"},
        # one token through a layer of many small experts
        {"name": "layer_t1", "kind": "layer", "t": 1, "e": 64, "top": 6, "h": 2048, "i": 1408, "weights": "bf16",
         "scoring": "softmax", "renormalize": True},
        # a batch of sequences through many small experts in 8-bit floats, sigmoid scores with a balancing bias
        {"name": "layer_t64_fp8", "kind": "layer", "t": 64, "e": 128, "top": 8, "h": 2048, "i": 768, "weights": "fp8",
         "scoring": "sigmoid", "renormalize": True},
        # sixteen sequences through few large experts, chosen by the program's own router
        {"name": "experts_t16", "kind": "experts", "t": 16, "e": 8, "top": 2, "h": 4096, "i": 14336, "weights": "bf16"},
        # half-precision experts with extents that line up with nothing; some choices live on another device
        {"name": "experts_t5_odd", "kind": "experts", "t": 5, "e": 60, "top": 4, "h": 1001, "i": 1411, "weights": "f16"},
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
    kind = rng.choice(["quantize", "product", "product", "product", "layer", "layer", "experts", "experts"])
    if kind == "quantize":
        return {"kind": kind, "m": _size(rng, 1, 16384, (1, 1, 16)), "k": _size(rng, 64, 16384),
                "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "rows": rng.choice([1, 1, 128])}
    if kind == "product":
        return {"kind": kind, "m": _size(rng, 1, 4096, (1, 1, 16)), "n": _size(rng, 256, 14336, (1, 16, 64, 128)),
                "k": _size(rng, 128, 14336, (1, 16, 128, 128)), "out": rng.choice(["bf16", "bf16", "f16", "f32"])}
    e = _size(rng, 4, 160, (1, 4, 8))
    case = {"kind": kind, "t": _size(rng, 1, 128, (1, 1, 8)), "e": e, "top": rng.randint(1, min(8, e)),
            "h": _size(rng, 512, 4096, (1, 16, 128, 128)), "i": _size(rng, 256, 14336, (1, 16, 128, 128)),
            "weights": rng.choice(["bf16", "bf16", "f16", "fp8", "fp8"])}
    if kind == "layer":
        case |= {"scoring": rng.choice(["softmax", "sigmoid"]), "renormalize": rng.choice([True, True, False])}
    return case


def draw(rng) -> dict:
    most, weights = max(map(_cost, listed())), 8 * 3 * 4096 * 14336
    while True:
        case = _drawn(rng)
        if _cost(case) <= most and ("e" not in case or case["e"] * 3 * case["h"] * case["i"] <= weights):
            return case


def _blocks(extent: int) -> int:
    return -(-extent // _BLOCK)


def _scale(amax):
    """An e4m3 number is at most 448; a block of zeros keeps a scale that can be divided by."""
    return (amax / 448.0).clamp(min=2.0 ** -126)


def _quantized(x, rows: int):
    """The plain form of the quantiser: x [.., M, K] -> (q, scales), blocks of `rows` x 128."""
    m, k = x.shape[-2:]
    i, g = -(-m // rows), _blocks(k)
    x = torch.nn.functional.pad(x.float(), (0, g * _BLOCK - k, 0, i * rows - m)).unflatten(-1, (g, _BLOCK)).unflatten(-3, (i, rows))
    scales = _scale(x.abs().amax(dim=(-1, -3)))
    q = (x / scales[..., :, None, :, None]).to(torch.float8_e4m3fn)
    return q.flatten(-2).flatten(-3, -2)[..., :m, :k], scales


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

    def weights(self, shape, kind: str):
        """(weights, their scales or None), of the deviation that keeps a product's result near its input's."""
        if kind == "fp8":
            parts = [_quantized(self.normal(shape[1:], shape[-1] ** -0.5), _BLOCK) for _ in range(shape[0])]
            return torch.stack([q.contiguous() for q, _ in parts]), torch.stack([s for _, s in parts])
        out = torch.empty(shape, dtype=_TORCH[kind], device="cuda")
        for part in out:
            part.copy_(self.normal(shape[1:], shape[-1] ** -0.5))
        return out, None


def prepare(case: dict, seed: int) -> dict:
    """Operands, outputs and what a program keeps from call to call."""
    r, kind = _Random(seed), case["kind"]
    s = dict(case)
    if kind == "quantize":
        m, k = case["m"], case["k"]
        s["x"] = r.activations((m, k), _TORCH[case["dtype"]]) if case["rows"] == 1 else r.normal((m, k), 0.02, _TORCH[case["dtype"]])
        s["q"] = torch.empty((m, k), dtype=torch.float8_e4m3fn, device="cuda")
        s["q_scales"] = torch.empty((-(-m // case["rows"]), _blocks(k)), device="cuda")
        return s
    if kind == "product":
        m, n, k = case["m"], case["n"], case["k"]
        a, s["a_scales"] = _quantized(r.activations((m, k), torch.bfloat16), 1)
        b, s["b_scales"] = _quantized(r.normal((n, k), k ** -0.5), _BLOCK)
        s["a"], s["b"] = a.contiguous(), b.contiguous()
        s["c"] = torch.empty((m, n), dtype=_TORCH[case["out"]], device="cuda")
        return s
    t, e, top, h, i = (case[name] for name in ("t", "e", "top", "h", "i"))
    dtype = torch.float16 if case["weights"] == "f16" else torch.bfloat16
    s["x"] = r.activations((t, h), dtype)
    s["gate_up"], s["gate_up_scales"] = r.weights((e, 2 * i, h), case["weights"])
    s["down"], s["down_scales"] = r.weights((e, h, i), case["weights"])
    s["out"] = torch.empty((t, h), dtype=dtype, device="cuda")
    if kind == "layer":
        s["router"] = r.normal((e, h), h ** -0.5, dtype)
        s["bias"] = r.normal((e,), 0.05) if case["scoring"] == "sigmoid" else None
        s["ids"] = torch.empty((t, top), dtype=torch.int32, device="cuda")
        s["chosen"] = torch.empty((t, top), device="cuda")
        return s
    noise = torch.rand((t, e), generator=r.generator, device="cuda")
    s["ids"] = noise.argsort(dim=-1)[:, :top].to(torch.int32)
    s["ids"][noise[:, :top] < 0.05] = -1
    s["chosen"] = torch.softmax(r.normal((t, top)), dim=-1)
    return s


def _dequantized(q, scales, rows: int):
    """fp32 values of q [.., M, K] with a scale for each block of `rows` x 128."""
    m, k = q.shape[-2:]
    wide = scales.repeat_interleave(rows, dim=-2)[..., :m, :].repeat_interleave(_BLOCK, dim=-1)[..., :k]
    return q.float() * wide


def _plain_route(s: dict):
    """(ids, weights, their weights spread over all experts)."""
    logits = s["x"].float() @ s["router"].float().t()
    score = torch.softmax(logits, dim=-1) if s["scoring"] == "softmax" else torch.sigmoid(logits)
    key = logits if s["bias"] is None else score + s["bias"]
    ids = key.sort(dim=-1, descending=True, stable=True).indices[:, :s["top"]]
    weights = score.gather(1, ids)
    if s["renormalize"]:
        weights = weights / weights.sum(dim=-1, keepdim=True)
    return ids, weights


def _plain_experts(s: dict, ids, weights):
    """Every expert for every token, weighted by zero where it was not chosen."""
    e, i, h, t = s["e"], s["i"], s["h"], s["t"]
    local = (ids >= 0) & (ids < e)
    spread = torch.zeros((t, e), device="cuda").scatter_add_(1, torch.where(local, ids, 0).long(), torch.where(local, weights, 0.0))
    first = s["gate_up"].float() if s["gate_up_scales"] is None else _dequantized(s["gate_up"], s["gate_up_scales"], _BLOCK)
    gate_up = (s["x"].float() @ first.view(e * 2 * i, h).t()).view(t, e, 2, i)
    hidden = gate_up[:, :, 0] * torch.sigmoid(gate_up[:, :, 0]) * gate_up[:, :, 1] * spread[:, :, None]
    second = s["down"].float() if s["down_scales"] is None else _dequantized(s["down"], s["down_scales"], _BLOCK)
    return (hidden.reshape(t, e * i) @ second.transpose(1, 2).reshape(e * i, h)).to(s["out"].dtype)


def run(s: dict):
    kind = s["kind"]
    if own:
        from vecops_amd import capi
        if kind == "quantize":
            capi.quantize_fp8_block(s["x"], s["q"], s["q_scales"], block_rows=s["rows"])
            return s["q"], s["q_scales"]
        if kind == "product":
            return capi.matmul_fp8_block(s["a"], s["a_scales"], s["b"], s["b_scales"], s["c"])
        if kind == "experts":
            return capi.moe_experts(s["x"], s["ids"], s["chosen"], s["gate_up"], s["down"], s["out"],
                                    gate_up_scales=s["gate_up_scales"], down_scales=s["down_scales"])
        capi.moe_layer(s["x"], s["router"], s["gate_up"], s["down"], s["ids"], s["chosen"], s["out"],
                       scoring=s["scoring"], renormalize=s["renormalize"], bias=s["bias"],
                       gate_up_scales=s["gate_up_scales"], down_scales=s["down_scales"])
        return s["ids"], s["chosen"], s["out"]
    if kind == "quantize":
        return _quantized(s["x"], s["rows"])
    if kind == "product":
        return (_dequantized(s["a"], s["a_scales"], 1) @ _dequantized(s["b"], s["b_scales"], _BLOCK).t()).to(s["c"].dtype)
    if kind == "experts":
        return _plain_experts(s, s["ids"], s["chosen"])
    ids, weights = _plain_route(s)
    return ids.to(torch.int32), weights, _plain_experts(s, ids, weights)


def work(case: dict) -> dict:
    kind = case["kind"]
    if kind == "quantize":
        m, k = case["m"], case["k"]
        scales = -(-m // case["rows"]) * _blocks(k)
        return {"bytes": m * k * (_BYTES[case["dtype"]] + 1) + 4 * scales, "flops": 3 * m * k}
    if kind == "product":
        m, n, k = case["m"], case["n"], case["k"]
        scales = (m + _blocks(n)) * _blocks(k)
        return {"bytes": (m + n) * k + 4 * scales + m * n * _BYTES[case["out"]], "flops": 2 * m * n * k}
    t, e, top, h, i = (case[name] for name in ("t", "e", "top", "h", "i"))
    # experts that t tokens name between them, each at random
    named = e * (1 - (1 - top / e) ** t)
    scales = 4 * (2 * _blocks(2 * i) * _blocks(h) if case["weights"] == "fp8" else 0)
    router = e * h if kind == "layer" else 0
    return {"bytes": named * (3 * h * i * _BYTES[case["weights"]] + scales) + 2 * router + 4 * t * h + 8 * t * top,
            "flops": 6 * t * top * h * i + 2 * t * router}


def _scales64(scales, rows: int, columns: int, per_row: int):
    """Each element's scale, by its indices."""
    i = torch.arange(rows, device="cuda") // per_row
    j = torch.arange(columns, device="cuda") // _BLOCK
    return scales.double()[i[:, None], j[None, :]]


def exact(case: dict, seed: int):
    """The definition in 64 bits.  An 8-bit result is given before it is rounded."""
    s, kind = prepare(case, seed), case["kind"]
    if kind == "quantize":
        x, rows = s["x"].double(), case["rows"]
        m, k = x.shape
        scales = torch.empty_like(s["q_scales"], dtype=torch.float64)
        for g in range(scales.shape[1]):
            most = x[:, g * _BLOCK:(g + 1) * _BLOCK].abs().max(dim=1).values
            if rows > 1:
                most = torch.stack([part.max() for part in most.split(rows)])
            scales[:, g] = torch.maximum(most / 448, torch.full_like(most, 2.0 ** -126))
        return x / _scales64(scales, m, k, rows), scales
    if kind == "product":
        (m, k), n = s["a"].shape, s["b"].shape[0]
        b = s["b"].double() * _scales64(s["b_scales"], n, k, _BLOCK)
        return torch.mm(s["a"].double() * _scales64(s["a_scales"], m, k, 1), b.t())
    x, ids, weights = s["x"].double(), s["ids"], s["chosen"].double()
    if kind == "layer":
        logits = torch.mm(x, s["router"].double().t())
        if case["scoring"] == "softmax":
            score = (logits - logits.max(dim=1, keepdim=True).values).exp()
            score = score / score.sum(dim=1, keepdim=True)
        else:
            score = 1 / (1 + (-logits).exp())
        key = logits if s["bias"] is None else score + s["bias"].double()
        ids = torch.argsort(key, dim=1, descending=True, stable=True)[:, :case["top"]].to(torch.int32)
        weights = torch.stack([score[row, ids[row].long()] for row in range(case["t"])])
        if case["renormalize"]:
            weights = weights / weights.sum(dim=1, keepdim=True)
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    i, h = case["i"], case["h"]
    for e in range(case["e"]):
        rows, places = (ids == e).nonzero(as_tuple=True)
        if len(rows):
            first, second = s["gate_up"][e].double(), s["down"][e].double()
            if case["weights"] == "fp8":
                first = first * _scales64(s["gate_up_scales"][e], 2 * i, h, _BLOCK)
                second = second * _scales64(s["down_scales"][e], h, i, _BLOCK)
            both = torch.mm(x[rows], first.t())
            gate, up = both[:, :i], both[:, i:]
            hidden = gate / (1 + (-gate).exp()) * up
            out.index_add_(0, rows, torch.mm(hidden, second.t()) * weights[rows, places][:, None])
    return out if kind == "experts" else (ids, weights, out)
