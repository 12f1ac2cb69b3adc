"""A decoder layer's feed-forward half for a batch of single tokens, on 8-bit floats: an output projection, then a
mixture-of-experts layer.

The weights are quantised once, in blocks of 128 x 128 (``quantize_fp8_block`` with ``block_rows=128``); the activations in front
of the projection at every step, in blocks of 1 x 128.  ``moe_layer`` chooses the experts and runs them on the tokens as they are.

    python examples/fp8_decode_layer.py [--tokens 16] [--steps 20]
"""
import argparse
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch  # noqa: E402

from vecops_amd import capi  # noqa: E402

FP8 = torch.float8_e4m3fn


def blocks(extent: int) -> int:
    return -(-extent // 128)


def quantized_weights(w):
    """[.., N, K] -> (e4m3, a scale for each block of 128 x 128)."""
    q = torch.empty(w.shape, dtype=FP8, device=w.device)
    scales = torch.empty((*w.shape[:-2], blocks(w.shape[-2]), blocks(w.shape[-1])), device=w.device)
    return capi.quantize_fp8_block(w, q, scales, block_rows=128)


class Layer:
    """Weights, and what a step writes: nothing is allocated in ``step``, so that it can be captured in a graph."""

    def __init__(self, tokens: int, hidden: int, inner: int, experts: int, top: int, device="cuda", seed: int = 0):
        g = torch.Generator(device=device).manual_seed(seed)
        n = lambda *shape: torch.randn(shape, generator=g, device=device)  # noqa: E731
        self.proj, self.proj_scales = quantized_weights((n(hidden, hidden) * hidden ** -0.5).bfloat16())
        self.gate_up, self.gate_up_scales = quantized_weights((n(experts, 2 * inner, hidden) * hidden ** -0.5).bfloat16())
        self.down, self.down_scales = quantized_weights((n(experts, hidden, inner) * inner ** -0.5).bfloat16())
        self.router = n(experts, hidden) * hidden ** -0.5
        self.q = torch.empty((tokens, hidden), dtype=FP8, device=device)
        self.scales = torch.empty((tokens, blocks(hidden)), device=device)
        self.x = torch.empty((tokens, hidden), dtype=torch.bfloat16, device=device)
        self.ids = torch.empty((tokens, top), dtype=torch.int32, device=device)
        self.weights = torch.empty((tokens, top), device=device)
        self.out = torch.empty((tokens, hidden), dtype=torch.bfloat16, device=device)
        self.scratch = [torch.empty(size, dtype=torch.uint8, device=device) for size in self.scratch_sizes()]

    def scratch_sizes(self):
        import ctypes
        at = lambda t: ctypes.byref(capi.operand(t))  # noqa: E731
        lib = capi.lib()
        return (lib.vecops_hip_matmul_fp8_block_workspace(at(self.q), at(self.scales), at(self.proj), at(self.proj_scales), at(self.x)),
                lib.vecops_hip_moe_layer_workspace(at(self.x), at(self.ids), at(self.down)))

    def step(self, attended):
        """attended [tokens, hidden] (bf16) -> [tokens, hidden]."""
        capi.quantize_fp8_block(attended, self.q, self.scales)
        capi.matmul_fp8_block(self.q, self.scales, self.proj, self.proj_scales, self.x, workspace=self.scratch[0])
        return capi.moe_layer(self.x, self.router, self.gate_up, self.down, self.ids, self.weights, self.out, scoring="softmax",
                              gate_up_scales=self.gate_up_scales, down_scales=self.down_scales, workspace=self.scratch[1])


def main() -> None:
    parse = argparse.ArgumentParser()
    parse.add_argument("--tokens", type=int, default=16)
    parse.add_argument("--steps", type=int, default=20)
    asked = parse.parse_args()
    layer = Layer(asked.tokens, hidden=2048, inner=768, experts=64, top=6)
    attended = torch.randn((asked.tokens, 2048), device="cuda").bfloat16()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())   # (which makes the weights)
    with torch.cuda.stream(side):   # (once before the capture: kernels are loaded on their first call)
        layer.step(attended)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.step(attended)
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    graph.replay()
    begin.record()
    for _ in range(asked.steps):
        graph.replay()
    end.record()
    torch.cuda.synchronize()
    print(f"{asked.tokens} tokens: {begin.elapsed_time(end) / asked.steps * 1e3:.1f} us a step, "
          f"first token's experts {layer.ids[0].tolist()}")


if __name__ == "__main__":
    main()
