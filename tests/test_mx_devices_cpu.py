"""Tensors of more than one GPU, or of another one than the current, in the microscaled and row entry points, and the stream that
scratch is taken on.  No GPU is needed: the tensors have a device and an address, and nothing reads through it."""
import contextlib

import pytest
import torch

from test_low_precision_devices_cpu import elsewhere
from vecops_amd import capi

FP4, FP8, E8M0 = torch.float4_e2m1fn_x2, torch.float8_e4m3fn, torch.float8_e8m0fnu
BF16, F32 = torch.bfloat16, torch.float32
T, H, N = 4, 128, 96
# the positional tensors of each entry point, and those that may be left out
CALLS = {
    "quantize_mx": ([(BF16, T, H), (FP4, T, H // 2), (E8M0, T, 4)], {}),
    "dequantize_mx": ([(FP8, T, H), (E8M0, T, 4), (F32, T, H)], {}),
    "matmul_mx": ([(FP8, T, H), (E8M0, T, 4), (FP4, N, H // 2), (E8M0, N, 4), (BF16, T, N)], {"workspace": (torch.uint8, 1 << 20)}),
    "rms_norm": ([(BF16, T, H), (F32, H), (FP8, T, H), (F32, T, 1)], {"out": (BF16, T, H), "residual": (BF16, T, H), "summed": (BF16, T, H)}),
    "silu_mul_quantize": ([(BF16, T, 2 * H), (FP8, T, H), (F32, T, 1)], {}),
}


@pytest.mark.parametrize("name", CALLS)
def test_tensors_of_two_devices(name):
    """Each tensor in turn on another device than the rest."""
    positional, named = CALLS[name]
    for odd in [*range(len(positional)), *named]:
        where = lambda at: "cuda:1" if at == odd else "cuda:0"  # noqa: E731, B023
        args = [elsewhere(where(at), *t) for at, t in enumerate(positional)]
        kwargs = {at: elsewhere(where(at), *t) for at, t in named.items()}
        with pytest.raises(ValueError, match="one GPU"):
            getattr(capi, name)(*args, **kwargs)


class Stream:
    def __init__(self, device, handle):
        self.device, self.cuda_stream = torch.device(device), handle


@pytest.mark.parametrize("name", CALLS)
def test_tensors_of_another_device_than_the_current(name, monkeypatch):
    """The work goes to their device; a stream of another one is refused."""
    class Library:
        def __getattr__(self, entry):
            return lambda *a: 0 if entry.endswith("_workspace") else launched.append((entry, current[-1], a[-1])) or 0

    @contextlib.contextmanager
    def on(device):
        current.append(str(device))
        yield
        current.pop()

    launched, current = [], ["cuda:0"]
    monkeypatch.setattr(capi, "lib", Library)
    monkeypatch.setattr(capi, "_calls", capi._NoNativeCalls())
    monkeypatch.setattr(torch.cuda, "device", on)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: Stream(current[-1], {"cuda:0": 10, "cuda:1": 11}[current[-1]]))
    positional, named = CALLS[name]
    args, kwargs = [elsewhere("cuda:1", *t) for t in positional], {at: elsewhere("cuda:1", *t) for at, t in named.items()}
    getattr(capi, name)(*args, **kwargs)
    getattr(capi, name)(*args, **kwargs, stream=Stream("cuda:1", 12))
    entry = "vecops_hip_" + name
    assert launched == [(entry, "cuda:1", 11), (entry, "cuda:1", 12)]
    with pytest.raises(ValueError, match="the stream is cuda:0's"):
        getattr(capi, name)(*args, **kwargs, stream=Stream("cuda:0", 10))


def test_tensors_on_the_host_are_refused():
    for name, (positional, _) in CALLS.items():
        with pytest.raises(ValueError, match="one GPU"):
            getattr(capi, name)(*(torch.empty(shape, dtype=dtype) for dtype, *shape in positional))


def turned_operands(device):
    """A product whose operands have to be copied."""
    q = lambda rows: torch.zeros((H // 2, rows), dtype=torch.uint8, device=device).t().view(FP4)  # noqa: E731
    s = lambda rows: torch.full((rows, 4), 127, dtype=torch.uint8, device=device).view(E8M0)  # noqa: E731
    return q(T), s(T), q(N), s(N), torch.empty((T, N), device=device)


def test_scratch_is_taken_on_the_stream_that_is_named(monkeypatch):
    """What the allocator hands out is free in the order of the stream it is handed out on."""
    class Library:
        def __getattr__(self, entry):
            return lambda *a: 4096 if entry.endswith("_workspace") else launched.append(entry) or 0

    current, taken, launched, stream = [None], [], [], Stream("cuda:0", 7)
    operands, empty = turned_operands("cpu"), torch.empty

    @contextlib.contextmanager
    def on(which):
        current.append(which)
        yield
        current.pop()

    def counted(*a, **k):
        taken.append(current[-1])
        return empty(*a, **k)

    monkeypatch.setattr(capi, "lib", Library)
    monkeypatch.setattr(capi, "_on_one_device", lambda *a: stream.device)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "stream", on)
    monkeypatch.setattr(torch, "empty", counted)
    capi.matmul_mx(*operands, stream=stream)
    assert len(launched) == 1 and taken == [stream]


@pytest.mark.gpu
def test_work_on_a_named_stream(device):
    """Every entry point on a stream of its own, behind work of that stream that is still under way."""
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        big = torch.randn((4096, 4096), device=device)
        for _ in range(8):
            big = big @ big * 1e-3
        x = torch.ones((T, 2 * H), device=device) + big[:T, :2 * H] * 0
    for native in (True, False):
        q, s = torch.zeros((T, H), dtype=torch.uint8, device=device).view(FP4), torch.zeros((T, 8), dtype=torch.uint8, device=device).view(E8M0)
        out = torch.zeros((T, 2 * H), device=device)
        torch.cuda.current_stream().synchronize()
        if native:
            with torch.cuda.stream(side):
                capi.quantize_mx(x, q, s)
                capi.dequantize_mx(q, s, out)
        else:
            capi.quantize_mx(x, q, s, stream=side)
            capi.dequantize_mx(q, s, out, stream=side)
        side.synchronize()
        assert bool((out == 1).all())
