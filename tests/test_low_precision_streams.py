"""On which stream the 8-bit float and mixture-of-experts entry points get the scratch that a call needs."""
import contextlib

import pytest
import torch

from vecops_amd import capi

FP8 = torch.float8_e4m3fn


def calls(device, t=6):
    """Each entry point that may need scratch, on operands where it does, as functions of the stream."""
    h, i, e, top = 144, 40, 5, 2
    g = torch.Generator().manual_seed(1)
    n = lambda *shape: torch.randn(shape, generator=g).to(device)  # noqa: E731
    x, router, gate_up, down = n(t, h).bfloat16(), n(e, h), n(e, 2 * i, h).bfloat16(), n(e, h, i).bfloat16()
    ids, weights, out = torch.zeros((t, top), dtype=torch.int32, device=device), torch.ones((t, top), device=device), torch.empty((t, h), device=device)
    a, b = n(h, t).clamp(-400, 400).to(FP8).t(), n(h, 130).clamp(-400, 400).to(FP8).t()   # (k not contiguous: copied)
    sa, sb, c = n(t, 2), n(2, 2), torch.empty((t, 130), device=device)
    return {"product": (lambda stream: capi.matmul_fp8_block(a, sa, b, sb, c, stream=stream)),
            "experts": (lambda stream: capi.moe_experts(x, ids, weights, gate_up, down, out, stream=stream)),
            "layer": (lambda stream: capi.moe_layer(x, router, gate_up, down, ids, weights, out, stream=stream))}


@pytest.mark.parametrize("name", ["product", "experts", "layer"])
def test_scratch_is_taken_on_the_stream_that_is_named(name, monkeypatch):
    """What the allocator hands out is free in the order of the stream it is handed out on.  (No GPU: the library's calls are
    counted, the streams are names.)"""
    class Library:
        def __getattr__(self, entry):
            return lambda *a: 4096 if entry.endswith("_workspace") else launched.append(entry) or 0

    class Stream:
        cuda_stream, device = 7, torch.device("cuda:0")

    current, taken, launched, stream = [None], [], [], Stream()

    @contextlib.contextmanager
    def on(which):
        current.append(which)
        yield
        current.pop()

    call, empty = calls("cpu")[name], torch.empty

    def counted(*a, **k):
        taken.append(current[-1])
        return empty(*a, **k)

    monkeypatch.setattr(capi, "lib", Library)
    monkeypatch.setattr(capi, "_on_one_device", lambda *a: stream.device)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "stream", on)
    monkeypatch.setattr(torch, "empty", counted)
    call(stream)
    assert len(launched) == 1 and taken == [stream]


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["product", "experts", "layer"])
def test_scratch_comes_back_on_the_stream_that_was_named(device, name, monkeypatch):
    """The scratch of a call on a named stream is never handed to the current stream while it may be in use."""
    call, empty, taken = calls(device)[name], torch.empty, []

    def noted(*a, **k):
        taken.append((torch.cuda.current_stream().cuda_stream, empty(*a, **k)))
        return taken[-1][1]

    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    for given in (stream, torch.cuda.ExternalStream(stream.cuda_stream)):
        with monkeypatch.context() as m:
            m.setattr(torch, "empty", noted)
            call(given)
        (on, scratch), = taken
        assert on == stream.cuda_stream
        at, size = scratch.data_ptr(), scratch.numel()
        taken.clear()
        del scratch
        here = [empty(size, dtype=torch.uint8, device=device) for _ in range(4)]
        assert at not in [v.data_ptr() for v in here]
        stream.synchronize()
