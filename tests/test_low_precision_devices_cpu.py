"""Tensors of more than one GPU, or of another one than the current, in the 8-bit float and mixture-of-experts entry points.  No
GPU is needed: the tensors have a device and an address, and nothing reads through it."""
import contextlib

import pytest
import torch

from vecops_amd import capi

FP8 = torch.float8_e4m3fn


def elsewhere(device, dtype, *shape):
    strides, step = [], 1
    for n in reversed(shape):
        strides.insert(0, step)
        step *= n
    storage = torch._C._construct_storage_from_data_pointer(0x10000, torch.device(device), step * dtype.itemsize)
    return torch._C._construct_CUDA_Tensor_From_Storage_And_Metadata(
        {"device": torch.device(device), "dtype": dtype, "size": shape, "stride": tuple(strides), "storage_offset": 0,
         "nbytes": step * dtype.itemsize}, storage)


T, E, H, I, TOP = 4, 3, 128, 64, 2
BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32
# the positional tensors of each entry point, and those that may be left out
CALLS = {
    "quantize_fp8_block": ([(BF16, T, H), (FP8, T, H), (F32, T, 1)], {}),
    "matmul_fp8_block": ([(FP8, T, H), (F32, T, 1), (FP8, H, H), (F32, 1, 1), (BF16, T, H)], {"workspace": (torch.uint8, 1 << 20)}),
    "moe_experts": ([(BF16, T, H), (I32, T, TOP), (F32, T, TOP), (FP8, E, 2 * I, H), (FP8, E, H, I), (F32, T, H)],
                    {"gate_up_scales": (F32, E, 1, 1), "down_scales": (F32, E, 1, 1), "workspace": (torch.uint8, 1 << 20)}),
    "moe_layer": ([(BF16, T, H), (F32, E, H), (FP8, E, 2 * I, H), (FP8, E, H, I), (I32, T, TOP), (F32, T, TOP), (F32, T, H)],
                  {"gate_up_scales": (F32, E, 1, 1), "down_scales": (F32, E, 1, 1), "workspace": (torch.uint8, 1 << 20)}),
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


@pytest.mark.parametrize("name", CALLS)
def test_tensors_of_another_device_than_the_current(name, monkeypatch):
    """The work goes to their device; a stream of another one is refused."""
    class Library:
        def __getattr__(self, entry):
            return lambda *a: 0 if entry.endswith("_workspace") else launched.append((entry, current[-1], a[-1])) or 0

    class Stream:
        def __init__(self, device, handle):
            self.device, self.cuda_stream = torch.device(device), handle

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
