"""The order of streams in the example of a decoder layer on 8-bit floats, and that it runs."""
import importlib.util
import os
import sys

import pytest
import torch


@pytest.fixture
def example():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "fp8_decode_layer.py")
    spec = importlib.util.spec_from_file_location("fp8_decode_layer", at)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_warm_up_waits_for_the_weights(example, monkeypatch):
    """What runs on the side stream reads what the current stream has written: the one waits for the other first.  (No GPU: a
    layer and streams that only note what is asked of them.)"""
    done, stack = [], ["current"]

    class Stream:
        def __init__(self, name="side"):
            self.name = name

        def wait_stream(self, other):
            done.append(f"{self.name} waits for {other.name}")

    class On:
        def __init__(self, name):
            self.name = name

        def __enter__(self):
            stack.append(self.name)

        def __exit__(self, *error):
            stack.pop()

    class Layer:
        def __init__(self, *a, **k):
            done.append(f"weights on {stack[-1]}")
            self.ids = torch.zeros((1, 1), dtype=torch.int32)

        def step(self, attended):
            done.append(f"step on {stack[-1]}")

    class Event:
        def __init__(self, **k):
            pass

        def record(self):
            pass

        def elapsed_time(self, other):
            return 1.0

    class Graph:
        def replay(self):
            pass

    monkeypatch.setattr(sys, "argv", ["fp8_decode_layer.py", "--tokens", "1", "--steps", "1"])
    monkeypatch.setattr(example, "Layer", Layer)
    monkeypatch.setattr(torch, "randn", lambda shape, device=None: torch.zeros(shape))
    for name, value in {"Stream": Stream, "stream": lambda s: On(s.name), "current_stream": lambda: Stream(stack[-1]), "CUDAGraph": Graph,
                        "graph": lambda g: On("capture"), "Event": Event, "synchronize": lambda: None}.items():
        monkeypatch.setattr(torch.cuda, name, value)
    example.main()
    assert done == ["weights on current", "side waits for current", "step on side", "current waits for side", "step on capture"]


@pytest.mark.gpu
def test_example_runs(device, example, monkeypatch, capsys):
    monkeypatch.setattr(sys, "argv", ["fp8_decode_layer.py", "--tokens", "3", "--steps", "2"])
    example.main()
    assert "us a step" in capsys.readouterr().out
