"""The timed cases of the dense operators call the library where torch works: on the current device and its current stream (no GPU)."""
import importlib.util
import os
import types

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture()
def operators():
    spec = importlib.util.spec_from_file_location("operators_under_test", os.path.join(ROOT, "perf", "operators.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_calls_follow_the_current_device_and_stream(operators, monkeypatch):
    import torch

    from denno_beta_b200 import cuda

    class Ctx:
        def __init__(self, device):
            self.device = device

        def set_stream(self, stream):
            self.stream = stream

    now = types.SimpleNamespace(device=0, stream=0)
    monkeypatch.setattr(cuda, "CudaCtx", Ctx)
    for where, what, value in ((torch.cuda, "current_device", lambda: now.device), (torch.cuda, "current_stream", lambda: types.SimpleNamespace(cuda_stream=now.stream)),
                               (torch._C, "_cuda_getDevice", lambda: now.device), (torch._C, "_cuda_getCurrentRawStream", lambda device: now.stream)):
        monkeypatch.setattr(where, what, value, raising=False)
    made = {}
    for device, stream in [(0, 0), (0, 0x5000), (1, 0), (0, 0), (1, 0x7000), (0, 0x5000)]:
        now.device, now.stream = device, stream
        ctx = operators._context()[1]
        assert (ctx.device, ctx.stream) == (device, stream or 1)  # 1: the default stream by its handle
        assert made.setdefault((device, stream), ctx) is ctx  # a context, and what it has laid out, is kept
