"""perf/operators.py: the library's calls go to the device and the stream that are current."""
import importlib.util
import os

import pytest
import torch

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "perf", "operators.py")


def workloads():
    spec = importlib.util.spec_from_file_location("workloads", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_calls_follow_the_current_device_and_stream(monkeypatch):
    from mimo_prismwing_b200 import runtime as R

    class Fake:
        def __init__(self, device):
            self.device, self.streams = device, []

        @classmethod
        def compile_with_fused_gate_up(cls, device):
            return cls(device)

        def set_stream(self, stream):
            self.streams.append(stream)

        def linear(self, *_, **__):
            return type("Execution", (), {"output": (self.device, self.streams[-1])})

    monkeypatch.setattr(R, "WideMoeRuntime", Fake)
    m = workloads()
    m.own = True
    state = {"case": {"op": "linear", "act": "none", "out": "bf16"}, "x": 0, "weight": 0, "bias": None, "residual": None}
    for device, stream in ((0, "a"), (0, "a"), (0, "b"), (1, "a"), (0, "a"), (1, "c")):
        monkeypatch.setattr(torch.cuda, "current_device", lambda: device)
        monkeypatch.setattr(torch.cuda, "current_stream", lambda: stream)
        monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda _: ord(stream), raising=False)
        assert m.run(state) == (device, stream)
    assert {d: r[0].streams for d, r in m._runtimes.items()} == {0: ["a", "b", "a"], 1: ["a", "c"]}


@pytest.mark.gpu
def test_a_side_stream_and_a_capture_give_the_same():
    m = workloads()
    m.own = True
    small = [c for c in m.listed() if c["name"] in ("norm decode", "norm odd f32", "linear decode", "fp8 down ragged")]
    for case in small:
        state = m.prepare(case, 1)

        def outputs():
            r = m.run(state)
            return [r[k] for k in sorted(r)] if isinstance(r, dict) else [r]

        want = outputs()
        torch.cuda.synchronize()
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            side = outputs()
            s.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                captured = outputs()
            for t in captured:
                t.view(torch.uint8).zero_()
            g.replay()
            s.synchronize()
        for a, b, c in zip(want, side, captured):
            assert torch.equal(a.float(), b.float()) and torch.equal(a.float(), c.float())
