"""HeadRotation and CacheAppend made on one stream and run on another: what the constructor puts on the
device (weights, the error word) is there when it returns."""
import types

import pytest

torch = pytest.importorskip("torch")

from paged_decode import rotary
from paged_decode.layout import Layout


def test_constructors_wait_for_what_they_put_on_the_device(monkeypatch):
    """On the host: the stream is waited for, and after the copies."""
    log = []
    stream = types.SimpleNamespace(synchronize=lambda: log.append("wait"))
    monkeypatch.setattr(rotary, "_cuda_device", lambda device: torch.device("cpu"))
    monkeypatch.setattr(rotary._native, "load", lambda: None)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: stream)
    zeros, to = torch.zeros, torch.Tensor.to
    monkeypatch.setattr(torch, "zeros", lambda *a, **kw: log.append("zeros") or zeros(*a, **kw))
    monkeypatch.setattr(torch.Tensor, "to", lambda x, *a, **kw: log.append("copy") or to(x, *a, **kw))
    rotation = rotary.HeadRotation(64, q_weight=torch.ones(64), k_weight=torch.ones(64).half())
    assert log[-1] == "wait" and {"zeros", "copy"} <= set(log)
    log.clear()
    rotary.CacheAppend(Layout(2, 4, 2, 64, 16, 8), rotation)
    assert log[-1] == "wait" and "zeros" in log


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="NVIDIA GPU required")
def test_made_behind_slow_work_on_another_stream():
    side, weight = torch.cuda.Stream(), torch.full((128,), 2.0, device="cuda")
    q = torch.randn((40, 8, 128), device="cuda")
    positions = torch.zeros(40, dtype=torch.int32, device="cuda")
    want = rotary.HeadRotation(128, q_weight=weight, eps=0.0).run(q, None, positions)[0]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)                       # some 10 ms of the side stream
        rotation = rotary.HeadRotation(128, q_weight=weight, eps=0.0)
    got = rotation.run(q, None, positions)[0]
    assert torch.equal(got, want) and rotation.read_errors() == 0
