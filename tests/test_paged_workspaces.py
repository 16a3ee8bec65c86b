"""Which workspace a call of a paged operator gets: one per device and stream, and one per
captured graph. Host only: the device, the capture and the memory are stand-ins."""

import pytest
import torch

from iron_b200 import _lib
from iron_b200.operators import PageFork, TreeAttention

SIZES = dict(num_kv_heads=2, head_dim=64, page_size=16, num_pages=8, max_pages=4)


@pytest.fixture
def gpu(monkeypatch):
    """A GPU's state: `device`, and `capture`, the id of the capture under way (0: none)."""

    class State:
        device, capture = 0, 0

    s = State()
    host = {n: getattr(torch, n) for n in ("zeros", "empty")}
    monkeypatch.setattr(torch.cuda, "current_device", lambda: s.device)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: s.capture != 0)
    for n in host:
        monkeypatch.setattr(torch, n, lambda *a, _n=n, device=None, **k: host[_n](*a, **k))

    def call(fn, stream, out):
        assert fn == "iron_capture_id"
        out._obj.value = s.capture

    monkeypatch.setattr(_lib, "call", call)
    return s


@pytest.mark.parametrize("make", [lambda: TreeAttention(batch=2, num_nodes=4, num_heads=4, **SIZES),
                                  lambda: PageFork(slots=2, num_layers=1, **SIZES)])
def test_one_per_device_stream_and_graph(make, gpu, monkeypatch):
    op = make()
    monkeypatch.setattr(type(op), "workspace_bytes", lambda self: 64)
    monkeypatch.setattr(type(op), "counter_bytes", lambda self: 32)
    first = op._workspace(0)
    assert op._workspace(0) == first
    assert op._workspace(7) != first
    gpu.device = 1  # the default stream is 0 on every device
    assert op._workspace(0) != first
    gpu.device = 0
    assert op._workspace(0) == first
    gpu.capture = 11
    graph = op._workspace(7)
    assert graph not in (first, op._workspace(8))  # streams of one graph may run side by side
    assert op._workspace(7) == graph
    held = op._captured
    gpu.capture = 12
    assert op._workspace(7) != graph and len(op._captured) == 1
    assert any(w[0] == graph[0] for w in held.values())
    gpu.capture = 0
    assert op._workspace(0) == first and op._captured == {}


def test_a_graphs_counters_start_at_zero(gpu, monkeypatch):
    op = TreeAttention(batch=2, num_nodes=4, num_heads=4, **SIZES)
    monkeypatch.setattr(type(op), "workspace_bytes", lambda self: 64)
    monkeypatch.setattr(type(op), "counter_bytes", lambda self: 32)
    plain = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, **k: plain(*a, **k).fill_(9))
    gpu.capture = 5
    op._workspace(7)
    (_, _, t), = op._captured.values()
    assert not bool(t[:32].any()) and bool((t[32:] == 9).all())


def test_buffers_of_another_device_are_refused():
    op = PageFork(slots=2, num_layers=1, **SIZES)

    class Buffer:
        is_cuda, device = True, "cuda:1"
        data_ptr = staticmethod(lambda: 4096)
        get_device = staticmethod(lambda: 1)

    with pytest.raises(ValueError, match="buffer 0 of PageFork is on cuda:1, the current device is 0"):
        op._refuse_device([Buffer], 0)
    with pytest.raises(RuntimeError, match="host tensor"):
        op._refuse_device([torch.zeros(2)], 0)
