"""Host side of the 4-bit cache's and the page table's calls, without a GPU."""
from __future__ import annotations

import threading

import pytest
import torch

from axion_b200.paged_kv import _DeviceCalls


class Tensor:
    """A workspace of `n` bytes made while `device` was current."""

    def __init__(self, n):
        self.n, self.device = n, Devices.current

    def data_ptr(self):
        return 4096

    def numel(self):
        return self.n


class Devices:
    """Two devices: the current one, and which have a stream under capture."""

    current, capturing = 0, set()

    def __init__(self, index):
        self.index = index

    def __enter__(self):
        self.was, Devices.current = Devices.current, self.index

    def __exit__(self, *exc):
        Devices.current = self.was


@pytest.fixture
def calls(monkeypatch):
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: Devices.current)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: 100 + d)
    monkeypatch.setattr(torch.cuda, "device", Devices)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: Devices.current in Devices.capturing)
    monkeypatch.setattr(torch, "empty", lambda n, dtype=None, device=None: Tensor(n))
    Devices.current, Devices.capturing = 0, set()
    c = _DeviceCalls()
    c._ref, c._dev, c._device, c._ws, c._lock = None, 1, 1, {}, threading.Lock()
    return c


@pytest.mark.parametrize("current", [0, 1])
def test_a_workspace_is_a_graphs_own_where_the_objects_stream_is_captured(calls, current):
    """Whichever device is current: the capture that counts is that of the stream the call goes to."""
    seen = []

    def fn(ref, ws, size, stream):
        seen.append((Devices.current, ws, size, stream))
        return 0

    Devices.current, Devices.capturing = current, {1}
    calls._call_ws(64, fn)
    assert not calls._ws and seen == [(1, 4096, 64, 101)]
    Devices.capturing = {0}                       # the other device's capture is none of ours
    calls._call_ws(64, fn)
    assert list(calls._ws) == [101] and Devices.current == current
