"""Host side of the 4-bit cache's and the page table's calls, without a GPU."""
from __future__ import annotations

import ctypes as C
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


@pytest.mark.parametrize("max_blocks,n_kv,rows,heads,word", [
    (4, 2, (1 << 20) + 1, 4, b"n_rows"), (4, 2, -1, 4, b"n_rows"), (1 << 26, 2, 8, 4, b"pages"),
    (1 << 20, 8, 1 << 10, 32, b"pages"), (4, 1 << 16, 1, 1 << 16, b"KV heads")])
def test_a_workspace_is_refused_where_the_decode_call_is(max_blocks, n_kv, rows, heads, word):
    """Both answer alike, before any work on a device."""
    from axion_b200 import _lib
    lib = _lib.load()
    c = C.byref(_lib.axkv4_cache_t(4096, 4096, 1 << 21, max_blocks, 8, n_kv, 64, 16))
    assert lib.axkv4_decode_attn_workspace(c, rows, heads) == -1
    assert word in lib.axq8_last_error() and b"workspace" in lib.axq8_last_error()
    rc = lib.axkv4_decode_attn(c, 4096, heads * 64, rows, heads, None, 4096, 4096, 4096, 1 << 40, None)
    assert rc in (_lib.AXQ8_ERR_INVALID, _lib.AXQ8_ERR_UNSUPPORTED) and word in lib.axq8_last_error()


@pytest.mark.parametrize("chunks,rows", [(65536, 1), (1, (1 << 24) + 1), (-1, 1), (1, -1)])
def test_a_workspace_is_refused_where_the_chunk_call_is(chunks, rows):
    from axion_b200 import _lib
    lib = _lib.load()
    c = C.byref(_lib.axkv4_cache_t(4096, 4096, 1 << 17, 4, 8, 2, 64, 16))
    assert lib.axkv4_chunk_attn_workspace(c, chunks, rows, 4) == -1
    assert b"chunks of at most" in lib.axq8_last_error()
    assert lib.axkv4_chunk_attn(c, 4096, 256, 8, chunks, rows, 4, None, 4096, 4096, 4096, 4096, 1 << 40,
                                None) == _lib.AXQ8_ERR_INVALID
