"""The page table over the fp16 and fp32 pages of axkv_cache (include/axkv.h): sequences
that share pages, forked, dropped and compacted, and attention over them through the C ABI."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest
import torch

import kv4_model as km
from test_kv4_gpu import clean_status, dev, ints, status  # noqa: F401

pytestmark = pytest.mark.gpu


class Cache:
    """K and V pages of one layer under a KVPages table, called through the C ABI."""

    def __init__(self, rng, kv, hd, fp32, n_seqs, max_blocks, n_pages):
        from axion_b200 import _lib
        from axion_b200.kv_pages import KVPages
        self.rng, self.kv, self.hd, self.lib, self.check = rng, kv, hd, _lib.load(), _lib.check
        self.type = torch.float32 if fp32 else torch.float16
        self.k, self.v = (torch.full((n_pages, kv, 16, hd), 3.0, dtype=self.type, device="cuda") for _ in range(2))
        self.pages = KVPages.empty([self.k, self.v], n_seqs, max_blocks)
        self.c = _lib.axkv_cache_t(self.k.data_ptr(), self.v.data_ptr(), self.pages.block_table.data_ptr(),
                                   n_pages, max_blocks, kv, hd, 16, int(fp32))
        self.held = [np.zeros((2, 0, kv, hd), np.float64) for _ in range(n_seqs)]

    def append(self, seq, n):
        first = self.held[seq].shape[1]
        x = self.rng.normal(0, 1, (2, n, self.kv, self.hd)).astype(np.float32)
        rows = dev(x.reshape(2, n, -1))
        s, p = ints([seq] * n), ints(range(first, first + n))
        self.check(self.lib.axkv_paged_append(C.byref(self.c), rows[0].data_ptr(), rows[1].data_ptr(), n,
                                              s.data_ptr(), p.data_ptr(), torch.cuda.current_stream().cuda_stream))
        x = torch.from_numpy(x).to(self.type).double().numpy()
        self.held[seq] = np.concatenate([self.held[seq], x], 1)
        torch.cuda.synchronize()

    def decode(self, q, heads, pos):
        need = self.lib.axkv_decode_attn_workspace(C.byref(self.c), len(pos), heads)
        ws, out, p = torch.zeros(need, dtype=torch.uint8, device="cuda"), torch.empty_like(q), ints(pos)
        self.check(self.lib.axkv_paged_decode_attn(C.byref(self.c), q.data_ptr(), len(pos), heads, p.data_ptr(),
                                                   out.data_ptr(), ws.data_ptr(), need,
                                                   torch.cuda.current_stream().cuda_stream))
        return out.cpu().numpy()

    def row(self, q, out, heads, seq, n):
        for h in range(heads):
            k, v = (x[:n, h // (heads // self.kv)] for x in self.held[seq])
            qh, scale = q.reshape(heads, -1)[h].astype(np.float64), 1 / np.sqrt(self.hd)
            err = np.abs(out.reshape(heads, -1)[h] - km.attention(qh, k, v, scale)).max()
            assert err <= km.tolerance(qh, k, v, scale), (seq, h, err)


@pytest.mark.parametrize("hd,heads,kv,fp32", [(64, 8, 2, False), (128, 8, 8, False), (64, 9, 1, False),
                                              (32, 4, 2, True), (128, 4, 1, True)])
def test_attention_over_shared_and_moved_pages(hd, heads, kv, fp32):
    rng = np.random.default_rng(hd + heads)
    t = Cache(rng, kv, hd, fp32, 4, 6, 14)
    t.pages.reserve(ints([0, 3]), ints([40, 30]))
    t.append(0, 40)
    t.append(3, 30)
    t.pages.fork(ints([0, 0]), ints([1, 2]), ints([40, 20]))
    t.held[1], t.held[2] = t.held[0].copy(), t.held[0][:, :20].copy()
    t.pages.reserve(ints([0, 1, 2]), ints([52, 49, 21]))
    for seq, n in ((0, 12), (1, 9), (2, 1)):
        t.append(seq, n)
    for drop in (None, 3, 0):
        if drop is not None:
            t.pages.free(ints([drop]))
            t.held[drop] = t.held[drop][:, :0]
            live = int(t.pages.compact())
            assert int(t.pages.block_table.max()) < live
        q = rng.normal(0, 1, (4, heads * hd)).astype(np.float32)
        pos = [x.shape[1] - 1 for x in t.held]
        out = t.decode(dev(q), heads, pos)
        for s in range(4):
            if pos[s] >= 0:
                t.row(q[s], out[s], heads, s, pos[s] + 1)
    assert status() == 0
    if not fp32 and heads // kv <= 8:                  # rows at positions 16 .. 19 of every sequence
        q = rng.normal(0, 1, (16, heads * hd)).astype(np.float32)
        qd, out = dev(q), torch.empty(16, heads * hd, device="cuda")
        t.check(t.lib.axkv_paged_prefill_attn(C.byref(t.c), qd.data_ptr(), heads * hd, 4, 4, 16, heads, out.data_ptr(),
                                              None, None, torch.cuda.current_stream().cuda_stream))
        for s in (1, 2):
            for j in range(4):
                t.row(q[4 * s + j], out.cpu().numpy()[4 * s + j], heads, s, 17 + j)


@pytest.mark.parametrize("hd,heads,kv,fp32", [(64, 8, 2, False), (64, 9, 1, False), (64, 8, 2, True)])
def test_a_sequence_without_pages_does_not_reach_beyond_the_pool(hd, heads, kv, fp32):
    """A refused reserve leaves -1 in the table: appends report it, and attention over those
    positions stays inside the pool and leaves the other sequences as they are."""
    from axion_b200 import _lib, ops
    rng = np.random.default_rng(hd + heads)
    t = Cache(rng, kv, hd, fp32, 2, 4, 3)
    t.pages.reserve(ints([0]), ints([40]))
    t.append(0, 40)
    t.pages.reserve(ints([1]), ints([64]))
    assert status() == _lib.AXQ8_ERR_ALLOC
    ops.status_clear()
    before = t.k.clone(), t.v.clone()
    t.append(1, 50)
    assert status() == _lib.AXQ8_ERR_INVALID
    assert torch.equal(t.k, before[0]) and torch.equal(t.v, before[1])
    q = rng.normal(0, 1, (2, heads * hd)).astype(np.float32)
    for _ in range(2):
        out = t.decode(dev(q), heads, [39, 49])
        t.row(q[0], out[0], heads, 0, 40)
        t.pages.block_table[1] = 2 ** 31 - 1           # not a page either
