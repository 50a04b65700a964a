"""The 4-bit cache and the page table without a GPU: the format's own properties
(numpy model) and the refusals of every entry point, which come before any
device work."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import kv4_model as km


@pytest.fixture(scope="module")
def lib():
    from axion_b200 import _lib
    return _lib.load()


def test_every_stored_value_is_an_fp16_number():
    rng = np.random.default_rng(0)
    x = rng.normal(0, 1, (64, 128)) * np.exp2(rng.integers(-24, 16, (64, 1)))
    v = km.values(x.astype(np.float32))
    assert np.array_equal(v, v.astype(np.float16).astype(np.float64))


@pytest.mark.parametrize("scale", [2.0 ** -18, 1e-3, 1.0, 300.0])
def test_values_are_within_half_a_step(scale):
    """Away from the smallest steps a value is off by at most d / 2, and d is at most
    1 + 2^-6 times the range / 15 (7 significant bits; 2^-20 apart at the very bottom)."""
    rng = np.random.default_rng(1)
    x = rng.normal(0, scale, (256, 32)).astype(np.float32)
    d = (np.maximum(x.max(-1), 0) - np.minimum(x.min(-1), 0)).astype(np.float64) / 15
    limit = (d * (1 + 2.0 ** -6) + 2.0 ** -20)[:, None] / 2 * (1 + 2.0 ** -20)
    assert np.all(np.abs(km.values(x) - x) <= limit)


def test_extreme_blocks():
    x = np.zeros((5, 32), np.float32)
    x[1] = 7.0                                # one sign: zero is still in the range
    x[2, 3] = np.nan
    x[2, 4] = 1.5
    x[3, 0], x[3, 1] = np.inf, -np.inf
    x[4] = 1e-30
    v = km.values(x)
    assert np.all(v[0] == 0) and np.all(v[2, :3] == 0) and v[2, 3] == 0
    assert np.all(np.abs(v[1] - 7) <= 0.3)
    assert abs(v[3, 0] - km.LIMIT) < 2300 and abs(v[3, 1] + km.LIMIT) < 2300
    assert np.all(v[4] == 0)


def test_layout_covers_every_byte_once():
    """Writing every token fills all bytes, and each token only its own."""
    for hd in (32, 64, 128):
        rng = np.random.default_rng(hd)
        k, v = rng.normal(0, 1, (2, 16, hd)).astype(np.float32)
        full = np.full(18 * hd, 255, np.uint8)
        for t in range(16):
            km.write_token(full, t, k[t], v[t])
        again = np.zeros(18 * hd, np.uint8)
        for t in rng.permutation(16):
            km.write_token(again, t, k[t], v[t])
        assert np.array_equal(full, again)


def _cache(_lib, **kw):
    f = dict(pages=4096, block_table=4096, n_seqs=2, max_blocks=4, n_pages=8, n_kv_heads=2,
             head_dim=64, page_tokens=16)
    f.update(kw)
    return _lib.axkv4_cache_t(*[f[n] for n, _ in _lib.axkv4_cache_t._fields_])


@pytest.mark.parametrize("field,value,code", [
    ("pages", 0, "INVALID"), ("block_table", 0, "INVALID"), ("pages", 4104, "INVALID"),
    ("n_seqs", 0, "INVALID"), ("max_blocks", 0, "INVALID"), ("n_pages", -1, "INVALID"),
    ("n_kv_heads", 0, "INVALID"), ("head_dim", 96, "UNSUPPORTED"), ("head_dim", 0, "UNSUPPORTED"),
    ("page_tokens", 32, "UNSUPPORTED"), ("max_blocks", 1 << 27, "UNSUPPORTED")])
def test_cache_refusals(lib, field, value, code):
    from axion_b200 import _lib
    c = C.byref(_cache(_lib, **{field: value}))
    want = getattr(_lib, "AXQ8_ERR_" + code)
    p = 4096
    assert lib.axkv4_append(c, p, p, 128, 1, p, p, None) == want
    assert lib.axkv4_read(c, p, p, 128, 1, p, p, None) == want
    assert lib.axkv4_decode_attn(c, p, 256, 1, 4, None, p, p, p, 1 << 20, None) == want
    assert lib.axkv4_chunk_attn(c, p, 256, 1, 1, 1, 4, None, p, p, p, p, 1 << 20, None) == want
    assert lib.axkv4_decode_attn_workspace(c, 1, 4) == -1
    assert lib.axkv4_chunk_attn_workspace(c, 1, 1, 4) == -1


def test_row_refusals(lib):
    from axion_b200 import _lib
    c, p, bad = C.byref(_cache(_lib)), 4096, _lib.AXQ8_ERR_INVALID
    for fn in (lib.axkv4_append, lib.axkv4_read):
        assert fn(c, p, p, 128, 0, None, None, None) == 0            # nothing to do
        assert fn(c, p, p, 128, -1, p, p, None) == bad
        assert fn(c, None, p, 128, 1, p, p, None) == bad
        assert fn(c, p, p, 128, 1, None, p, None) == bad
        assert fn(c, p, p, 124, 1, p, p, None) == bad                # rows overlap
        assert fn(c, p, p, 130, 1, p, p, None) == bad                # not a multiple of 4
        assert fn(c, p + 4, p, 128, 1, p, p, None) == bad            # alignment
    assert lib.axkv4_append(None, p, p, 128, 1, p, p, None) == bad


def test_attention_refusals(lib):
    from axion_b200 import _lib
    c, p, bad = C.byref(_cache(_lib)), 4096, _lib.AXQ8_ERR_INVALID

    def decode(q=p, ldq=256, n=2, heads=4, seq=None, pos=p, out=p, ws=p, size=1 << 24):
        return lib.axkv4_decode_attn(c, q, ldq, n, heads, seq, pos, out, ws, size, None)

    def chunk(q=p, ldq=256, n=2, chunks=2, rows=3, heads=4, seq=None, start=p, pos=p, out=p, ws=p,
              size=1 << 24):
        return lib.axkv4_chunk_attn(c, q, ldq, n, chunks, rows, heads, seq, start, pos, out, ws, size, None)

    for fn in (decode, chunk):
        for kw in (dict(heads=3), dict(heads=0), dict(heads=34, ldq=4096), dict(n=-1), dict(q=None),
                   dict(pos=None), dict(out=None), dict(ws=None), dict(q=p + 4), dict(out=p + 8),
                   dict(ws=p + 4), dict(ldq=252), dict(ldq=258), dict(size=0)):
            assert fn(**kw) == bad, (fn.__name__, kw)
        assert fn(n=0) == 0
    assert decode(n=3) == bad                  # three rows, two sequences, no q_seq
    assert chunk(chunks=3) == bad
    assert chunk(rows=-1) == bad and chunk(chunks=-1) == bad and chunk(start=None) == bad
    assert chunk(rows=0) == 0 and chunk(chunks=0) == 0
    assert lib.axkv4_decode_attn_workspace(c, 0, 4) == -1
    assert lib.axkv4_chunk_attn_workspace(c, 1, 0, 4) == -1


def test_page_refusals(lib):
    from axion_b200 import _lib
    p, bad = 4096, _lib.AXQ8_ERR_INVALID

    def pages(**kw):
        f = dict(block_table=p, ref_count=p, pools=p, page_bytes=1024, n_pools=2, n_seqs=4, max_blocks=4,
                 n_pages=16)
        f.update(kw)
        return C.byref(_lib.axkv_pages_t(*[f[n] for n, _ in _lib.axkv_pages_t._fields_]))

    def calls(c, n=1, a=p, ws=p, size=1 << 20):
        return [lib.axkv_pages_reserve(c, a, p, n, ws, size, None),
                lib.axkv_pages_fork(c, a, p, p, n, ws, size, None),
                lib.axkv_pages_compact(c, a, ws, size, None),
                lib.axkv_pages_free(c, a, n, None), lib.axkv_pages_copy(c, a, p, n, None)]

    for kw in (dict(block_table=0), dict(ref_count=0), dict(pools=0), dict(page_bytes=0),
               dict(page_bytes=1000), dict(n_pools=-1), dict(n_seqs=0), dict(max_blocks=0),
               dict(n_pages=0)):
        assert calls(pages(**kw)) == [bad] * 5, kw
        assert lib.axkv_pages_workspace(pages(**kw), 1) == -1
    for kw in (dict(max_blocks=1 << 27), dict(n_pages=2000001)):
        assert calls(pages(**kw)) == [_lib.AXQ8_ERR_UNSUPPORTED] * 5, kw
    assert calls(pages(), a=None) == [bad] * 5
    assert calls(pages(), size=16)[:3] == [bad] * 3 and calls(pages(), ws=None)[:3] == [bad] * 3
    c = calls(pages(), n=-1)
    assert c[:2] == [bad] * 2 and c[3:] == [bad] * 2
    assert lib.axkv_pages_reserve(pages(), None, None, 0, None, 0, None) == 0
    assert lib.axkv_pages_free(pages(), None, 0, None) == 0
    assert lib.axkv_pages_workspace(pages(), 4) > 0


def test_python_classes_refuse_what_is_not_on_a_gpu():
    import torch
    from axion_b200.kv_pages import KVPages
    from axion_b200.paged_kv import PagedKVCache4
    table = torch.zeros(1, 4, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        PagedKVCache4(2, 64, pages=torch.zeros(4, 2, 18 * 64, dtype=torch.uint8), block_table=table)
    with pytest.raises(RuntimeError, match="CUDA"):
        KVPages([torch.zeros(4, 16)], table, torch.zeros(4, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="head_dim"):
        PagedKVCache4(2, 96)
    with pytest.raises(RuntimeError, match="come together"):
        PagedKVCache4(2, 64, block_table=table)
