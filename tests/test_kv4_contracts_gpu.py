"""What include/axkv.h promises of calls that are refused or leave rows out: nothing else is
touched, and the rest of the call is done."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest
import torch

from test_kv4_gpu import Case, check_rows, clean_status, dev, ints, run_chunks, status  # noqa: F401
from test_kv_pages_gpu import make, same

pytestmark = pytest.mark.gpu


def test_refused_reserves_and_forks_leave_every_page():
    from axion_b200 import _lib, ops
    model, pages = make(6, 4, 12, words=700)
    model.reserve([0, 1], [40, 64])
    pages.reserve(ints([0, 1]), ints([40, 64]))
    invalid, alloc = _lib.AXQ8_ERR_INVALID, _lib.AXQ8_ERR_ALLOC
    refused = [("reserve", ([2, 2], [16, 16]), invalid), ("reserve", ([0, 9], [64, 1]), invalid),
               ("reserve", ([2, 3], [64, 32]), alloc), ("fork", ([0], [1], [16]), invalid),
               ("fork", ([0, 0], [2, 2], [17, 17]), invalid), ("fork", ([0, 2], [2, 3], [17, 0]), invalid),
               ("fork", ([0, 7], [2, 3], [40, 1]), invalid), ("fork", ([0], [2], [49]), invalid)]
    for call, args, code in refused:
        before = [p.clone() for p in pages.pools]
        ops.status_clear()
        getattr(pages, call)(*(ints(a) for a in args))
        assert status() == code, (call, args)
        same(model, pages)
        assert all(torch.equal(a, b) for a, b in zip(before, pages.pools)), (call, args)
    ops.status_clear()
    before = [p.clone() for p in pages.pools]
    copies = model.fork([0, 0, 0, 1], [2, 3, 4, 5], [40, 39, 1, 64])
    pages.fork(ints([0, 0, 0, 1]), ints([2, 3, 4, 5]), ints([40, 39, 1, 64]))
    for w in before:
        for s, d in copies:
            w[d] = w[s]
    same(model, pages)
    assert all(torch.equal(a, b) for a, b in zip(before, pages.pools)) and status() == 0


@pytest.mark.parametrize("heads,kv,scale", [(4, 2, 1), (14, 2, 1), (32, 8, 40)])
def test_chunks_that_are_left_out_leave_their_rows(heads, kv, scale):
    """Starts outside the rows, a chunk of too many rows, starts that fall: rows of such chunks stay,
    their neighbours are right.  With 40 times the rows, in the tiles of long chunks."""
    from axion_b200 import _lib, ops
    hd, k = 64, scale
    rng = np.random.default_rng(heads)
    case = Case(rng, kv, hd, (20 + 10 * k, 20 + 10 * k))
    q = rng.normal(0, 1, (8 * k, heads * hd)).astype(np.float32)
    # starts, most rows, the chunk that is done and its rows
    for start, most, done, a, b in (([0, 4 * k, 8 * k + 1], 8 * k, 0, 0, 4 * k), ([-1, 4 * k, 8 * k], 8 * k, 1, 4 * k, 8 * k),
                                    ([0, 6 * k, 8 * k], 5 * k, 1, 6 * k, 8 * k), ([4 * k, 2 * k, 8 * k], 8 * k, 1, 2 * k, 8 * k)):
        ops.status_clear()
        out = torch.full((8 * k, heads * hd), 7.0, device="cuda")
        case.cache.chunk_attention(dev(q), heads, ints(start), ints([10, 12]), most, out=out)
        assert status() == (0 if start[1] < start[0] else _lib.AXQ8_ERR_INVALID), start
        out = out.cpu().numpy()
        rest = np.ones(8 * k, bool)
        rest[a:b] = False
        assert (out[rest] == 7.0).all(), start
        pick = sorted({a, a + 1, (a + b) // 2, b - 1})
        check_rows(case, q[pick], out[pick], heads, [done] * len(pick), [(10, 12)[done] + r - a + 1 for r in pick])


@pytest.mark.parametrize("heads,kv,rows", [(8, 2, 1), (16, 1, 3), (32, 8, 300)])
def test_a_workspace_of_any_contents_and_one_too_small(heads, kv, rows):
    """All ones before each call; a byte less than asked for is refused."""
    from axion_b200 import _lib
    lib, hd = _lib.load(), 128
    rng = np.random.default_rng(rows)
    case = Case(rng, kv, hd, (1000 + rows, 30 + rows))
    c, n = C.byref(case.cache.c), 2 * rows
    q = rng.normal(0, 1, (n, heads * hd)).astype(np.float32)
    qd, out, start = dev(q), torch.empty(n, heads * hd, device="cuda"), ints([0, rows, n])
    seq, pos = ints([0, 1]), ints([1000, 30])
    calls = [(lib.axkv4_chunk_attn_workspace(c, 2, rows, heads),
              lambda ws, size: lib.axkv4_chunk_attn(c, qd.data_ptr(), heads * hd, n, 2, rows, heads, seq.data_ptr(),
                                                    start.data_ptr(), pos.data_ptr(), out.data_ptr(), ws, size, None))]
    if rows == 1:
        calls.append((lib.axkv4_decode_attn_workspace(c, 2, heads),
                      lambda ws, size: lib.axkv4_decode_attn(c, qd.data_ptr(), heads * hd, 2, heads, seq.data_ptr(),
                                                             pos.data_ptr(), out.data_ptr(), ws, size, None)))
    for need, call in calls:
        ws = torch.empty(need, dtype=torch.uint8, device="cuda")
        for _ in range(2):
            ws.fill_(255)
            out.fill_(7)
            torch.cuda.synchronize()
            assert call(ws.data_ptr(), need) == 0
            torch.cuda.synchronize()
            for s in range(2):
                pick = sorted({0, rows // 2, rows - 1})
                at = [s * rows + r for r in pick]
                check_rows(case, q[at], out.cpu().numpy()[at], heads, [s] * len(pick), [(1001, 31)[s] + r for r in pick])
        if need > 16:                                       # the long chunks' kernel uses none
            assert call(ws.data_ptr(), need - 1) == _lib.AXQ8_ERR_INVALID
    assert status() == 0


@pytest.mark.parametrize("heads,kv,rows", [(8, 2, 1), (16, 1, 5), (32, 8, 300)])
def test_the_result_may_take_the_queries_place(heads, kv, rows):
    rng = np.random.default_rng(rows + 1)
    case = Case(rng, kv, 128, (5000 + rows, 70 + rows))
    q = dev(rng.normal(0, 1, (2 * rows, heads * 128)).astype(np.float32))
    args = (heads, ints([0, rows, 2 * rows]), ints([5000, 70]), rows)
    want = case.cache.chunk_attention(q, *args)
    x = q.clone()
    assert torch.equal(case.cache.chunk_attention(x, *args, out=x), want)
    if rows == 1:
        want = case.cache.decode_attention(q, heads, ints([5000, 70]))
        x = q.clone()
        assert torch.equal(case.cache.decode_attention(x, heads, ints([5000, 70]), out=x), want)
