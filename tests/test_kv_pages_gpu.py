"""Page-table operators (include/axkv.h, axkv_pages) against Python lists, and a run of them
with the 4-bit cache as a serving loop uses them."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kv4_model as km
from test_kv4_gpu import ints

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def clean_status(cuda):
    from axion_b200 import ops
    ops.status_clear()
    yield
    ops.status_clear()


def status():
    from axion_b200 import ops
    return ops.status()


def make(n_seqs, max_blocks, n_pages, pools=2, words=8):
    """A model, the table on the GPU, and pools whose pages hold random 16-byte words."""
    from axion_b200.kv_pages import KVPages
    data = [torch.randint(0, 2 ** 31 - 1, (n_pages, words, 4), dtype=torch.int32, device="cuda")
            for _ in range(pools)]
    return km.Table(n_seqs, max_blocks, n_pages), KVPages.empty(data, n_seqs, max_blocks)


def same(model, pages):
    assert np.array_equal(pages.block_table.cpu().numpy(), model.array())
    assert np.array_equal(pages.ref_count.cpu().numpy(), model.counts())


@pytest.mark.parametrize("n_seqs,max_blocks,n_pages,words", [
    (1, 1, 1, 1), (5, 3, 9, 3), (40, 7, 200, 8), (6, 200, 1100, 513), (2100, 2, 5000, 1),
    (8, 1500, 9000, 2)])
def test_random_calls(n_seqs, max_blocks, n_pages, words):
    """Reserves, forks, frees and compactions in random order, refused ones among them: table,
    counts and page contents follow the model after each."""
    from axion_b200 import _lib, ops
    rng = np.random.default_rng(n_seqs + n_pages)
    model, pages = make(n_seqs, max_blocks, n_pages, words=words)
    for step in range(24):
        want = [p.clone() for p in pages.pools]
        op = rng.choice(["reserve", "reserve", "fork", "fork", "free", "compact"])
        n = int(rng.integers(1, min(n_seqs, 1500) + 1))
        ops.status_clear()
        expect = 0
        if op == "reserve":
            seqs = [int(x) for x in rng.permutation(n_seqs)[:n]]
            tokens = [int(x) for x in rng.integers(0, 16 * max_blocks + 1, n) // int(rng.integers(1, 5))]
            free, need = len(model._free()), model.array()
            if model.reserve(seqs, tokens) is None:
                expect = _lib.AXQ8_ERR_ALLOC
            pages.reserve(ints(seqs), ints(tokens))
        elif op == "fork":
            live = [i for i in range(n_seqs) if model.rows[i]]
            empty = [i for i in range(n_seqs) if not model.rows[i]][:n]
            if not live or not empty:
                continue
            parents = [int(rng.choice(live)) for _ in empty]
            tokens = [int(rng.integers(0, 16 * len(model.rows[p]) + 1)) for p in parents]
            copies = model.fork(parents, empty, tokens)
            pages.fork(ints(parents), ints(empty), ints(tokens))
            if copies is None:
                expect = _lib.AXQ8_ERR_ALLOC
            for w in want:
                for s, d in copies or []:
                    w[d] = w[s]
        elif op == "free":
            seqs = [int(x) for x in rng.integers(0, n_seqs, max(1, n // 3))]       # some twice
            model.free(seqs)
            pages.free(ints(seqs))
        else:
            live, moves = model.compact()
            assert int(pages.compact()) == live
            for w in want:
                if moves:
                    s, d = (torch.tensor(x, device="cuda") for x in zip(*moves))
                    w[d] = w[s]
        assert status() == expect, (step, op)
        same(model, pages)
        for a, b in zip(pages.pools, want):
            assert torch.equal(a, b), (step, op)


def test_refused_calls_change_nothing():
    from axion_b200 import _lib, ops
    model, pages = make(6, 4, 12)
    model.reserve([0, 1], [40, 64])
    pages.reserve(ints([0, 1]), ints([40, 64]))
    same(model, pages)
    before = [p.clone() for p in pages.pools]
    invalid, alloc = _lib.AXQ8_ERR_INVALID, _lib.AXQ8_ERR_ALLOC
    for seqs, tokens, code in (([2, 2], [16, 16], invalid), ([6], [1], invalid), ([-1], [1], invalid),
                               ([2], [65], invalid), ([2], [-1], invalid), ([2, 3], [64, 32], alloc),
                               ([0, 9], [64, 1], invalid)):
        ops.status_clear()
        pages.reserve(ints(seqs), ints(tokens))
        assert status() == code, (seqs, tokens)
        same(model, pages)
    for par, kid, tokens, code in (([0], [1], [16], invalid),            # the child holds pages
                                   ([0, 0], [2, 2], [16, 16], invalid),  # a child twice
                                   ([0, 2], [2, 3], [16, 0], invalid),   # a child that is a parent
                                   ([0], [0], [16], invalid), ([0], [6], [1], invalid),
                                   ([7], [2], [1], invalid), ([0], [2], [49], invalid),
                                   ([0], [2], [-3], invalid), ([4], [2], [1], invalid),
                                   ([0, 1, 0, 1], [2, 3, 4, 5], [1, 17, 33, 49], 0)):
        ops.status_clear()
        if code == 0:
            model.fork(par, kid, tokens)
        pages.fork(ints(par), ints(kid), ints(tokens))
        assert status() == code, (par, kid, tokens)
        same(model, pages)
    ops.status_clear()
    pages.free(ints([5]))
    model.free([5])
    pages.reserve(ints([5]), ints([64]))      # more than the freed and the spare pages
    assert status() == alloc
    same(model, pages)
    ops.status_clear()
    pages.free(ints([1, 17, -2, 1]))
    model.free([1])
    assert status() == invalid
    same(model, pages)
    assert before[0].shape == pages.pools[0].shape


def test_fork_without_room_changes_nothing():
    from axion_b200 import _lib
    model, pages = make(5, 3, 4)
    model.reserve([0], [40])
    pages.reserve(ints([0]), ints([40]))
    before = [p.clone() for p in pages.pools]
    pages.fork(ints([0, 0]), ints([1, 2]), ints([40, 33]))       # two copies, one free page
    assert status() == _lib.AXQ8_ERR_ALLOC
    same(model, pages)
    assert all(torch.equal(a, b) for a, b in zip(before, pages.pools))


@pytest.mark.parametrize("words", [1, 511, 512, 1025])
def test_copy(words):
    from axion_b200 import _lib
    _, pages = make(1, 1, 50, pools=3, words=words)
    want = [p.clone() for p in pages.pools]
    src, dst = [3, 3, 40, 49], [0, 7, 12, 1]
    for w in want:
        for s, d in zip(src, dst):
            w[d] = w[s]
    pages.copy(ints(src), ints(dst))
    assert all(torch.equal(a, b) for a, b in zip(want, pages.pools)) and status() == 0
    pages.copy(ints([50, -1, 2]), ints([4, 5, 50]))
    assert all(torch.equal(a, b) for a, b in zip(want, pages.pools))
    assert status() == _lib.AXQ8_ERR_INVALID


def test_pools_past_32_bits():
    """Pools of more than 4 GiB: pages from the end are copied and moved to the front."""
    from axion_b200.kv_pages import KVPages
    n = 70000
    pool = torch.empty(n, 65536, dtype=torch.uint8, device="cuda")
    pool[n - 3:] = torch.arange(3, dtype=torch.uint8, device="cuda")[:, None] + 5
    table = torch.full((2, 4), -1, dtype=torch.int32, device="cuda")
    table[0, :3] = ints([n - 1, n - 3, n - 2])
    ref = torch.zeros(n, dtype=torch.int32, device="cuda")
    ref[n - 3:] = 1
    pages = KVPages([pool], table, ref)
    pages.fork(ints([0]), ints([1]), ints([40]))                 # copies page n - 2 to page 0
    assert int(pages.compact()) == 4
    assert table.tolist() == [[3, 1, 2, -1], [3, 1, 0, -1]]
    assert ref[:5].tolist() == [1, 2, 1, 2, 0]
    assert [int(pool[i].min()) for i in range(4)] == [6, 5, 6, 7]
    assert [int(pool[i].max()) for i in range(4)] == [6, 5, 6, 7] and status() == 0


def test_refusals_of_the_class():
    from axion_b200.kv_pages import KVPages
    _, pages = make(2, 2, 4)
    with pytest.raises(RuntimeError):
        pages.free(torch.zeros(1, dtype=torch.int64, device="cuda"))
    with pytest.raises(RuntimeError):
        pages.fork(ints([0]), ints([1]), ints([1, 2]))
    with pytest.raises(RuntimeError):
        KVPages([torch.zeros(3, 16, device="cuda")], pages.block_table, pages.ref_count)
    with pytest.raises(RuntimeError):
        KVPages([torch.zeros(4, 3, device="cuda")], pages.block_table, pages.ref_count)


@pytest.mark.parametrize("hd,heads,kv", [(64, 8, 2), (128, 8, 4)])
def test_serving_run(hd, heads, kv):
    """Two layers: a prompt, two samples forked from it, tokens appended to each, one dropped, the
    pools compacted, another prompt in the freed pages - every attention against 64 bits."""
    from axion_b200.kv_pages import KVPages
    from axion_b200.paged_kv import PagedKVCache4
    rng = np.random.default_rng(hd)
    pools = [torch.full((24, kv, 18 * hd), 255, dtype=torch.uint8, device="cuda") for _ in range(2)]
    pages = KVPages.empty(pools, 4, 12)
    layers = [PagedKVCache4(kv, hd, pages=p, block_table=pages.block_table) for p in pools]
    hist = [[(np.zeros((0, kv, hd), np.float32),) * 2 for _ in range(4)] for _ in layers]
    scale = 1 / np.sqrt(hd)

    def step(seqs, n):
        """n tokens appended to each sequence, and their attention, in every layer."""
        rows = len(seqs) * n
        first = [len(hist[0][s][0]) for s in seqs]
        pages.reserve(ints(seqs), ints(f + n for f in first))
        seq, pos = ints(s for s in seqs for _ in range(n)), ints(f + j for f in first for j in range(n))
        for layer, h in zip(layers, hist):
            k, v, q = (rng.normal(0, 1, (rows, w)).astype(np.float32) for w in (kv * hd, kv * hd, heads * hd))
            layer.append_rows(torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), seq, pos)
            for i, s in enumerate(seqs):
                at = slice(i * n, i * n + n)
                h[s] = tuple(np.concatenate([a, x[at].reshape(n, kv, hd)]) for a, x in zip(h[s], (k, v)))
            qd = torch.from_numpy(q).cuda()
            if n == 1:
                out = layer.decode_attention(qd, heads, ints(first), ints(seqs))
            else:
                out = layer.chunk_attention(qd, heads, ints(range(0, rows + 1, n)), ints(first), n, ints(seqs))
            out = out.cpu().numpy()
            for i, s in enumerate(seqs):
                kk, vv = (km.values(x) for x in h[s])
                for j in range(n):
                    for hh in range(heads):
                        m, g = first[i] + j + 1, hh // (heads // kv)
                        qh = q[i * n + j].reshape(heads, hd)[hh].astype(np.float64)
                        ref = km.attention(qh, kk[:m, g], vv[:m, g], scale)
                        tol = km.tolerance(qh, kk[:m, g], vv[:m, g], scale)
                        assert np.abs(out[i * n + j].reshape(heads, hd)[hh] - ref).max() <= tol

    step([0], 75)
    pages.fork(ints([0, 0]), ints([1, 2]), ints([75, 70]))
    for h in hist:
        h[1], h[2] = tuple(x.copy() for x in h[0]), tuple(x[:70].copy() for x in h[0])
    for _ in range(9):
        step([0, 1, 2], 1)
    pages.free(ints([0]))
    for h in hist:
        h[0] = (np.zeros((0, kv, hd), np.float32),) * 2
    live = int(pages.compact())
    assert live == 4 + 2 + 1                 # 84 and 79 tokens: four shared full pages, two and one of their own
    assert int(pages.block_table.max()) < live
    step([1, 2], 1)
    step([3], 40)
    step([3, 1, 2], 4)
    step([2, 3], 1)
    assert status() == 0
