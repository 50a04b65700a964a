"""The 4-bit paged KV cache on the GPU against the 64-bit model of its format."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest
import torch

import kv4_model as km

pytestmark = pytest.mark.gpu


def dev(a, dtype=None):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda() if dtype is None \
        else torch.tensor(a, dtype=dtype, device="cuda")


def ints(a):
    return torch.tensor([int(x) for x in a], dtype=torch.int32, device="cuda")


class Case:
    """A cache of sequences of given lengths over shuffled pages; slots past a
    sequence's end and the spare pages are all ones (scales that read as NaN)."""

    def __init__(self, rng, kv, hd, lens, spare=3, max_blocks=None, scale=1.0):
        from axion_b200.paged_kv import PagedKVCache4
        self.kv, self.hd, self.lens = kv, hd, list(lens)
        blocks = [-(-n // 16) for n in lens]
        n_pages = sum(blocks) + spare
        order = rng.permutation(n_pages).astype(np.int32)
        self.table = np.full((len(lens), max_blocks or max(max(blocks), 1)), -1, np.int32)
        at = 0
        for s, b in enumerate(blocks):
            self.table[s, :b] = order[at:at + b]
            at += b
        self.k = [(rng.normal(0, scale, (n, kv, hd))).astype(np.float32) for n in lens]
        self.v = [rng.normal(0, 1, (n, kv, hd)).astype(np.float32) for n in lens]
        self.pages = torch.full((n_pages, kv, 18 * hd), 255, dtype=torch.uint8, device="cuda")
        self.cache = PagedKVCache4(kv, hd, pages=self.pages, block_table=dev(self.table))
        self.append(0, None)

    def append(self, a, b):
        """Positions a .. b - 1 of every sequence that has them, rows in shuffled order."""
        seq, pos = [], []
        for s, n in enumerate(self.lens):
            for p in range(a, n if b is None else min(n, b)):
                seq.append(s)
                pos.append(p)
        if not seq:
            return
        mix = np.random.default_rng(3).permutation(len(seq))
        seq, pos = np.array(seq)[mix], np.array(pos)[mix]
        k, v = (np.stack([x[s][p] for s, p in zip(seq, pos)]).reshape(len(seq), -1) for x in (self.k, self.v))
        self.cache.append_rows(dev(k), dev(v), ints(seq), ints(pos))

    def held(self, s, n, head):
        """The first n tokens' K and V of a kv head in 64 bits."""
        return km.values(self.k[s][:n, head]), km.values(self.v[s][:n, head])


def check_rows(case, q, out, heads, seqs, ctx):
    """Row r of q and out is sequence seqs[r] over ctx[r] tokens."""
    scale = 1 / np.sqrt(case.hd)
    worst = 0.0
    held = {}
    for r, (s, n) in enumerate(zip(seqs, ctx)):
        for h in range(heads):
            kvh = h // (heads // case.kv)
            if (s, kvh) not in held:
                held[s, kvh] = case.held(s, case.lens[s], kvh)
            k, v = (x[:max(n, 0)] for x in held[s, kvh])
            qh = q[r].reshape(heads, -1)[h].astype(np.float64)
            ref, got = km.attention(qh, k, v, scale), out[r].reshape(heads, -1)[h]
            tol = km.tolerance(qh, k, v, scale)
            err = np.abs(got - ref).max()
            assert err <= tol, (r, h, n, err, tol)
            worst = max(worst, err / tol if tol else 0.0)
    return worst


@pytest.fixture(autouse=True)
def clean_status(cuda):
    from axion_b200 import ops
    ops.status_clear()
    yield
    ops.status_clear()


def status():
    from axion_b200 import ops
    return ops.status()


# ---- append and read ---------------------------------------------------------------

@pytest.mark.parametrize("hd,kv", [(32, 1), (32, 5), (64, 3), (128, 1), (128, 8)])
@pytest.mark.parametrize("lens", [(1,), (16, 17), (37, 5, 64)])
def test_append_stores_the_format_bit_for_bit(hd, kv, lens):
    rng = np.random.default_rng(hd + kv + lens[0])
    case = Case(rng, kv, hd, lens)
    want = np.full(tuple(case.pages.shape), 255, np.uint8)
    for s, n in enumerate(lens):
        for p in range(n):
            for h in range(kv):
                km.write_token(want[case.table[s, p // 16], h], p % 16, case.k[s][p, h], case.v[s][p, h])
    assert np.array_equal(case.pages.cpu().numpy(), want)
    for s, n in enumerate(lens):
        k, v = case.cache.read_rows(ints([s] * n), ints(range(n)))
        assert np.array_equal(k.cpu().numpy(), km.values(case.k[s]).reshape(n, -1))
        assert np.array_equal(v.cpu().numpy(), km.values(case.v[s]).reshape(n, -1))
    assert status() == 0


@pytest.mark.parametrize("hd", [32, 64, 128])
def test_append_at_the_borders_of_the_format(hd):
    """Ties of the rounding, exact multiples of 15 steps, zeros, tiny and large values."""
    from axion_b200.paged_kv import PagedKVCache4
    rng = np.random.default_rng(hd)
    n = 64
    x = rng.normal(0, 1, (n, hd)).astype(np.float32) * np.exp2(rng.integers(-22, 13, (n, 1))).astype(np.float32)
    x[0] = 0
    x[1] = 7.5
    x[2] = -3.25
    step = np.float32(0.203125)               # 13 / 64
    x[3] = step * (rng.integers(-14, 16, hd) / 2).astype(np.float32)
    x[3, :2] = step * 7.5, -step * 7.5        # range 15 steps: every half step is a tie
    x[4] = np.nextafter(x[3], np.float32(np.inf))
    x[5] = np.nextafter(x[3], np.float32(-np.inf))
    x[6] = 1e-38
    x[7] = np.float32(2.0 ** -20) * rng.integers(-7, 8, hd)
    kv = PagedKVCache4(1, hd, max_seqs=1, max_tokens=n)
    kv.append(dev(x), dev(x[::-1].copy()))
    assert np.array_equal(kv.materialize_keys().cpu().numpy(), km.values(x))
    assert np.array_equal(kv.materialize_values().cpu().numpy(), km.values(x[::-1]))
    assert status() == 0


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf, 1e6, -40000.0])
def test_append_reports_what_it_cannot_hold(value):
    from axion_b200 import _lib
    from axion_b200.paged_kv import PagedKVCache4
    x = np.random.default_rng(0).normal(0, 1, (3, 64)).astype(np.float32)
    x[1, 40] = value
    kv = PagedKVCache4(1, 64, max_tokens=16)
    kv.append(dev(x), dev(np.zeros_like(x)))
    assert status() == _lib.AXQ8_ERR_INVALID
    assert np.array_equal(kv.materialize_keys().cpu().numpy(), km.values(x))


def test_append_from_a_slice_of_wider_rows():
    """K and V as columns of the Q|K|V rows (16-byte aligned), and as unaligned ones."""
    from axion_b200.paged_kv import PagedKVCache4
    rng = np.random.default_rng(5)
    for off in (256, 257):
        qkv = dev(rng.normal(0, 1, (9, 600)).astype(np.float32))
        kv = PagedKVCache4(2, 64, max_tokens=16)
        k, v = qkv[:, off:off + 128], qkv[:, off + 128:off + 256]
        kv.append(k, v)
        assert np.array_equal(kv.materialize_keys().cpu().numpy(), km.values(k.cpu().numpy().reshape(9, 2, 64)).reshape(9, -1))
        assert np.array_equal(kv.materialize_values().cpu().numpy(), km.values(v.cpu().numpy().reshape(9, 2, 64)).reshape(9, -1))


def test_positions_outside_the_table_are_left_out_and_reported():
    from axion_b200 import _lib, ops
    rng = np.random.default_rng(6)
    case = Case(rng, 2, 64, (20, 20), max_blocks=3)
    before = case.pages.clone()
    row = torch.ones(1, 128, device="cuda")
    bad = [(0, 48), (0, -1), (2, 0), (-1, 0), (1, 40), (0, 2 ** 31 - 1)]   # (1, 40): no page there
    for s, p in bad:
        ops.status_clear()
        case.cache.append_rows(row, row, ints([s]), ints([p]))
        assert status() == _lib.AXQ8_ERR_INVALID, (s, p)
        ops.status_clear()
        k, v = case.cache.read_rows(ints([s]), ints([p]))
        assert status() == _lib.AXQ8_ERR_INVALID, (s, p)
        assert not k.any() and not v.any()
    case.cache.block_table[1, 2] = case.pages.shape[0]      # a page past the pool
    ops.status_clear()
    case.cache.append_rows(row, row, ints([1]), ints([33]))
    assert status() == _lib.AXQ8_ERR_INVALID
    assert torch.equal(case.pages, before)


# ---- one row per sequence ------------------------------------------------------------

SHAPES = [(32, 1, 1), (32, 8, 2), (64, 4, 4), (64, 14, 2), (64, 8, 1), (64, 32, 2), (128, 1, 1),
          (128, 16, 4), (128, 6, 2), (128, 9, 1), (128, 32, 2)]


@pytest.mark.parametrize("hd,heads,kv", SHAPES)
@pytest.mark.parametrize("lens", [(1,), (15, 16, 17, 31, 33), (700, 2, 129)])
def test_decode_attention(hd, heads, kv, lens):
    rng = np.random.default_rng(hd * heads + len(lens))
    case = Case(rng, kv, hd, lens, scale=1.5)
    q = rng.normal(0, 1, (len(lens), heads * hd)).astype(np.float32)
    args = (dev(q), heads, ints(n - 1 for n in lens))
    out = case.cache.decode_attention(*args)
    check_rows(case, q, out.cpu().numpy(), heads, range(len(lens)), lens)
    assert torch.equal(out, case.cache.decode_attention(*args))     # bit for bit, workspace reused
    assert status() == 0


def test_decode_rows_of_chosen_sequences_and_positions():
    """Sequences in another order, twice, at earlier positions; empty and padded rows."""
    rng = np.random.default_rng(11)
    case = Case(rng, 2, 128, (90, 40, 300))
    seqs, ctx = [2, 0, 2, 1, 0, 1, 2], [300, 90, 17, 1, 0, 40, -5]
    wide = torch.zeros(7, 8 * 128 + 4, device="cuda")
    q = rng.normal(0, 1, (7, 8 * 128)).astype(np.float32)
    wide[:, :8 * 128] = dev(q)
    out = torch.full((7, 8 * 128), 7.0, device="cuda")
    got = case.cache.decode_attention(wide[:, :8 * 128], 8, ints(n - 1 for n in ctx), ints(seqs), out=out)
    assert got is out
    check_rows(case, q, out.cpu().numpy(), 8, seqs, ctx)
    assert not out[4].any() and not out[6].any() and status() == 0


@pytest.mark.parametrize("hd,heads,kv,rows", [(128, 8, 2, 300), (64, 14, 2, 129), (128, 32, 2, 140), (64, 4, 4, 128)])
def test_decode_of_many_rows(hd, heads, kv, rows):
    """More tiles than CTAs: runs that end inside tiles, several tiles to a run, more entries than
    are kept in shared memory; empty rows among them."""
    rng = np.random.default_rng(rows)
    case = Case(rng, kv, hd, (700, 2, 129, 1500, 16))
    seqs = rng.integers(0, 5, rows)
    ctx = np.array([int(rng.integers(0, case.lens[s] + 1)) for s in seqs])
    ctx[:5], seqs[:5] = case.lens, range(5)
    q = rng.normal(0, 1, (rows, heads * hd)).astype(np.float32)
    args = (dev(q), heads, ints(ctx - 1), ints(seqs))
    out = case.cache.decode_attention(*args)
    pick = sorted({0, 1, 2, 3, 4, rows // 2, rows - 2, rows - 1} | set(rng.integers(0, rows, 24).tolist()))
    check_rows(case, q[pick], out.cpu().numpy()[pick], heads, seqs[pick], ctx[pick])
    assert not out[torch.from_numpy(ctx == 0).cuda()].any()
    assert torch.equal(out, case.cache.decode_attention(*args)) and status() == 0


def test_empty_calls_and_other_types():
    from axion_b200.kv_pages import KVPages
    rng = np.random.default_rng(16)
    case = Case(rng, 2, 64, (40, 20))
    none, rows = ints([]), torch.zeros(0, 128, device="cuda")
    case.cache.append_rows(rows, rows, none, none)
    assert [tuple(x.shape) for x in case.cache.read_rows(none, none)] == [(0, 128), (0, 128)]
    q = torch.zeros(0, 256, device="cuda")
    assert case.cache.decode_attention(q, 4, none).shape == (0, 256)
    assert case.cache.chunk_attention(q, 4, ints([0]), none, 0).shape == (0, 256)
    pages = KVPages.empty([torch.zeros(4, 16, device="cuda")], 2, 2)
    pages.reserve(none, none), pages.fork(none, none, none), pages.free(none), pages.copy(none, none)
    assert int(pages.compact()) == 0 and status() == 0
    # 16-bit queries are taken as the fp32 numbers they are
    q16 = torch.from_numpy(rng.normal(0, 1, (2, 256)).astype(np.float16)).cuda()
    out = case.cache.decode_attention(q16, 4, ints([39, 19]))
    assert out.dtype == torch.float32
    check_rows(case, q16.float().cpu().numpy(), out.cpu().numpy(), 4, [0, 1], [40, 20])


def test_decode_long_context_keeps_its_ends():
    """20,011 tokens: the first and last token carry most of the weight, the slot behind the
    last would carry all of it, so a token lost or gained at either end shows."""
    rng = np.random.default_rng(12)
    n, hd = 20011, 128
    case = Case(rng, 1, hd, (n,))
    u = rng.normal(0, 1, hd).astype(np.float32)
    case.k[0][0], case.k[0][n - 1] = u, u
    for p in (0, n - 1):
        case.cache.append_rows(dev(case.k[0][p]), dev(case.v[0][p]), ints([0]), ints([p]))
    q = np.tile(u * 1.2, 4)[None].astype(np.float32)
    out = case.cache.decode_attention(dev(q), 4, ints([n - 1])).cpu().numpy()
    k, v = case.held(0, n, 0)
    s = np.exp((k @ q[0, :hd]) / np.sqrt(hd))
    assert s[0] / s.sum() > 0.2 and s[-1] / s.sum() > 0.2
    check_rows(case, q, out, 4, [0], [n])


def test_bad_pages_count_as_masked_and_are_reported():
    from axion_b200 import _lib, ops
    rng = np.random.default_rng(13)
    for bad in (-1, 10 ** 6, -7):
        case = Case(rng, 2, 64, (80,))
        case.cache.block_table[0, 2] = bad
        q = rng.normal(0, 1, (1, 4 * 64)).astype(np.float32)
        ops.status_clear()
        out = case.cache.decode_attention(dev(q), 4, ints([79])).cpu().numpy()
        assert status() == _lib.AXQ8_ERR_INVALID
        ops.status_clear()
        out2 = case.cache.chunk_attention(dev(q), 4, ints([0, 1]), ints([79]), 1).cpu().numpy()
        assert status() == _lib.AXQ8_ERR_INVALID
        keep = [p for p in range(80) if p // 16 != 2]
        case.k[0], case.v[0], case.lens = case.k[0][keep], case.v[0][keep], [64]
        check_rows(case, q, out, 4, [0], [64])
        check_rows(case, q, out2, 4, [0], [64])


def test_sequences_and_positions_outside_the_table():
    from axion_b200 import _lib, ops
    rng = np.random.default_rng(14)
    case = Case(rng, 2, 64, (32, 32))
    q = rng.normal(0, 1, (1, 4 * 64)).astype(np.float32)
    for seq, pos, ctx in ((2, 5, 0), (-1, 5, 0), (1, 32, 32), (0, 10 ** 9, 32)):
        ops.status_clear()
        out = case.cache.decode_attention(dev(q), 4, ints([pos]), ints([seq])).cpu().numpy()
        assert status() == _lib.AXQ8_ERR_INVALID
        check_rows(case, q, out, 4, [seq if ctx else 0], [ctx])


def test_offsets_past_32_bits():
    """A pool of more than 4 GiB: the last pages hold the sequence."""
    from axion_b200.paged_kv import PagedKVCache4
    kv, hd = 8, 128
    n_pages = (1 << 32) // (kv * 18 * hd) + 40
    pages = torch.empty(n_pages, kv, 18 * hd, dtype=torch.uint8, device="cuda")
    rng = np.random.default_rng(15)
    small = Case(rng, kv, hd, (70,))
    table = np.arange(n_pages - 5, n_pages, dtype=np.int32)[None]
    pages[n_pages - 5:] = 255
    cache = PagedKVCache4(kv, hd, pages=pages, block_table=dev(table))
    cache.append(dev(small.k[0].reshape(70, -1)), dev(small.v[0].reshape(70, -1)))
    q = rng.normal(0, 1, (70, 16 * hd)).astype(np.float32)
    out = cache.decode_attention(dev(q[:1]), 16, ints([69])).cpu().numpy()
    check_rows(small, q, out, 16, [0], [70])
    out = cache.chunk_attention(dev(q), 16, ints([0, 70]), ints([0]), 70).cpu().numpy()
    check_rows(small, q, out, 16, [0] * 70, range(1, 71))
    assert status() == 0


# ---- chunks ------------------------------------------------------------------------

def run_chunks(case, q, heads, rows, past, seqs=None, extra=0, max_rows=None):
    start = np.concatenate([[0], np.cumsum(rows)])
    out = torch.full((int(start[-1]) + extra, heads * case.hd), 7.0, device="cuda")
    got = case.cache.chunk_attention(dev(q), heads, ints(start), ints(past), max_rows or max(rows),
                                     None if seqs is None else ints(seqs), out=out)
    return got


@pytest.mark.parametrize("hd,heads,kv", SHAPES)
@pytest.mark.parametrize("rows,past", [((1,), (0,)), ((5, 1, 3), (44, 0, 200)), ((70,), (0,)),
                                       ((130, 17), (3, 250))])
def test_chunk_attention(hd, heads, kv, rows, past):
    rng = np.random.default_rng(hd * heads + sum(rows))
    case = Case(rng, kv, hd, [a + b for a, b in zip(rows, past)], scale=1.5)
    q = rng.normal(0, 1, (sum(rows), heads * hd)).astype(np.float32)
    out = run_chunks(case, q, heads, rows, past)
    seqs = [i for i, n in enumerate(rows) for _ in range(n)]
    ctx = [p + j + 1 for n, p in zip(rows, past) for j in range(n)]
    check_rows(case, q, out.cpu().numpy(), heads, seqs, ctx)
    assert torch.equal(out, run_chunks(case, q, heads, rows, past))
    assert status() == 0


@pytest.mark.parametrize("hd,heads,kv", [(64, 8, 2), (128, 4, 4), (128, 8, 2)])
def test_chunk_rows_of_no_chunk_stay(hd, heads, kv):
    """Empty chunks, more room than rows, chosen sequences, positions before the start."""
    rng = np.random.default_rng(21)
    case = Case(rng, kv, hd, (150, 60, 200))
    rows, past, seqs = (0, 40, 0, 33, 2, 6), (9, 100, 0, 20, -1, -9), (0, 0, 1, 2, 1, 1)
    total, extra = sum(rows), 13
    q = rng.normal(0, 1, (total + extra, heads * hd)).astype(np.float32)
    out = run_chunks(case, q, heads, rows, past, seqs, extra, max_rows=300).cpu().numpy()
    which = [s for s, n in zip(seqs, rows) for _ in range(n)]
    ctx = [p + j + 1 for n, p in zip(rows, past) for j in range(n)]
    check_rows(case, q, out, heads, which, ctx)
    assert np.all(out[total:] == 7.0) and status() == 0


def test_chunk_starts_that_do_not_fit_are_reported():
    from axion_b200 import _lib, ops
    rng = np.random.default_rng(22)
    case = Case(rng, 2, 64, (64, 64))
    q = rng.normal(0, 1, (8, 4 * 64)).astype(np.float32)
    for start, rows in (([0, 4, 9], 8), ([-1, 4, 8], 8), ([0, 6, 8], 5), ([4, 2, 8], 8)):
        ops.status_clear()
        out = torch.full((8, 4 * 64), 7.0, device="cuda")
        case.cache.chunk_attention(dev(q), 4, ints(start), ints([10, 10]), rows, out=out)
        want = 0 if start == [4, 2, 8] else _lib.AXQ8_ERR_INVALID
        assert status() == want, start


def test_chunk_long_past():
    """A few rows over 9,000 tokens (work split over the past), and 200 of them."""
    rng = np.random.default_rng(23)
    for rows in (3, 200):
        case = Case(rng, 1, 64, (9000 + rows,))
        q = rng.normal(0, 1.5, (rows, 2 * 64)).astype(np.float32)
        out = run_chunks(case, q, 2, (rows,), (9000,)).cpu().numpy()
        pick = sorted({0, 1, rows // 2, rows - 1})
        check_rows(case, q[pick], out[pick], 2, [0] * len(pick), [9001 + i for i in pick])


# (hd, heads, kv, rows, past): enough rows and KV heads for the tensor-core tiles
TILES = [(128, 32, 8, (300, 1, 129, 64), (0, 700, 3, 0)), (64, 32, 8, (200, 255, 0, 40), (130, 0, 5, 1)),
         (32, 16, 16, (400, 33), (0, 250)), (128, 16, 16, (257, 256), (15, 0)), (64, 48, 16, (97, 200), (0, 64)),
         (64, 56, 8, (130, 131), (17, 0)), (128, 64, 4, (100, 120), (0, 333))]


@pytest.mark.parametrize("hd,heads,kv,rows,past", TILES)
def test_chunk_attention_of_long_chunks(hd, heads, kv, rows, past):
    """Rows at and beside the tiles' borders, against 64 bits; rows behind the last stay."""
    rng = np.random.default_rng(hd + heads + rows[0])
    case = Case(rng, kv, hd, [a + b for a, b in zip(rows, past)], scale=1.5)
    total = sum(rows)
    q = (rng.normal(0, 1, (total + 5, heads * hd)) * np.exp2(rng.integers(-3, 3, (total + 5, 1)))).astype(np.float32)
    start = np.concatenate([[0], np.cumsum(rows)])
    out = torch.full((total + 5, heads * hd), 7.0, device="cuda")
    args = (dev(q), heads, ints(start), ints(past), max(rows))
    case.cache.chunk_attention(*args, out=out)
    first = out.clone()
    seqs = np.array([i for i, n in enumerate(rows) for _ in range(n)])
    ctx = np.array([p + j + 1 for n, p in zip(rows, past) for j in range(n)])
    border = 128 * kv // heads
    pick = sorted({int(s + j) for s, n in zip(start, rows) for j in (0, 1, 15, 16, border - 1, border, 2 * border - 1,
                   2 * border, n // 2, n - 2, n - 1) if 0 <= j < n})
    check_rows(case, q[pick], out.cpu().numpy()[pick], heads, seqs[pick], ctx[pick])
    assert bool((out[total:] == 7.0).all()) and status() == 0
    case.cache.chunk_attention(*args, out=out)
    assert torch.equal(out, first)                   # bit for bit


@pytest.mark.parametrize("heads,hd,kv,rows,past", [(32, 128, 8, 200, 16000), (16, 64, 8, 330, 7000)])
def test_long_chunks_over_a_long_past(heads, hd, kv, rows, past):
    """Sums of values of one sign over thousands of tokens: what the tensor cores drop at each of
    their sums (at most a unit in the last place, always the same way) must not pile up.  1024
    tokens summed there take 128 products, each dropping at most 2^-23 of a sum that grows
    evenly: 128 / 2 * 2^-23 = 7.6e-6; the rest (weights kept to 2^-22, partial sums added in
    fp32) is below 2e-6."""
    rng = np.random.default_rng(past)
    case = Case(rng, kv, hd, (past + rows,))
    case.v[0][:] = np.abs(case.v[0]) + 0.5
    case.append(0, None)
    q = rng.normal(0, 1, (rows, heads * hd)).astype(np.float32)
    out = run_chunks(case, q, heads, (rows,), (past,))
    assert torch.equal(out, run_chunks(case, q, heads, (rows,), (past,)))
    out, worst = out.cpu().numpy(), 0.0
    for kvh in range(kv):
        k, v = case.held(0, past + rows, kvh)
        h = kvh * (heads // kv)
        for r in (0, rows // 2, rows - 1):
            n = past + r + 1
            ref = km.attention(q[r].reshape(heads, hd)[h].astype(np.float64), k[:n], v[:n], 1 / np.sqrt(hd))
            err = np.linalg.norm(out[r].reshape(heads, hd)[h] - ref) / np.linalg.norm(ref)
            worst = max(worst, err)
    assert worst <= 1e-5, worst
    assert status() == 0


def test_long_chunks_with_empty_rows_and_bad_pages():
    """Positions before the start, a page outside the pool, a sequence outside the table."""
    from axion_b200 import _lib
    rng = np.random.default_rng(27)
    case = Case(rng, 8, 64, (300, 300), scale=1.5)
    case.cache.block_table[1, 9] = 10 ** 6
    q = rng.normal(0, 1, (900, 32 * 64)).astype(np.float32)
    out = run_chunks(case, q, 32, (300, 300, 300), (-40, 0, 0), (0, 1, 5)).cpu().numpy()
    assert status() == _lib.AXQ8_ERR_INVALID
    assert not out[:40].any() and not out[600:].any()
    check_rows(case, q[[40, 41, 299]], out[[40, 41, 299]], 32, [0] * 3, [1, 2, 260])
    check_rows(case, q[[300, 443]], out[[300, 443]], 32, [1] * 2, [1, 144])
    keep = [p for p in range(300) if p // 16 != 9]
    case.k[1], case.v[1], case.lens = case.k[1][keep], case.v[1][keep], [300, 284]
    check_rows(case, q[[450, 599]], out[[450, 599]], 32, [1] * 2, [144, 284])


@pytest.mark.parametrize("hd,heads,kv,long", [(128, 16, 4, False), (64, 16, 2, False), (128, 9, 1, False),
                                              (64, 32, 8, True), (128, 32, 8, True), (32, 16, 16, True)])
def test_growing_scores_and_values(hd, heads, kv, long):
    """Scores that grow by 60 and values by 2^12 along the sequence move the softmax reference and
    the value scale many times; then both fall again."""
    rng = np.random.default_rng(hd + heads)
    n = 420
    case = Case(rng, kv, hd, (n, n))
    u = rng.normal(0, 1, hd)
    up = np.concatenate([np.linspace(-30, 30, n // 2), np.linspace(30, -30, n - n // 2)])
    for s in range(2):
        case.k[s][:] = (0.3 * case.k[s] + (up * np.sqrt(hd) / (u @ u))[:, None, None] * u).astype(np.float32)
        case.v[s][:] = case.v[s] * np.exp2(up / 5)[:, None, None].astype(np.float32)
    case.append(0, None)
    rows = n if long else 1
    q = np.tile(u, (2 * rows, heads)).astype(np.float32) * rng.uniform(0.9, 1.1, (2 * rows, 1)).astype(np.float32)
    past = n - rows
    if long:
        out = run_chunks(case, q, heads, (rows, rows), (past, past)).cpu().numpy()
        pick = [0, 1, 100, 209, 210, 260, n - 1, n, n + 130, 2 * n - 1]
    else:
        out = case.cache.decode_attention(dev(q), heads, ints([n - 1, n - 1])).cpu().numpy()
        pick = [0, 1]
    check_rows(case, q[pick], out[pick], heads, [r // rows for r in pick], [past + r % rows + 1 for r in pick])
    assert status() == 0


def test_calls_from_two_threads():
    """Two threads on one cache and one stream: the kernels of their calls do not mix."""
    import threading
    rng = np.random.default_rng(28)
    case = Case(rng, 2, 128, (3000, 2500))
    qs = [dev(rng.normal(0, 1, (2, 8 * 128)).astype(np.float32)) for _ in range(2)]
    pos = ints([2999, 2499])
    want = [case.cache.decode_attention(x, 8, pos) for x in qs]
    bad = []

    def work(i):
        for _ in range(200):
            if not torch.equal(case.cache.decode_attention(qs[i], 8, pos), want[i]):
                bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_masked_slots_do_not_leak():
    """Later tokens of the same page and tile hold the largest values the format has."""
    rng = np.random.default_rng(24)
    case = Case(rng, 2, 128, (200,))
    n = 90
    case.k[0][n:] = 30000.0 * np.sign(rng.normal(0, 1, case.k[0][n:].shape))
    case.v[0][n:] = 30000.0
    case.append(n, None)
    q = rng.normal(0, 1, (n, 8 * 128)).astype(np.float32)
    out = run_chunks(case, q, 8, (n,), (0,)).cpu().numpy()
    check_rows(case, q, out, 8, [0] * n, range(1, n + 1))
    out = case.cache.decode_attention(dev(q[:1]), 8, ints([n - 1])).cpu().numpy()
    check_rows(case, q[:1], out, 8, [0], [n])
    case = Case(rng, 8, 128, (500,))            # the same in the tiles of long chunks
    case.k[0][400:] = 30000.0 * np.sign(rng.normal(0, 1, case.k[0][400:].shape))
    case.v[0][400:] = 30000.0
    case.append(400, None)
    q = rng.normal(0, 1, (400, 32 * 128)).astype(np.float32)
    out = run_chunks(case, q, 32, (400,), (0,)).cpu().numpy()
    pick = [0, 127, 128, 383, 384, 399]
    check_rows(case, q[pick], out[pick], 32, [0] * 6, [p + 1 for p in pick])


# ---- streams and graphs ----------------------------------------------------------------

def test_two_captured_graphs_and_an_eager_call_at_once():
    """Two graphs over one cache replayed on two streams beside eager calls: same results."""
    rng = np.random.default_rng(31)
    case = Case(rng, 2, 128, (3000, 2500))
    q = [dev(rng.normal(0, 1, (2, 8 * 128)).astype(np.float32)) for _ in range(3)]
    pos = ints([2999, 2499])
    want = [case.cache.decode_attention(x, 8, pos) for x in q]
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(3)]
    for x in q[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(case.cache.decode_attention(x, 8, pos))
        graphs.append(g)
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            third = case.cache.decode_attention(q[2], 8, pos)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
        assert torch.equal(third, want[2])
    assert status() == 0


def test_a_captured_step_follows_its_inputs():
    """Append and both attentions captured once, replayed with other rows and positions."""
    rng = np.random.default_rng(32)
    case = Case(rng, 2, 64, (40, 40))
    k, v, q = (torch.zeros(2, w, device="cuda") for w in (128, 128, 256))
    seq, pos = ints([0, 1]), ints([0, 0])
    start = ints([0, 1, 2])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        case.cache.append_rows(k, v, seq, pos)
        a = case.cache.decode_attention(q, 4, pos)
        b = case.cache.chunk_attention(q, 4, start, pos, 1)
    for p in (7, 30, 39):
        new = [rng.normal(0, 1, (2, w)).astype(np.float32) for w in (128, 128, 256)]
        for t, x in zip((k, v, q), new):
            t.copy_(dev(x))
        pos.copy_(ints([p, p // 2]))
        g.replay()
        for s, at in ((0, p), (1, p // 2)):
            case.k[s][at], case.v[s][at] = new[0][s].reshape(2, 64), new[1][s].reshape(2, 64)
        for out in (a, b):
            check_rows(case, new[2], out.cpu().numpy(), 4, [0, 1], [p + 1, p // 2 + 1])


def test_the_c_entry_points_on_a_stream_of_their_own():
    """The C ABI with caller workspaces: zero before, usable again after."""
    from axion_b200 import _lib
    rng = np.random.default_rng(33)
    lib = _lib.load()
    case = Case(rng, 2, 128, (1000, 30, 500))
    q = rng.normal(0, 1, (3, 8 * 128)).astype(np.float32)
    s = torch.cuda.Stream()
    qd, pos, out = dev(q), ints([999, 29, 499]), torch.empty(3, 8 * 128, device="cuda")
    need = lib.axkv4_decode_attn_workspace(C.byref(case.cache.c), 3, 8)
    ws = torch.zeros(need, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    for _ in range(3):
        out.fill_(0)
        torch.cuda.synchronize()
        _lib.check(lib.axkv4_decode_attn(C.byref(case.cache.c), qd.data_ptr(), 8 * 128, 3, 8, None,
                                         pos.data_ptr(), out.data_ptr(), ws.data_ptr(), need, s.cuda_stream))
        s.synchronize()
        check_rows(case, q, out.cpu().numpy(), 8, range(3), [1000, 30, 500])


def test_the_reference_names():
    """initialize / append / materialize / attention / prefill_attention as PagedKVCache has them."""
    from axion_b200.paged_kv import PagedKVCache4
    rng = np.random.default_rng(34)
    kv = PagedKVCache4(2, 64, max_seqs=2, max_tokens=64)
    kv.initialize(128, 16)
    k = rng.normal(0, 1, (2, 30, 128)).astype(np.float32)
    v = rng.normal(0, 1, (2, 30, 128)).astype(np.float32)
    for s in range(2):
        for a, b in ((0, 10), (10, 11), (11, 30)):
            kv.append(dev(k[s, a:b]), dev(v[s, a:b]), seq=s)
        assert np.array_equal(kv.materialize_keys(s).cpu().numpy(), km.values(k[s].reshape(30, 2, 64)).reshape(30, -1))
    q = rng.normal(0, 1, (10, 256)).astype(np.float32)
    out = kv.prefill_attention(dev(q), 4, 5, 25).cpu().numpy()
    dec = kv.attention(dev(q[[4, 9]]), 4).cpu().numpy()
    for s in range(2):
        kk, vv = (km.values(x[s].reshape(30, 2, 64)) for x in (k, v))
        for t in range(5):
            for h in range(4):
                n, qh = 26 + t, q[s * 5 + t].reshape(4, 64)[h].astype(np.float64)
                ref = km.attention(qh, kk[:n, h // 2], vv[:n, h // 2], 0.125)
                tol = km.tolerance(qh, kk[:n, h // 2], vv[:n, h // 2], 0.125)
                assert np.abs(out[s * 5 + t].reshape(4, 64)[h] - ref).max() <= tol
                if t == 4:
                    assert np.abs(dec[s].reshape(4, 64)[h] - ref).max() <= tol
    with pytest.raises(RuntimeError):
        kv.initialize(64)
    with pytest.raises(RuntimeError):
        kv.append(dev(k[0]), dev(v[0][:3]))
    with pytest.raises(RuntimeError):
        kv.append(dev(np.zeros((40, 128), np.float32)), dev(np.zeros((40, 128), np.float32)))
    with pytest.raises(RuntimeError):
        kv.prefill_attention(dev(q), 4, 5, 27)
    with pytest.raises(RuntimeError):
        kv.decode_attention(dev(q), 3, ints(range(10)))
    with pytest.raises(RuntimeError):
        kv.decode_attention(dev(q), 4, torch.zeros(10, dtype=torch.int64, device="cuda"))
