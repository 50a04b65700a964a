"""The 4-bit cache's attention where tolerances that grow with the context hide a
fault: non-finite queries, long sums of equal terms, values of very different size,
and pages at the seams of split contexts."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kv4_model as km
from test_kv4_gpu import Case, check_rows, clean_status, dev, ints, run_chunks, status  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd,heads,kv", [(128, 8, 2), (64, 14, 2), (128, 16, 1)])
@pytest.mark.parametrize("n", [1, 100, 20000])
def test_a_query_that_is_no_number_shows_in_its_heads(hd, heads, kv, n):
    """One NaN and one infinite element: softmax of these scores is NaN, in those heads alone,
    whether the context is one CTA's work or shared among many."""
    rng = np.random.default_rng(n + heads)
    case = Case(rng, kv, hd, (n,))
    q = rng.normal(0, 1, (1, heads, hd)).astype(np.float32)
    q[0, 1, 5], q[0, 4, hd - 1] = np.nan, np.inf
    args = (dev(q.reshape(1, -1)), heads)
    for out in (case.cache.decode_attention(*args, ints([n - 1])),
                case.cache.chunk_attention(*args, ints([0, 1]), ints([n - 1]), 1)):
        out = out.cpu().numpy().reshape(heads, hd)
        bad = [1, 4]
        assert np.isnan(out[bad]).all()
        rest = [h for h in range(heads) if h not in bad]
        assert np.isfinite(out[rest]).all()
        for h in (0, 2, heads - 1):
            k, v = case.held(0, n, h // (heads // kv))
            scale = 1 / np.sqrt(hd)
            ref = km.attention(q[0, h].astype(np.float64), k, v, scale)
            assert np.abs(out[h] - ref).max() <= km.tolerance(q[0, h].astype(np.float64), k, v, scale)


def equal_tokens(rng, case, n):
    """Every token of every sequence the same K and the same positive V: the result is V itself."""
    k, v = rng.normal(0, 1, (case.kv, case.hd)), rng.uniform(0.5, 1.5, (case.kv, case.hd))
    for s in range(len(case.lens)):
        case.k[s][:], case.v[s][:] = k, v
    case.append(0, None)
    return np.stack([case.held(0, 1, h)[1][0] for h in range(case.kv)])          # [kv, hd]


@pytest.mark.parametrize("heads,hd,kv,rows,past", [(32, 128, 8, 200, 16000), (16, 64, 8, 330, 7000)])
def test_long_chunks_of_equal_tokens(heads, hd, kv, rows, past):
    """Equal weights round the same way at every addition, and equal products are cut alike.
    The weights' sum is taken 128 tokens at a time (two chains of 64 additions of at most 2^-24:
    3.8e-6) and joined without loss.  O: a tensor core aligns the 16 products of an instruction
    and the sum to the largest and cuts them, at least two bits below the sum's last place (as
    measured by Fasi, Higham, Mikaitis and Pranesh, Numerical behavior of NVIDIA tensor cores,
    2021), so 16 / 4 + 1 = 5 units of at most 2^-23 of the sum; 128 instructions are a piece of
    1024 tokens, whose sum grows evenly: 128 / 2 * 5 * 2^-23 = 3.8e-5.  The weights' fp16 pairs
    2.4e-7, 17 pieces of 2^-24.  (One chain of additions was 1.3e-4 and 7e-5 off here.)"""
    rng = np.random.default_rng(past + 1)
    case = Case(rng, kv, hd, (past + rows,))
    v = equal_tokens(rng, case, past + rows)
    q = rng.normal(0, 1, (rows, heads * hd)).astype(np.float32)
    out = run_chunks(case, q, heads, (rows,), (past,)).cpu().numpy().reshape(rows, kv, -1, hd)
    worst = np.abs(out / v[None, :, None] - 1).max()
    assert worst <= 128 / 2 * 5 * 2.0 ** -23 + 64 * 2.0 ** -24 + 2.0 ** -22 + 17 * 2.0 ** -24, worst
    assert status() == 0


def test_many_long_sequences_of_equal_tokens():
    """64 sequences over the same 131,072 tokens, each page a copy of the first: a CTA walks
    thousands of pages of one tile.  It takes 1024 of them at a time, 256 a warp: 256 additions
    of weights, and of products, of at most 2^-24 of sums that grow evenly; a step's products
    start from zero, 4 instructions of at most 5 units of 2^-23 (test_long_chunks_of_equal_tokens);
    2^-22 for the weights' pairs; 8 pieces and 4 warps of 2^-24.  (3.9e-5 off in one chain.)"""
    limit = 2 * 256 / 2 * 2.0 ** -24 + 4 * 5 * 2.0 ** -23 + 2.0 ** -22 + 12 * 2.0 ** -24
    from axion_b200.paged_kv import PagedKVCache4
    rng = np.random.default_rng(64)
    n, kv, hd, heads = 131072, 8, 128, 32
    k, v = rng.normal(0, 1, (kv, hd)).astype(np.float32), rng.uniform(0.5, 1.5, (kv, hd)).astype(np.float32)
    pages = torch.empty(n // 16, kv, 18 * hd, dtype=torch.uint8, device="cuda")
    table = np.tile(np.arange(n // 16, dtype=np.int32), (64, 1))
    cache = PagedKVCache4(kv, hd, pages=pages, block_table=dev(table))
    kd, vd = (dev(x.reshape(1, -1)).repeat(16, 1) for x in (k, v))
    kd[3] *= 1.25                               # not every weight is a power of two
    cache.append_rows(kd, vd, ints([0] * 16), ints(range(16)))
    pages[1:] = pages[0]
    held = km.values(v)
    for per, seqs in ((1, 64), (4, 48)):       # 4 columns of a tile, and 16
        q = rng.normal(0, 1, (seqs * per, heads * hd)).astype(np.float32)
        if per == 1:
            out = cache.decode_attention(dev(q), heads, ints([n - 1] * seqs))
        else:
            out = cache.chunk_attention(dev(q), heads, ints(range(0, seqs * per + 1, per)), ints([n - per] * seqs), per)
        out = out.cpu().numpy().reshape(seqs * per, kv, -1, hd)
        worst = np.abs(out / held[None, :, None] - 1).max()
        assert worst <= limit, (per, worst)
    assert status() == 0


def check_sizes(case, q, out, heads, seqs, ctx):
    """As check_rows, relative to what each output sums instead of the largest value of all:
    tolerance's factor times sum p |v|, and what a weight held as an fp16 pair may be off at
    the bottom (2^-32 of the largest weight, for every token)."""
    scale = 1 / np.sqrt(case.hd)
    for r, (s, n) in enumerate(zip(seqs, ctx)):
        for h in range(heads):
            k, v = case.held(s, n, h // (heads // case.kv))
            qh = q[r].reshape(heads, -1)[h].astype(np.float64)
            p = np.exp((k @ qh) * scale - ((k @ qh) * scale).max())
            p /= p.sum()
            tol = km.tolerance(qh, k, np.ones((1, 1)), scale) * (p @ np.abs(v)) + 2.0 ** -32 * p.max() * np.abs(v).sum(0)
            err = np.abs(out[r].reshape(heads, -1)[h] - p @ v)
            assert (err <= tol).all(), (r, h, n, float((err / tol).max()))


@pytest.mark.parametrize("hd,heads,kv", [(32, 8, 2), (64, 14, 2), (128, 8, 2), (128, 4, 4), (128, 16, 1)])
def test_values_of_very_different_size(hd, heads, kv):
    """Blocks of dims and tokens whose values differ by up to 2^22, small ones with the weight."""
    rng = np.random.default_rng(hd + heads)
    n = 230
    case = Case(rng, kv, hd, (n, n, n))
    for b in range(hd // 32):                                   # sequence 0: by block of dims
        case.v[0][..., 32 * b:32 * b + 32] *= 1000.0 * 10.0 ** (-2 * b)
    case.v[1] *= np.exp2(rng.integers(-9, 13, (n, 1, 1))).astype(np.float32)     # 1: by token
    u = rng.normal(0, 1, hd)                                    # 2: huge values of no weight
    far = rng.permutation(n)[:n // 3]
    case.v[2][far] *= 8000.0
    for s in (1, 2):
        case.v[s] = np.clip(case.v[s], -32768, 32768)
    case.k[2][far] = (-60 * np.sqrt(hd) / (u @ u) * u).astype(np.float32)
    case.k[2][[i for i in range(n) if i not in far]] *= 0.1
    case.append(0, None)
    q = rng.normal(0, 1, (3, heads * hd)).astype(np.float32)
    q[2] = np.tile(u, heads)
    out = case.cache.decode_attention(dev(q), heads, ints([n - 1] * 3)).cpu().numpy()
    check_sizes(case, q, out, heads, range(3), [n] * 3)
    out = run_chunks(case, np.repeat(q, 2, 0), heads, (2, 2, 2), (n - 2,) * 3).cpu().numpy()
    check_sizes(case, np.repeat(q, 2, 0), out, heads, [0, 0, 1, 1, 2, 2], [n - 1, n] * 3)
    assert status() == 0


@pytest.mark.parametrize("hd,heads,kv", [(64, 8, 2), (128, 8, 4), (128, 32, 8)])
def test_later_rows_of_a_chunk_do_not_show_in_earlier_ones(hd, heads, kv):
    """Draft rows whose last tokens hold the largest values there are: the rows before see none
    of them, and come out as they do without them."""
    rng = np.random.default_rng(hd * heads)
    rows, past = 6, 87
    case = Case(rng, kv, hd, (past + rows,))
    q = rng.normal(0, 1, (rows, heads * hd)).astype(np.float32)
    case.k[0][past + 3:] = 30000.0 * np.sign(rng.normal(0, 1, (3, kv, hd)))
    case.v[0][past + 3:] = 30000.0
    case.append(past, None)
    out = run_chunks(case, q, heads, (rows,), (past,)).cpu().numpy()
    check_rows(case, q[:3], out[:3], heads, [0] * 3, [past + 1, past + 2, past + 3])
    check_sizes(case, q[:3], out[:3], heads, [0] * 3, [past + 1, past + 2, past + 3])


@pytest.mark.parametrize("heads,hd,kv,rows", [(8, 128, 2, 1), (14, 64, 2, 1), (16, 32, 1, 1), (8, 128, 2, 5)])
def test_every_page_of_a_long_context_counts(heads, hd, kv, rows):
    """20,011 tokens in a split context, 1e-5 of the result's norm: a page lost or taken twice at a
    seam is about 8e-4 of the weight, 80 times that.  The bound: scores 16 products each dropping
    at most 2^-23 of a sum |q k| / sqrt(hd) of about 2, 4e-6; weights 2^-22; sums in pieces of
    at most 32 additions of 2^-24, 2e-6."""
    rng = np.random.default_rng(heads + rows)
    n = 20011
    case = Case(rng, kv, hd, (n, n - 777))
    for s in range(2):
        case.v[s][:] = np.abs(case.v[s]) + 0.5
    case.append(0, None)
    q = rng.normal(0, 0.3, (2 * rows, heads * hd)).astype(np.float32)
    if rows == 1:
        out = case.cache.decode_attention(dev(q), heads, ints(x - 1 for x in case.lens))
    else:
        out = run_chunks(case, q, heads, (rows, rows), [x - rows for x in case.lens])
    out = out.cpu().numpy().reshape(2 * rows, heads, hd)
    for s in range(2):
        for kvh in range(kv):
            k, v = case.held(s, case.lens[s], kvh)
            for r in {0, rows - 1}:
                m = case.lens[s] - rows + r + 1
                for h in range(kvh * heads // kv, (kvh + 1) * heads // kv, 3):
                    qh = q[s * rows + r].reshape(heads, hd)[h].astype(np.float64)
                    ref = km.attention(qh, k[:m], v[:m], 1 / np.sqrt(hd))
                    err = np.linalg.norm(out[s * rows + r, h] - ref) / np.linalg.norm(ref)
                    assert err <= 1e-5, (s, r, h, err)
    assert status() == 0
