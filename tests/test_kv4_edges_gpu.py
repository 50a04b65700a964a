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
