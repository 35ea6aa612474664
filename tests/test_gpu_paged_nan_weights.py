"""Added-up weights where a row has none that are numbers."""
import numpy as np
import pytest

import paged_model as pm
from test_gpu_paged import TYPES, dev, fill_new, held, on_gpu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act,kind", TYPES)
@pytest.mark.parametrize("window,first", [(0, 0), (40, 3)])
def test_a_row_of_nan_reaches_only_the_tokens_that_it_sees(pkg, act, kind, window, first):
    """NaN in a query of one row, for one kv head; in a key that only the last rows of another sequence see; one row that is all"""
    kv, heads, dim = 2, 6, 64
    B = pm.Batch(43, [300, 61, 0, 700], [4, 5, 1, 2], kv, dim, 16, weights=True)
    fill_new(B)
    p, i = B.slot(1, 61 + 2)
    B.k[p, 1, i, 5] = np.nan
    q = B.rng.standard_normal((B.total, heads, dim))
    q[1, 2, 7] = np.nan          # the second row of the first sequence: it does not see the last two rows' tokens
    q[9, 0, 0] = np.nan
    q64, qt = held(q.reshape(B.total, -1), act)
    cache, k64, v64 = on_gpu(pkg, B, kind)
    pkg.op_paged_attention(cache, qt, dev(B.row_start), 5, heads, 0.125, window=window, first=first, accumulate=True)
    _, added, _, _ = pm.attend(B, q64.reshape(-1, heads, dim), k64, v64, heads, 0.125, window, first)
    got = cache.weight.double().cpu().numpy()
    want = B.weight.astype(np.float32).astype(np.float64) + added
    assert 0 < np.isnan(added).sum() < 2000
    assert np.array_equal(np.isnan(got), np.isnan(want))
    ok = ~np.isnan(want)
    assert np.all(np.abs(got - want)[ok] <= 2e-5 * (1 + want[ok]))
