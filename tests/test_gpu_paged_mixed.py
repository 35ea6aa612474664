"""Batches in which what may be odd is odd at once: pages that are not there, rows behind the table, windows, queries, keys and values that are
not finite, batches padded and of empty sequences, with and without added-up weights."""
import numpy as np
import pytest
import torch

import paged_model as pm
from test_gpu_paged import TYPES, dev, fill_new, held, on_gpu
from test_gpu_paged_odd_values import alike

pytestmark = pytest.mark.gpu


def batch(seed, many):
    rng = np.random.default_rng(seed)
    kv, group = int(rng.choice([1, 2, 8])), int(rng.choice([1, 2, 3, 7]))
    dim, page = int(rng.choice([8, 64, 72, 128, 256])), int(rng.choice([16, 32, 128]))
    n = int(rng.integers(1, 6))
    lens = rng.integers(0, 500, n)
    rows = rng.integers(0, 6, n)
    if many:   # prompts: 300 rows of 16 heads at least
        kv, group = 8, int(rng.choice([2, 3]))
        rows[rng.integers(n)] = rng.integers(260, 330)
    ld = int(rng.choice([0, 0, 16, 4000])) or None
    if ld == 16:
        ld = max(2, 512 // page)
    extra = [0] * 40 if many and rng.random() < 0.5 else []   # so that a workgroup has more rows
    B = pm.Batch(seed, lens.tolist() + extra, rows.tolist() + extra, kv, dim, page, table_ld=ld, weights=True)
    fill_new(B)
    return rng, B, kv * group


@pytest.mark.parametrize("act,kind", TYPES)
@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("seed", range(12))
def test_all_at_once(pkg, act, kind, many, seed):
    """A weight is off by f32's half step times 2 (256 + 8 6) for a score of up to 6 and 600 for the sum, 7e-5 relative; with bf16 rows
    by bf16's, as the result is, of values below 4"""
    rng, B, heads = batch(1000 + seed, many)
    if B.total == 0:
        B, heads = pm.Batch(seed, [5], [2], 1, 64, 16, weights=True), 2
        fill_new(B)
    for b in range(len(B.lens)):          # pages that are not there
        for i in range(B.ld):
            if B.table[b, i] >= 0 and rng.random() < 0.08:
                B.table[b, i] = int(rng.choice([-1, B.n_pages, 2 ** 31 - 1, -2 ** 31]))
    for _ in range(8):                    # values that are not finite; a key that is NaN
        b = int(rng.integers(len(B.lens)))
        end = min(B.lens[b] + B.rows[b], B.ld * B.page)
        if end:
            t = int(rng.integers(end))
            if B.there(b, t):
                p, i = B.slot(b, t)
                B.v[p, int(rng.integers(B.kv)), i, int(rng.integers(B.dim))] = rng.choice([np.inf, -np.inf, np.nan])
                if rng.random() < 0.1:
                    B.k[p, int(rng.integers(B.kv)), i, 0] = np.nan
    q = B.rng.standard_normal((B.total + 4, heads, B.dim))
    if B.total > 3:
        q[int(rng.integers(B.total)), int(rng.integers(heads)), 0] = np.nan
    window, first = (int(rng.integers(1, 200)), int(rng.choice([0, 1, 40]))) if rng.random() < 0.6 else (0, 0)
    q64, qt = held(q.reshape(B.total + 4, -1), act)
    cache, k64, v64 = on_gpu(pkg, B, kind)
    old = cache.weight.clone()
    most = max(B.rows)
    want, added, _, _ = pm.attend(B, q64.reshape(-1, heads, B.dim), k64, v64, heads, B.dim ** -0.5, window, first)
    for accumulate in (False, True):
        out = torch.full((B.total + 4, heads * B.dim), 7.5, dtype=qt.dtype, device="cuda")
        scratch = None
        if accumulate and seed % 2 and B.total + 4 > 128:   # for passes of 128 rows
            scratch = pkg.op_paged_attention_scratch(cache, 128, min(most, 128), heads, True, window, first)
        pkg.op_paged_attention(cache, qt, dev(B.row_start), most, heads, B.dim ** -0.5, window=window, first=first, accumulate=accumulate, out=out,
                               scratch=scratch)
        got = out.double().cpu().numpy()
        assert np.all(got[B.total:] == 7.5)
        alike(got[:B.total].reshape(want.shape), want, 2 ** -5 if act == "bf16" else 1e-4)
        if not accumulate:
            assert torch.equal(torch.nan_to_num(cache.weight, nan=-1.0), torch.nan_to_num(old, nan=-1.0))
    there = ~np.isnan(old.cpu().numpy())
    got, sums = cache.weight.double().cpu().numpy()[there], (old.double().cpu().numpy() + added)[there]
    assert np.array_equal(np.isnan(got), np.isnan(sums))
    ok = ~np.isnan(sums)
    assert np.all(np.abs(got - sums)[ok] <= 1e-4 * (1 + sums[ok]))
