"""Batches in which what may be odd is odd at once: pages that are not there, rows behind the table, windows, queries, keys and values that are
not finite, batches padded and of empty sequences, with and without added-up weights."""
import numpy as np
import pytest
import torch

import paged_model as pm
from test_gpu_paged import TYPES, check_evict, check_verify, dev, drafted, fill_new, held, on_gpu
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


@pytest.mark.parametrize("act,kind", TYPES)
@pytest.mark.parametrize("seed", range(6))
def test_append_all_at_once(pkg, act, kind, seed):
    """Up to 200 sequences, some without rows, pages that are not there, rows behind the table and behind the rotation's, a padded batch;
    in place where the seed is odd. One rounding to each type, two products and a sum in f32 in front of it."""
    rng = np.random.default_rng(2000 + seed)
    n, kv, group = int(rng.choice([1, 5, 64, 65, 200])), int(rng.choice([1, 2, 5])), int(rng.choice([1, 3, 7]))
    dim = int(rng.choice([8, 64, 72, 128, 256]))
    rot, page = 8 * int(rng.integers(0, dim // 8 + 1)), int(rng.choice([16, 64]))
    rows = np.where(rng.random(n) < 0.4, 0, rng.integers(0, 7, n)).tolist()
    rows[-1] = 2
    B = pm.Batch(seed, rng.integers(0, 90, n).tolist(), rows, kv, dim, page, table_ld=int(rng.choice([1, 3, 8])), weights=True)
    B.table[rng.random(B.table.shape) < 0.1] = -1
    heads, pad = kv * group, 5
    fused = rng.standard_normal((B.total + pad, (heads + 2 * kv) * dim))
    f64, ft = held(fused, act)
    q, k, v = ft[:, :heads * dim], ft[:, heads * dim:(heads + kv) * dim], ft[:, (heads + kv) * dim:]
    positions = 95
    sin, cos = pkg.op_rope_table(positions, rot, 1e4) if rot else (None, None)
    pos = rng.integers(0, 120, n).astype(np.int32) if rng.random() < 0.5 else None
    cache, want_k, want_v = on_gpu(pkg, B, kind)
    want_w = cache.weight.double().cpu().numpy()
    want_q = f64[:, :heads * dim].copy()
    out = q if seed % 2 else torch.from_numpy(want_q).cuda().to(ft.dtype)
    pkg.op_paged_append(cache, q, k, v, dev(B.row_start), sin, cos, pos=None if pos is None else dev(pos), out=out)
    sn, cs = (sin.cpu().numpy(), cos.cpu().numpy()) if rot else (None, None)
    size_q, size_k = np.zeros_like(want_q), np.zeros_like(want_k)
    for b, n_old in enumerate(B.lens):
        for j in range(B.rows[b]):
            r, slot = int(B.row_start[b]) + j, n_old + j
            at = (n_old if pos is None else int(pos[b])) + j
            if rot and at >= positions:
                continue
            x = f64[r].reshape(-1, dim)
            want_q[r] = pm.rotate(x[:heads], at, rot, sn, cs).reshape(-1)
            size_q[r] = np.abs(x).max()
            if B.there(b, slot):
                p, i = B.slot(b, slot)
                want_k[p, :, i], want_v[p, :, i] = pm.rotate(x[heads:heads + kv], at, rot, sn, cs), x[heads + kv:]
                size_k[p, :, i], want_w[p, :, i] = np.abs(x).max(), 0.0
    for got, want, size, to in ((out, want_q, size_q, act), (cache.k, want_k, size_k, kind), (cache.v, want_v, 0.0, kind)):
        got = got.double().cpu().numpy()
        assert np.array_equal(np.isnan(got), np.isnan(want))
        tol = pm.HALF[to] * np.abs(want) * 1.01 + 3 * 2.0 ** -24 * size + 2.0 ** -25 * (to == "f16")
        assert np.all((np.abs(got - want) <= tol) | np.isnan(want))
    assert np.array_equal(cache.weight.double().cpu().numpy(), want_w, equal_nan=True)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("seed", range(8))
def test_evict_all_at_once(pkg, kind, seed):
    """Weights of few values, NaN and infinities among them, pages that are not there, other pages' sizes, tables with room for more than the
    selection holds in LDS"""
    rng = np.random.default_rng(3000 + seed)
    n, kv, dim, page = int(rng.integers(1, 7)), int(rng.choice([1, 3])), int(rng.choice([8, 64, 72])), int(rng.choice([16, 64]))
    ld = 40000 // page if seed % 4 == 3 else None
    B = pm.Batch(seed, rng.choice([0, 1, 15, 300, 1023, 1024, 1025, 2500], n).tolist(), [0] * n, kv, dim, page, table_ld=ld, weights=True)
    if seed % 2:
        few = np.array([0.0, -0.0, 1.0, 1.0 + 2.0 ** -23, 2.0, -1.0, np.inf, -np.inf, np.nan, 1e-45])
        B.weight = np.where(np.isnan(B.weight), np.nan, rng.choice(few, B.weight.shape))
    B.table[rng.random(B.table.shape) < 0.05] = -1
    budget = int(rng.choice([1, 2, 100, 777]))
    first = int(rng.integers(0, budget + 1))
    check_evict(pkg, B, kind, budget, first, int(rng.integers(0, budget - first + 1)), page=int(rng.choice([16, 32, 128])))


@pytest.mark.parametrize("seed", range(10))
def test_verify_all_at_once(pkg, seed):
    """Batches of up to 150 sequences of up to 20 rows, some without, in tensors with more rows than the sequences have"""
    rng = np.random.default_rng(4000 + seed)
    V, draft = int(rng.choice([3, 50, 4096, 4097, 9000])), bool(rng.random() < 0.5)
    rows = np.where(rng.random(150) < 0.3, 0, rng.integers(1, 21, 150))[:int(rng.choice([1, 3, 64, 65, 150]))].tolist()
    if V > 4096:
        rows = rows[:20]
    rows[-1] = max(rows[-1], 1)
    starts, logits, other, tokens, uniform, choice = drafted(rng, rows, V, draft)
    logits[rng.random(logits.shape) < 0.2] = -np.inf
    logits[:, 0] = np.where(np.isfinite(logits).any(1), logits[:, 0], 0.0)
    temperature = float(rng.choice([0.0, 0.5, 1.0, 2.0]))
    want = pm.verify(logits, starts, tokens, uniform, choice, temperature, other)
    pad = lambda x: None if x is None else np.concatenate([x, x[:3]])  # noqa: E731
    check_verify(pkg, starts, pad(logits), pad(other), pad(tokens), pad(uniform), choice, temperature, want=want)
