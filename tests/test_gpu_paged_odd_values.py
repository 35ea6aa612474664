"""Attention on a paged cache where values, queries or keys are not finite: results as the formula has them, wherever the tiles' borders are."""
import numpy as np
import pytest
import torch

import paged_model as pm
from test_gpu_paged import TYPES, dev, fill_new, held, on_gpu

pytestmark = pytest.mark.gpu


def alike(got, want, tol):
    """NaN where NaN is, infinities of the same sign, and the rest near"""
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(np.where(np.isinf(got), np.sign(got), 0), np.where(np.isinf(want), np.sign(want), 0))
    ok = np.isfinite(want)
    assert np.all(np.abs(got[ok] - want[ok]) <= tol)


# (kv heads, query heads, dim, page, tokens, rows, table's pages, sequences without rows)
SHAPES = [
    (2, 12, 128, 16, 300, 1, None, 0),      # one row: tiles seen whole, shared by workgroups
    (1, 4, 64, 32, 70, 4, None, 0),         # a few, not shared
    (2, 4, 256, 16, 900, 2, 4096, 0),       # on a table with room
    (2, 14, 72, 16, 300, 9, None, 2),       # four wavefronts' rows
    (16, 16, 64, 16, 90, 400, None, 0),     # a prompt, 32 rows of a workgroup
    (8, 16, 128, 32, 200, 270, None, 0),
    (8, 16, 256, 64, 100, 270, None, 0),
    (8, 8, 80, 32, 200, 300, None, 40),     # 256 rows of a workgroup, or 128
    (8, 8, 64, 16, 300, 400, None, 40),
    (8, 8, 256, 64, 100, 270, None, 40),
]


@pytest.mark.parametrize("act,kind", TYPES)
@pytest.mark.parametrize("kv,heads,dim,page,length,rows,ld,empty", SHAPES)
def test_infinite_values_wherever_they_lie(pkg, act, kind, kv, heads, dim, page, length, rows, ld, empty):
    """Among them two of either sign for one dimension, and one of a token with next to no weight (2^-300 of the row's largest)"""
    B = pm.Batch(41, [length] + [3] * empty, [rows] + [0] * empty, kv, dim, page, table_ld=ld)
    fill_new(B)
    odd = [(2, 1, np.inf), (33, 3, -np.inf), (length // 2, 5, np.nan), (length - 9, 6, np.inf), (length - 1, 7, -np.inf), (5, 8 % dim, np.inf),
           (length // 2, 8 % dim, -np.inf), (length + rows - 1, 9 % dim, np.inf)]
    for t, d, x in odd:
        p, i = B.slot(0, t)
        B.v[p, :, i, d % dim] = x
    far, other = 20, 10 % dim
    p, i = B.slot(0, far)
    B.v[p, :, i, other] = np.inf
    q = B.rng.standard_normal((rows, heads, dim)) * 0.5
    q[:, :, 0] = 16.0
    B.k[p, :, i, 0] = -13.0 * dim ** 0.5      # a score of 208 less than the others'
    q64, qt = held(q.reshape(rows, -1), act)
    cache, k64, v64 = on_gpu(pkg, B, kind)
    for window, first in ((0, 0), (37, 21)):
        got = pkg.op_paged_attention(cache, qt, dev(B.row_start), rows, heads, dim ** -0.5, window=window, first=first)
        want = pm.attend(B, q64.reshape(rows, heads, dim), k64, v64, heads, dim ** -0.5, window, first)[0].reshape(rows, -1)
        assert np.isinf(want).any() and np.isfinite(want).any() and (window or np.isnan(want).any())
        alike(got.double().cpu().numpy(), want, 2 ** -5 if act == "bf16" else 1e-4)


@pytest.mark.parametrize("act,kind", TYPES)
def test_an_infinite_value_of_a_share_without_weight(pkg, act, kind):
    """One sequence that many workgroups share; all the weight lies in the last tokens, 2^-600 of it where the infinity is"""
    kv, heads, dim, length = 1, 2, 64, 4000
    B = pm.Batch(42, [length], [1], kv, dim, 16)
    fill_new(B)
    for t in range(length + 1):
        p, i = B.slot(0, t)
        B.k[p, :, i] *= 0.25
        B.k[p, :, i, 0] = 26.0 * t / length
    for t, d, x in ((3, 4, np.inf), (1500, 5, -np.inf), (3990, 6, np.inf)):
        p, i = B.slot(0, t)
        B.v[p, 0, i, d] = x
    q = B.rng.standard_normal((1, heads, dim)) * 0.25
    q[:, :, 0] = 128.0
    q64, qt = held(q.reshape(1, -1), act)
    cache, k64, v64 = on_gpu(pkg, B, kind)
    got = pkg.op_paged_attention(cache, qt, dev(B.row_start), 1, heads, dim ** -0.5)
    want = pm.attend(B, q64.reshape(1, heads, dim), k64, v64, heads, dim ** -0.5)[0].reshape(1, -1)
    assert np.isinf(want).sum() == 3 * heads
    alike(got.double().cpu().numpy(), want, 2 ** -5 if act == "bf16" else 1e-3)
