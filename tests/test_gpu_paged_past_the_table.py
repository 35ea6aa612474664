"""Rows that stand behind the last token their sequence's table has room for: they see what their own places let them see."""
import numpy as np
import pytest
import torch

import paged_model as pm
from test_gpu_paged import TYPES, dev, fill_new, on_gpu, run_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act,kind", TYPES)
@pytest.mark.parametrize("window,first", [(0, 0), (1, 0), (3, 2), (9, 0), (40, 17), (2 ** 31 - 1, 0)])
@pytest.mark.parametrize("kv,heads,dim,page,ld,lens,rows", [
    (2, 6, 64, 16, 4, [60, 64, 20, 75], [8, 3, 2, 1]),                # 64 slots; the second and the fourth have none left
    (1, 2, 128, 16, 3, [45], [7]),                                    # an odd number of half tiles
    (16, 16, 64, 16, 16, [90, 300], [250, 40]),                       # prompts, to the slots 339 of 256
    (8, 16, 128, 32, 16, [290, 500], [300, 100]),                     # 599 of 512
    (8, 8, 256, 16, 30, [100], [500]),
    (8, 8, 128, 32, 16, [290, 500] + [9] * 40, [300, 100] + [0] * 40),   # more rows of a workgroup
])
def test_windows(pkg, act, kind, window, first, kv, heads, dim, page, ld, lens, rows):
    B = pm.Batch(44, lens, rows, kv, dim, page, table_ld=ld)
    fill_new(B)
    run_attention(pkg, B, act, kind, heads, window, first)


@pytest.mark.parametrize("act,kind", TYPES)
@pytest.mark.parametrize("window,first", [(3, 2), (40, 17)])
def test_weights(pkg, act, kind, window, first):
    B = pm.Batch(45, [60, 64, 20, 75], [8, 3, 2, 1], 2, 64, 16, table_ld=4, weights=True)
    fill_new(B)
    run_attention(pkg, B, act, kind, 6, window, first, accumulate=True)


def test_queries_are_rotated_to_their_own_positions(pkg):
    """A sequence of 100 tokens on a table for 32: nothing is written, and its queries stand at 100 and 101"""
    B = pm.Batch(46, [100], [2], 1, 64, 16, table_ld=2)
    cache, _, _ = on_gpu(pkg, B, "f32")
    q, k, v = (torch.randn(2, 64, device="cuda") for _ in range(3))
    sin, cos = pkg.op_rope_table(128, 64, 1e4)
    before = torch.nan_to_num(cache.k, nan=-1.0)
    got = pkg.op_paged_append(cache, q, k, v, dev(B.row_start), sin, cos).double().cpu().numpy()
    assert torch.equal(torch.nan_to_num(cache.k, nan=-1.0), before)
    for j in range(2):
        x = q[j].double().cpu().numpy()[None]
        want = pm.rotate(x, 100 + j, 64, sin.cpu().numpy(), cos.cpu().numpy())[0]
        assert np.all(np.abs(got[j] - want) <= 3 * 2.0 ** -24 * np.abs(x).max() + 2.0 ** -24 * np.abs(want))
