"""Attention on a paged cache with queries and scales near the ends of f32, whose scores are ordinary numbers."""
import numpy as np
import pytest

import paged_model as pm
from test_gpu_paged import TYPES, dev, fill_new, held, on_gpu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act,kind", TYPES)
@pytest.mark.parametrize("size,scale", [(2.0 ** 110, 2.0 ** -113), (2.0 ** -105, 2.0 ** 102), (2.0 ** -100, 2.0 ** -100), (2.0 ** -140, 1.0), (1.0, 2.0 ** -149),
                                        (2.0 ** 100, -2.0 ** -103), (2.0 ** 118, 2.0 ** -121), (2.0 ** -112, 2.0 ** 109)])
@pytest.mark.parametrize("rows", [2, 600])
def test_far_queries_and_scales(pkg, act, kind, size, scale, rows):
    """Scores are below 8: a weight is as near as f32 products bring it, 2^-24 (64 + 8 8) and bf16's half step with bf16 rows. Queries
    of 2^-140 have few bits, and none that shows in a score."""
    B = pm.Batch(47, [90], [rows], 16, 64, 16)
    fill_new(B)
    q64, qt = held(np.clip(B.rng.standard_normal((rows, 16 * 64)), -3, 3) * size, act)
    cache, k64, v64 = on_gpu(pkg, B, kind)
    got = pkg.op_paged_attention(cache, qt, dev(B.row_start), rows, 16, scale).double().cpu().numpy()
    want, _, mass, top = pm.attend(B, q64.reshape(rows, 16, 64), k64, v64, 16, scale)
    assert top < 8
    tol = 2.0 ** -24 * (2 * (64 + 8 * top) + 700) * mass
    if act == "bf16":
        tol = tol + pm.HALF["bf16"] * (np.abs(want) + mass)
    assert np.all(np.abs(got.reshape(want.shape) - want) <= tol)
