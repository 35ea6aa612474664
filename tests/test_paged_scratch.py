"""How much scratch memory attention with added-up weights asks for, on the host alone."""
import ctypes

import pytest

from test_paged_refusals import cache, rows

GIB = 1 << 30


def need(pkg, c, r, accumulate=1):
    return pkg.lib().w4a32_op_paged_attention_scratch_bytes(ctypes.byref(c), ctypes.byref(r), accumulate)


def batch(pkg, tokens, n_seqs, n_rows, most, heads=28, kv=4, dim=128, dtype=None):
    c = cache(pkg, table_ld=tokens // 64, page=64, n_pages=1 << 16, n_seqs=n_seqs, kv_heads=kv, dim=dim, dtype=dtype or pkg.CACHE_BF16)
    return c, rows(pkg, rows=n_rows, max_rows=most, heads=heads, ldq=heads * dim, ldo=heads * dim)


@pytest.mark.parametrize("tokens,n_seqs,n_rows", [(8192, 1, 8192), (16384, 1, 16384), (65536, 1, 65536), (131072, 1, 2048), (16384, 8, 6000)])
def test_weights_of_a_long_prompt_go_by_passes(pkg, tokens, n_seqs, n_rows):
    """A pass of 128 rows and 28 heads on 131072 tokens: 14 + 1 items of 64 rows, 4 kv heads, 64 x 4 x 131072 bytes; the rest is sums"""
    size = need(pkg, *batch(pkg, tokens, n_seqs, n_rows, n_rows))
    assert 0 < size < 2.2 * GIB
