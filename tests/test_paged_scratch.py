"""How much scratch memory attention with added-up weights asks for, on the host alone."""
import ctypes

import pytest

from test_paged_refusals import P, attend, cache, rows

GIB = 1 << 30


def need(pkg, c, r, window=None, first=0, accumulate=1):
    c, r = ctypes.byref(c), ctypes.byref(r)
    if window is None:
        return pkg.lib().w4a32_op_paged_attention_scratch_bytes(c, r, accumulate)
    return pkg.lib().w4a32_op_paged_attention_window_scratch_bytes(c, r, window, first, accumulate)


def batch(pkg, tokens, n_seqs, n_rows, most, heads=28, kv=4, dim=128, dtype=None):
    c = cache(pkg, table_ld=tokens // 64, page=64, n_pages=1 << 16, n_seqs=n_seqs, kv_heads=kv, dim=dim, dtype=dtype or pkg.CACHE_BF16)
    return c, rows(pkg, rows=n_rows, max_rows=most, heads=heads, ldq=heads * dim, ldo=heads * dim)


@pytest.mark.parametrize("tokens,n_seqs,n_rows", [(8192, 1, 8192), (16384, 1, 16384), (65536, 1, 65536), (131072, 1, 2048), (16384, 8, 6000)])
def test_weights_of_a_long_prompt_go_by_passes(pkg, tokens, n_seqs, n_rows):
    """A pass of 128 rows and 28 heads on 131072 tokens: 14 + 1 items of 64 rows, 4 kv heads, 64 x 4 x 131072 bytes; the rest is sums"""
    size = need(pkg, *batch(pkg, tokens, n_seqs, n_rows, n_rows))
    assert 0 < size < 2.2 * GIB


@pytest.mark.parametrize("window,first", [(1, 0), (1024, 4), (100000, 500), (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("tokens,n_seqs,n_rows,most", [(131072, 1, 512, 512), (131072, 64, 320, 5), (1024, 3, 5, 3), (131072, 16, 4000, 900), (65536, 1, 65536, 65536)])
@pytest.mark.parametrize("accumulate", [0, 1])
def test_a_window_takes_no_more_than_none(pkg, window, first, tokens, n_seqs, n_rows, most, accumulate):
    """And scratch memory for any window serves each one: a call that gets that far is refused for less alone"""
    c, r = batch(pkg, tokens, n_seqs, n_rows, most, heads=12, kv=2)
    every, one = need(pkg, c, r, accumulate=accumulate), need(pkg, c, r, window, first, accumulate)
    assert 0 < one and need(pkg, c, r, 0, 0, accumulate) == every
    assert attend(pkg, c, r, window=window, first=first, accumulate=accumulate, size=255) == -1
    if n_rows <= 512:
        assert one <= every
    if (window, tokens, n_rows, accumulate) == (1024, 131072, 512, 1):
        assert one < GIB / 8 < every   # 98 items x 51 tiles x 8 KB, and 33 MB of sums that shares leave


def test_a_window_is_enough_where_all_tokens_are_too_many(pkg):
    """20000 sequences with room for a million tokens: 2^15 tiles each for 4 kv heads, of which a window has 35"""
    c, r = batch(pkg, 1 << 20, 20000, 20000, 1)
    assert need(pkg, c, r, accumulate=0) == 0 and attend(pkg, c, r) == -2
    assert 0 < need(pkg, c, r, 1024, 4, accumulate=0) < GIB
    for bad in ((-1, 0), (0, -1)):
        assert need(pkg, c, r, *bad) == 0


def test_which_prompts_share_their_keys(pkg):
    """The prompts' kernel takes next to no scratch memory, the rows' kernel room for the shares' sums. 256 dims of f32 rows on a bf16 cache,
    16 heads on 4: the former for a prompt alone, through a small window, or of many rows; the latter on a long context"""
    def size(tokens, n, window=0, act=0, dtype=None):
        c, r = batch(pkg, tokens, 1, n, n, heads=16, kv=4, dim=256, dtype=dtype)
        r.act_bf16 = act
        return need(pkg, c, r, window, 4, accumulate=0)
    assert size(512, 512) == size(832, 800) == size(1280, 1024) == size(4608, 512, 500) == size(6144, 2048) == 256
    assert size(4608, 512) > 1 << 20 and size(5120, 1024) > 1 << 20 and size(4608, 512, 1000) > 1 << 20
    assert size(4608, 512, act=1) == size(4608, 512, dtype=pkg.CACHE_F16) == 256
