"""What attention of sequences that share prefixes refuses, on the host alone: no call here gets past its checks."""
import ctypes

import pytest

from test_paged_refusals import BAD_CACHES, BAD_ROWS, EINVAL, ENOTSUP, ESHAPE, P, cache, rows


def attend(pkg, c, r, scale=0.1, starts=P, prefix=P, groups=2, scratch=P, size=1 << 50):
    return pkg.lib().w4a32_op_paged_prefix_attention(ctypes.byref(c), ctypes.byref(r), scale, starts, prefix, groups, scratch, size, None)


def need(pkg, c, r, groups=2):
    return pkg.lib().w4a32_op_paged_prefix_attention_scratch_bytes(ctypes.byref(c), ctypes.byref(r), groups)


@pytest.mark.parametrize("bad,code", BAD_CACHES)
def test_caches(pkg, bad, code):
    c = cache(pkg, **bad)
    assert attend(pkg, c, rows(pkg)) == code and need(pkg, c, rows(pkg)) == 0


@pytest.mark.parametrize("bad,code", BAD_ROWS)
def test_rows(pkg, bad, code):
    r = rows(pkg, **bad)
    assert attend(pkg, cache(pkg), r) == code and need(pkg, cache(pkg), r) == 0


@pytest.mark.parametrize("bad", [dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=3e38), dict(starts=None), dict(prefix=None), dict(starts=P + 2),
                                 dict(prefix=P + 1), dict(groups=0), dict(groups=-1), dict(scratch=None), dict(scratch=P + 8), dict(size=0)])
def test_arguments(pkg, bad):
    assert attend(pkg, cache(pkg), rows(pkg), **bad) == EINVAL


def test_more(pkg):
    assert attend(pkg, cache(pkg), rows(pkg), groups=4) == ESHAPE and need(pkg, cache(pkg), rows(pkg), 4) == 0   # of three sequences
    assert attend(pkg, cache(pkg), rows(pkg, d_q=None)) == EINVAL
    for dtype in (pkg.CACHE_F32, pkg.CACHE_F16):
        assert attend(pkg, cache(pkg, dtype=dtype), rows(pkg, act_bf16=1)) == ENOTSUP
    size = need(pkg, cache(pkg), rows(pkg))
    assert size > 0 and attend(pkg, cache(pkg), rows(pkg), size=size - 1) == EINVAL
