"""What forking, copying and compacting pages refuse, on the host alone: no call here gets past its checks."""
import ctypes

import pytest

from test_paged_refusals import BAD_CACHES, EINVAL, ESHAPE, P, cache


def fork(pkg, c, scratch=P, size=1 << 40, **kw):
    base = dict(d_parent=P, d_keep=P, d_row_start=P, d_refs=P, d_moves=P, d_counts=P, rows=5, max_rows=3)
    a = pkg.ForkArgs(**{**base, **kw})
    return pkg.lib().w4a32_op_paged_fork(ctypes.byref(c), ctypes.byref(a), scratch, size, None)


def copy(pkg, caches, moves=P, count=P, most=4, n=None):
    refs = (ctypes.c_void_p * max(1, len(caches)))(*[ctypes.addressof(c) for c in caches])
    return pkg.lib().w4a32_op_paged_copy(refs, len(caches) if n is None else n, moves, count, most, None)


def compact(pkg, c, refs=P, moves=P, counts=P, scratch=P, size=1 << 40):
    return pkg.lib().w4a32_op_paged_compact(ctypes.byref(c), refs, moves, counts, scratch, size, None)


@pytest.mark.parametrize("bad,code", BAD_CACHES)
def test_caches(pkg, bad, code):
    c, L = cache(pkg, **bad), pkg.lib()
    assert fork(pkg, c) == code and compact(pkg, c) == code
    assert copy(pkg, [c]) == code and copy(pkg, [cache(pkg), c]) == code
    assert L.w4a32_op_paged_fork_scratch_bytes(ctypes.byref(c), 5) == 0 == L.w4a32_op_paged_compact_scratch_bytes(ctypes.byref(c))


@pytest.mark.parametrize("bad", [dict(d_refs=None), dict(d_moves=None), dict(d_counts=None), dict(d_refs=P + 2), dict(d_moves=P + 1), dict(d_counts=P + 2),
                                 dict(d_parent=P + 2), dict(d_keep=P + 1), dict(d_row_start=P + 2), dict(rows=0), dict(max_rows=0), dict(rows=-1),
                                 dict(scratch=None), dict(scratch=P + 8), dict(size=0)])
def test_fork(pkg, bad):
    assert fork(pkg, cache(pkg), **bad) == EINVAL


def test_fork_of_sizes_that_are_too_large(pkg):
    L = pkg.lib()
    assert fork(pkg, cache(pkg), rows=1 << 30) == ESHAPE
    for bad in (dict(n_seqs=1 << 14, table_ld=(1 << 12) + 1), dict(n_pages=(1 << 26) + 1, kv_heads=1)):
        c = cache(pkg, **bad)
        assert fork(pkg, c) == ESHAPE and compact(pkg, c) == ESHAPE
        assert L.w4a32_op_paged_fork_scratch_bytes(ctypes.byref(c), 5) == 0 == L.w4a32_op_paged_compact_scratch_bytes(ctypes.byref(c))
    c = cache(pkg)
    assert L.w4a32_op_paged_fork_scratch_bytes(ctypes.byref(c), -1) == 0 == L.w4a32_op_paged_fork_scratch_bytes(ctypes.byref(c), 1 << 30)
    need = L.w4a32_op_paged_fork_scratch_bytes(ctypes.byref(c), 5)
    assert 0 < L.w4a32_op_paged_fork_scratch_bytes(ctypes.byref(c), 0) <= need and fork(pkg, c, size=need - 1) == EINVAL


@pytest.mark.parametrize("bad", [dict(moves=None), dict(count=None), dict(moves=P + 2), dict(count=P + 1), dict(most=0), dict(most=-3), dict(n=0), dict(n=-1)])
def test_copy(pkg, bad):
    assert copy(pkg, [cache(pkg)], **bad) == EINVAL


@pytest.mark.parametrize("other", [dict(dtype=1), dict(n_pages=9), dict(page=32), dict(kv_heads=1), dict(dim=72), dict(d_weight=None)])
def test_copy_in_caches_of_other_sizes(pkg, other):
    assert copy(pkg, [cache(pkg), cache(pkg), cache(pkg, **other)]) == ESHAPE


def test_copy_without_caches_and_of_a_page_that_is_too_large(pkg):
    assert pkg.lib().w4a32_op_paged_copy(None, 1, P, P, 4, None) == EINVAL
    assert copy(pkg, [cache(pkg, page=1 << 20, table_ld=1, dim=256, kv_heads=8)]) == ESHAPE


@pytest.mark.parametrize("bad", [dict(refs=None), dict(moves=None), dict(counts=None), dict(refs=P + 2), dict(moves=P + 1), dict(counts=P + 2),
                                 dict(scratch=None), dict(scratch=P + 8), dict(size=0)])
def test_compact(pkg, bad):
    assert compact(pkg, cache(pkg), **bad) == EINVAL


def test_compact_without_room(pkg):
    c = cache(pkg)
    need = pkg.lib().w4a32_op_paged_compact_scratch_bytes(ctypes.byref(c))
    assert need > 0 and compact(pkg, c, size=need - 1) == EINVAL
