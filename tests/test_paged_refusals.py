"""What the paged operators refuse, on the host alone: no call here gets past its checks."""
import ctypes

import pytest

EINVAL, ESHAPE, ENOTSUP = -1, -2, -4
P = 1 << 20   # an address on 16 bytes: nothing reads it


def cache(pkg, **kw):
    base = dict(d_k=P, d_v=P, d_weight=P, d_table=P, d_len=P, dtype=pkg.CACHE_BF16, n_pages=8, page=16, kv_heads=2, dim=64, n_seqs=3,
                table_ld=4)
    return pkg.PagedCacheArgs(**{**base, **kw})


def rows(pkg, **kw):
    base = dict(d_row_start=P, rows=5, max_rows=3, heads=4, act_bf16=0, d_q=P, d_out=P, ldq=256, ldo=256)
    return pkg.PagedRowsArgs(**{**base, **kw})


BAD_CACHES = [
    (dict(d_k=None), EINVAL), (dict(d_v=None), EINVAL), (dict(d_table=None), EINVAL), (dict(d_len=None), EINVAL),
    (dict(d_k=P + 8), EINVAL), (dict(d_v=P + 2), EINVAL), (dict(d_table=P + 1), EINVAL), (dict(dtype=0), EINVAL), (dict(dtype=4), EINVAL),
    (dict(n_pages=0), EINVAL), (dict(kv_heads=0), EINVAL), (dict(n_seqs=0), EINVAL), (dict(table_ld=-1), EINVAL), (dict(dim=0), EINVAL),
    (dict(page=8), ESHAPE), (dict(page=48), ESHAPE), (dict(page=-16), EINVAL), (dict(dim=60), ESHAPE), (dict(dim=264), ENOTSUP),
    (dict(table_ld=1 << 26), ESHAPE), (dict(page=1 << 30, table_ld=1), ESHAPE),
]
BAD_ROWS = [
    (dict(d_row_start=None), EINVAL), (dict(rows=0), EINVAL), (dict(max_rows=0), EINVAL), (dict(heads=0), EINVAL), (dict(heads=3), ESHAPE),
    (dict(ldq=248), EINVAL), (dict(ldo=255), EINVAL), (dict(ldq=260), EINVAL), (dict(d_q=P + 4), EINVAL), (dict(d_out=None), EINVAL),
    (dict(rows=1 << 30), ESHAPE), (dict(rows=1 << 28, max_rows=1), ESHAPE),   # rows * heads
]


def append(pkg, c, r, **kw):
    a = {**dict(k=P, ldk=128, v=P, ldv=128, pos=None, sin=P, cos=P, rot=64, table=10), **kw}
    return pkg.lib().w4a32_op_paged_append(ctypes.byref(c), ctypes.byref(r), a["k"], a["ldk"], a["v"], a["ldv"], a["pos"], a["sin"],
                                           a["cos"], a["rot"], a["table"], None)


def attend(pkg, c, r, scale=0.1, window=0, first=0, accumulate=0, scratch=P, size=1 << 40):
    return pkg.lib().w4a32_op_paged_attention(ctypes.byref(c), ctypes.byref(r), scale, window, first, accumulate, scratch, size, None)


@pytest.mark.parametrize("bad,code", BAD_CACHES)
def test_caches(pkg, bad, code):
    c, good, r = cache(pkg, **bad), cache(pkg), rows(pkg)
    assert append(pkg, c, r) == code
    assert attend(pkg, c, r) == code
    assert pkg.lib().w4a32_op_paged_attention_scratch_bytes(ctypes.byref(c), ctypes.byref(r), 0) == 0
    assert pkg.lib().w4a32_op_paged_evict_scratch_bytes(ctypes.byref(c), 16) == 0
    for a, b in ((c, good), (good, c)):
        assert pkg.lib().w4a32_op_paged_evict(ctypes.byref(a), ctypes.byref(b), 16, 0, 0, None, P, 1 << 40, None) == code


@pytest.mark.parametrize("bad,code", BAD_ROWS)
def test_rows(pkg, bad, code):
    c, r = cache(pkg), rows(pkg, **bad)
    assert append(pkg, c, r) == code
    assert attend(pkg, c, r) == code
    assert pkg.lib().w4a32_op_paged_attention_scratch_bytes(ctypes.byref(c), ctypes.byref(r), 0) == 0


def test_bf16_rows_want_a_bf16_cache(pkg):
    for dtype in (pkg.CACHE_F32, pkg.CACHE_F16):
        c, r = cache(pkg, dtype=dtype), rows(pkg, act_bf16=1)
        assert append(pkg, c, r) == ENOTSUP and attend(pkg, c, r) == ENOTSUP


@pytest.mark.parametrize("bad,code", [
    (dict(k=None), EINVAL), (dict(v=P + 4), EINVAL), (dict(ldk=120), EINVAL), (dict(ldv=130), EINVAL), (dict(rot=4), ESHAPE),
    (dict(rot=72), ESHAPE), (dict(rot=-8), ESHAPE), (dict(sin=None), EINVAL), (dict(cos=P + 4), EINVAL), (dict(table=0), EINVAL),
    (dict(pos=P + 2), EINVAL),
])
def test_append(pkg, bad, code):
    assert append(pkg, cache(pkg), rows(pkg), **bad) == code


@pytest.mark.parametrize("bad", [dict(scale=float("nan")), dict(scale=float("-inf")), dict(scale=3e38), dict(window=-1), dict(first=-1), dict(scratch=None), dict(scratch=P + 8),
                                 dict(size=0)])
def test_attention(pkg, bad):
    assert attend(pkg, cache(pkg), rows(pkg), **bad) == EINVAL


def test_attention_without_queries_weights_or_room(pkg):
    assert attend(pkg, cache(pkg), rows(pkg, d_q=None)) == EINVAL
    assert attend(pkg, cache(pkg, d_weight=None), rows(pkg), accumulate=1) == EINVAL
    c, r = cache(pkg, table_ld=64), rows(pkg)
    need = [pkg.lib().w4a32_op_paged_attention_scratch_bytes(ctypes.byref(c), ctypes.byref(r), a) for a in (0, 1)]
    assert 0 < need[0] < need[1]
    assert attend(pkg, c, r, size=need[0] - 1) == EINVAL
    assert attend(pkg, c, r, accumulate=1, size=need[1] - 1) == EINVAL


def test_evict(pkg):
    L, c, to = pkg.lib(), cache(pkg), cache(pkg, d_len=P + 64, d_table=P + 64)

    def call(c=c, to=to, budget=16, first=0, recent=0, kept=None, scratch=P, size=1 << 40):
        return L.w4a32_op_paged_evict(ctypes.byref(c), ctypes.byref(to), budget, first, recent, kept, scratch, size, None)

    assert call(budget=0) == EINVAL and call(first=-1) == EINVAL and call(recent=-1) == EINVAL
    assert call(first=10, recent=7) == ESHAPE and call(budget=65) == ESHAPE and call(first=2 ** 31 - 1, recent=2 ** 31 - 1) == ESHAPE
    assert call(scratch=None) == EINVAL and call(size=3 * 2 * 16 * 4 - 1) == EINVAL and call(kept=P + 2) == EINVAL
    assert call(c=cache(pkg, d_weight=None)) == EINVAL and call(to=cache(pkg, d_len=P + 64, d_table=P + 64, d_weight=None)) == EINVAL
    assert call(to=c) == EINVAL   # the lengths of both
    assert call(to=cache(pkg, d_len=P + 64)) == EINVAL   # the pages of both, one pool of three among them
    for pool in ("d_k", "d_v", "d_weight"):
        others = {name: P + 4096 for name in ("d_k", "d_v", "d_weight") if name != pool}
        assert call(to=cache(pkg, d_len=P + 64, **others)) == EINVAL
    many = dict(n_seqs=1 << 21, kv_heads=2, table_ld=1)
    assert call(c=cache(pkg, **many), to=cache(pkg, d_len=P + 64, d_table=P + 64, **many)) == ESHAPE
    for other in (dict(dtype=pkg.CACHE_F16), dict(dim=128), dict(kv_heads=1), dict(n_seqs=2)):
        assert call(to=cache(pkg, **{"d_len": P + 64, "d_table": P + 64, **other})) == ESHAPE


def test_verify(pkg):
    L = pkg.lib()
    base = dict(d_logits=P, d_draft=P, d_row_start=P, d_tokens=P, d_uniform=P, d_choice=P, d_count=P, d_next=P, d_len=P, rows=6, max_rows=3,
                n_seqs=2, vocab=1000, ldl=1000, ldd=1000, temperature=1.0)

    def call(scratch=P, size=1 << 40, **kw):
        return L.w4a32_op_verify_drafts(ctypes.byref(pkg.VerifyArgs(**{**base, **kw})), scratch, size, None)

    for bad in (dict(d_logits=None), dict(d_row_start=None), dict(d_tokens=None), dict(d_count=None), dict(d_next=None), dict(d_uniform=None),
                dict(d_choice=None), dict(rows=0), dict(max_rows=0), dict(n_seqs=0), dict(vocab=0), dict(ldl=999), dict(ldd=999),
                dict(temperature=-1.0), dict(temperature=float("nan")), dict(temperature=float("inf")), dict(d_logits=P + 2),
                dict(d_tokens=P + 4), dict(d_next=P + 4), dict(d_count=P + 1), dict(scratch=None), dict(scratch=P + 8), dict(size=0),
                dict(size=L.w4a32_op_verify_drafts_scratch_bytes(6, 1000, 2) - 1)):
        assert call(**bad) == EINVAL, bad
    assert call(rows=1 << 30) == ESHAPE and call(vocab=1 << 30, ldl=1 << 30, ldd=1 << 30) == ESHAPE
    for sizes in ((0, 10, 1), (1, 0, 1), (1, 10, 0), (1 << 30, 10, 1), (1 << 20, 1 << 29, 1), (1 << 20, 4096 * 16, 1),
                  (1, 4096 * 8, 1 << 20)):
        assert L.w4a32_op_verify_drafts_scratch_bytes(*sizes) == 0
