"""The operators of a batch of sequences on a paged cache against their definitions in 64 bits."""
import numpy as np
import pytest
import torch

import paged_model as pm

pytestmark = pytest.mark.gpu

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TYPES = [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("bf16", "bf16")]


def dev(a, kind=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if kind is None else t.to(TORCH[kind])


def held(a, kind):
    """the values that a tensor of this type holds, in 64 bits, and the tensor"""
    t = dev(a, kind)
    return t.double().cpu().numpy(), t


def on_gpu(pkg, B, kind):
    k64, k = held(B.k, kind)
    v64, v = held(B.v, kind)
    w = None if B.weight is None else dev(B.weight, "f32")
    cache = pkg.PagedCache(k, v, dev(B.table), dev(np.array(B.lens, np.int32)), w)
    return cache, k64, v64


def fill_new(B):
    """Tokens of the step's own rows, as an append would have left them"""
    for b, n in enumerate(B.lens):
        for t in range(n, n + B.rows[b]):
            if B.there(b, t):
                p, i = B.slot(b, t)
                B.k[p, :, i], B.v[p, :, i] = B.rng.standard_normal((B.kv, B.dim)), B.rng.standard_normal((B.kv, B.dim))
                if B.weight is not None:
                    B.weight[p, :, i] = 0.0


def near(got, want, mass, act, cache, top, dim, keys):
    """Elementwise: a score is off by its f32 sum of `dim` products (dim half steps of what is summed, of which |s| is all but
    the cancelled part; 8 |top| stands for it) and a weight by e to that and by the sums over `keys` weights; with bf16 rows a
    weight is rounded to bf16 (half a step) before it meets the value, and the result after."""
    e = 2.0 ** -24
    rel = 2 * e * (dim + 8 * top) + e * (keys + 16)
    tol = rel * mass + 1e-30
    if act == "bf16":
        tol = tol + pm.HALF["bf16"] * (np.abs(want) + mass)
    d = np.abs(got - want)
    assert np.all(d <= tol), f"off by {d.max()} where {tol.flat[d.argmax()]} is allowed"
    if act == "f32":   # and together: roundings of either sign, so that their squares add up
        assert np.linalg.norm(got - want) <= 4 * e * (8 + top) * max(np.linalg.norm(mass), 1e-30)


def run_attention(pkg, B, act, kind, heads, window=0, first=0, accumulate=False, max_rows=None, pad_rows=0, stride=0, scale=None,
                  scratch=None):
    q = B.rng.standard_normal((B.total + pad_rows, heads * B.dim + stride)) * 2.0
    q64, qt = held(q, act)
    q64 = q64[:, :heads * B.dim].reshape(-1, heads, B.dim)[:B.total]
    qt = qt[:, :heads * B.dim]
    cache, k64, v64 = on_gpu(pkg, B, kind)
    scale = B.dim ** -0.5 if scale is None else scale
    out = torch.full((B.total + pad_rows, heads * B.dim), 7.5, dtype=qt.dtype, device="cuda")
    got = pkg.op_paged_attention(cache, qt, dev(B.row_start), max_rows or max(1, max(B.rows)), heads, scale, window=window, first=first,
                                 accumulate=accumulate, out=out, scratch=scratch)
    torch.cuda.synchronize()
    want, added, mass, top = pm.attend(B, q64, k64, v64, heads, scale, window, first)
    got = got.double().cpu().numpy()
    assert np.all(got[B.total:] == 7.5)
    near(got[:B.total].reshape(-1, heads, B.dim), want, mass, act, kind, top, B.dim, max(n + r for n, r in zip(B.lens, B.rows)))
    if accumulate:
        w = cache.weight.double().cpu().numpy()
        old = B.weight.astype(np.float32).astype(np.float64)
        there = ~np.isnan(old)
        assert np.array_equal(np.isnan(w), ~there)
        tol = added[there] * 2.0 ** -24 * (2 * B.dim + 16 * top + 64) + 2.0 ** -23 * old[there] + 1e-12
        assert np.all(np.abs(w[there] - old[there] - added[there]) <= tol)


@pytest.mark.parametrize("act,kind", TYPES)
@pytest.mark.parametrize("heads,kv,dim,page,lens,rows", [
    (12, 2, 128, 16, [200], [1]),
    (1, 1, 64, 16, [0], [1]),                                   # a first token sees itself alone
    (7, 1, 128, 32, [5, 31, 32, 33, 0, 64], [1, 1, 1, 1, 1, 1]),  # lengths about a tile's border
    (8, 8, 64, 64, [100, 3], [1, 2]),                           # a head of its own for every query head
    (6, 2, 80, 16, [47, 129], [3, 1]),
    (4, 2, 256, 128, [130, 17, 255], [1, 4, 1]),
    (34, 2, 72, 32, [70, 9], [2, 1]),                           # a group that does not fit into 16 rows
    (4, 1, 8, 16, [40], [2]),
    (6, 2, 96, 16, [0, 60, 3], [37, 0, 21]),                    # prompts, and a sequence without rows
])
def test_attention(pkg, act, kind, heads, kv, dim, page, lens, rows):
    B = pm.Batch(1, lens, rows, kv, dim, page)
    fill_new(B)
    run_attention(pkg, B, act, kind, heads)


@pytest.mark.parametrize("act,kind", TYPES)
@pytest.mark.parametrize("heads,kv,dim,page,lens,rows", [
    (14, 2, 128, 32, [5, 31, 300, 33, 0, 64], [1, 4, 3, 1, 2, 0]),   # up to 28 rows of a kv head: two wavefronts'
    (12, 2, 64, 16, [70, 9, 400], [9, 2, 17]),                      # four
    (34, 2, 72, 32, [70, 9], [2, 1]),
    (4, 2, 256, 128, [130, 17, 255], [1, 14, 1]),
])
def test_attention_on_a_long_table(pkg, act, kind, heads, kv, dim, page, lens, rows):
    """Room for so many tokens that a workgroup has 32 or 64 rows"""
    B = pm.Batch(34, lens, rows, kv, dim, page, table_ld=65536 // page, weights=True)
    fill_new(B)
    run_attention(pkg, B, act, kind, heads)
    run_attention(pkg, B, act, kind, heads, window=60, first=3, accumulate=True)


@pytest.mark.parametrize("act,kind", TYPES)
@pytest.mark.parametrize("heads,kv,dim,page,lens,rows,window,first", [
    # few workgroups, so of 32 rows: all sequences alike; beside sequences that are not the prompts' kernel's; odd sizes, windows
    (8, 8, 128, 32, [0, 70], [600, 601], 0, 0),
    (14, 2, 64, 16, [33, 200, 5, 0], [700, 3, 1, 450], 0, 0),
    (16, 8, 80, 64, [100, 0], [257, 333], 50, 5),
    (8, 8, 256, 16, [31], [700], 200, 40),
    (12, 12, 8, 128, [0], [1100], 0, 0),
    (7, 7, 96, 16, [130, 0], [450, 449], 1, 0),
    # workgroups of 256 or 128 rows (sequences without rows count among its workgroups)
    (8, 8, 128, 32, [0, 70] + [9] * 40, [300, 401] + [0] * 40, 0, 0),
    (14, 2, 64, 16, [33, 200, 5, 0] + [3] * 140, [300, 3, 1, 250] + [0] * 140, 0, 0),
    (16, 8, 80, 64, [100, 0] + [3] * 40, [257, 333] + [1] * 20 + [0] * 20, 50, 5),
    (8, 8, 256, 16, [31] + [0] * 40, [400] + [0] * 40, 200, 40),
    (8, 8, 8, 128, [0] + [0] * 70, [500] + [2] * 70, 0, 0),   # more sequences than a wavefront has lanes
    (7, 7, 96, 16, [130, 0] + [40] * 40, [350, 449] + [0] * 40, 1, 0),
])
def test_prompts(pkg, act, kind, heads, kv, dim, page, lens, rows, window, first):
    B = pm.Batch(25, lens, rows, kv, dim, page)
    fill_new(B)
    run_attention(pkg, B, act, kind, heads, window, first, pad_rows=3, stride=16)


@pytest.mark.parametrize("act,kind", TYPES)
@pytest.mark.parametrize("heads,kv,dim,page,lens,rows,window,first", [
    # rows of one token and prompts where the table has room for so many tokens that they are two kernels'
    (14, 2, 64, 16, [33, 2600, 5, 0], [700, 3, 1, 450], 0, 0),
    (8, 8, 128, 32, [0, 70] + [9] * 40, [300, 401] + [2] * 40, 0, 0),
    (16, 8, 80, 64, [100, 0, 2800], [257, 333, 1], 2700, 5),
    (8, 8, 256, 16, [31, 200], [700, 5], 0, 0),
])
def test_prompts_beside_few_rows_on_long_tables(pkg, act, kind, heads, kv, dim, page, lens, rows, window, first):
    B = pm.Batch(33, lens, rows, kv, dim, page, table_ld=3200 // page)
    fill_new(B)
    run_attention(pkg, B, act, kind, heads, window, first, pad_rows=3, stride=16)


@pytest.mark.parametrize("act,kind", TYPES)
@pytest.mark.parametrize("many", [0, 20])
def test_prompts_with_missing_pages_and_odd_values(pkg, act, kind, many):
    many = many * [3]
    B = pm.Batch(26, [90, 40] + many, [500, 400] + [0] * len(many), 16, 64, 16)
    fill_new(B)
    B.table[0, 3], B.table[0, 20], B.table[1, 0] = -1, B.n_pages + 7, -2 ** 31
    run_attention(pkg, B, act, kind, 16)
    run_attention(pkg, B, act, kind, 16, window=100, first=70)
    for bad, t in ((np.inf, 200), (np.nan, 89), (-np.inf, 10)):
        B = pm.Batch(27, [90] + many, [600] + [0] * len(many), 16, 64, 16)
        fill_new(B)
        p, i = B.slot(0, t)
        B.v[p, 5, i, 7] = bad
        q64, q = held(B.rng.standard_normal((600, 16 * 64)), act)
        cache, k64, v64 = on_gpu(pkg, B, kind)
        for window, first in ((0, 0), (64, 4)):
            got = pkg.op_paged_attention(cache, q, dev(B.row_start), 600, 16, 0.125, window=window, first=first).double().cpu().numpy()
            want = pm.attend(B, q64.reshape(600, 16, 64), k64, v64, 16, 0.125, window, first)[0].reshape(600, -1)
            ok = np.isfinite(want)
            assert np.array_equal(np.isfinite(got), ok)
            assert np.all(np.abs(got[ok] - want[ok]) <= (2 ** -6 if act == "bf16" else 1e-5))


def test_a_padded_prompt_that_turns_out_short(pkg):
    """Buffers and max_rows for 900 rows, of which the device says there are 2, then none"""
    B = pm.Batch(28, [50], [2], 16, 64, 16)
    fill_new(B)
    q = torch.randn(900, 16 * 64, device="cuda")
    cache, k64, v64 = on_gpu(pkg, B, "bf16")
    for rows in (2, 0):
        out = torch.full_like(q, 7.5)
        pkg.op_paged_attention(cache, q, dev(np.array([0, rows], np.int32)), 900, 16, 0.125, out=out)
        got = out.double().cpu().numpy()
        assert np.all(got[rows:] == 7.5)
        B.total, B.rows = rows, [rows]
        want = pm.attend(B, q.double().cpu().numpy().reshape(900, 16, 64), k64, v64, 16, 0.125)[0].reshape(rows, 1024)
        assert np.all(np.abs(got[:rows] - want) <= 1e-5)


@pytest.mark.parametrize("act,kind", TYPES)
@pytest.mark.parametrize("window,first", [(1, 0), (1, 1), (5, 2), (16, 4), (33, 37), (64, 500), (100000, 3), (2 ** 31 - 1, 2 ** 31 - 1)])
def test_window_and_first_tokens(pkg, act, kind, window, first):
    B = pm.Batch(2, [150, 31, 0, 64, 90], [1, 3, 5, 0, 2], 2, 64, 16)
    fill_new(B)
    run_attention(pkg, B, act, kind, 6, window, first)


@pytest.mark.parametrize("act,kind", TYPES)
def test_long_sequences_are_split_and_joined(pkg, act, kind):
    B = pm.Batch(3, [2100, 40, 701], [1, 2, 1], 2, 128, 32, std_k=1.5)
    fill_new(B)
    run_attention(pkg, B, act, kind, 6)


@pytest.mark.parametrize("act,kind", TYPES)
@pytest.mark.parametrize("window,first", [(0, 0), (40, 3)])
def test_weights_are_added_up(pkg, act, kind, window, first):
    B = pm.Batch(4, [300, 17, 0, 96, 1500], [2, 4, 3, 0, 1], 2, 64, 32, weights=True)
    fill_new(B)
    run_attention(pkg, B, act, kind, 14, window, first, accumulate=True)


@pytest.mark.parametrize("act,kind", TYPES)
def test_rows_of_a_wider_tensor_and_a_padded_batch(pkg, act, kind):
    B = pm.Batch(5, [33, 90], [2, 1], 1, 64, 16)
    fill_new(B)
    run_attention(pkg, B, act, kind, 4, pad_rows=5, stride=48, max_rows=9)


@pytest.mark.parametrize("act,kind", TYPES)
def test_pages_that_are_not_there_are_not_seen(pkg, act, kind):
    B = pm.Batch(6, [200, 77, 40], [2, 1, 1], 2, 64, 16)
    fill_new(B)
    B.table[0, 1], B.table[0, 7], B.table[0, 8] = -1, B.n_pages, 2 ** 31 - 1
    B.table[1, :] = -5          # a sequence that sees nothing
    B.table[2, 0] = -2 ** 31
    run_attention(pkg, B, act, kind, 4)
    run_attention(pkg, B, act, kind, 4, window=30, first=20)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_a_length_past_the_table_and_rows_past_their_number(pkg, kind):
    B = pm.Batch(7, [40, 10, 20], [1, 3, 2], 1, 64, 16, table_ld=3)
    fill_new(B)
    q = B.rng.standard_normal((B.total, 128)).astype(np.float32)
    lens = np.array([2 ** 31 - 1, -7, 20], np.int32)   # clamped: 48 tokens (all there are), none, 20
    B.k, B.v = np.nan_to_num(B.k), np.nan_to_num(B.v)
    k64, k = held(B.k, kind)
    v64, v = held(B.v, kind)
    cache = pkg.PagedCache(k, v, dev(B.table), dev(lens))
    out = torch.full((B.total, 128), 3.0, device="cuda")
    pkg.op_paged_attention(cache, dev(q), dev(B.row_start), 2, 2, 0.125, out=out)
    torch.cuda.synchronize()
    got = out.double().cpu().numpy()
    assert np.all(got[3] == 3.0)   # the third row of a sequence that has at most two
    B.lens, B.rows = [47, 0, 20], [1, 3, 2]
    want, _, mass, top = pm.attend(B, q.astype(np.float64).reshape(-1, 2, 64), k64, v64, 2, 0.125)
    sel = [0, 1, 2, 4, 5]
    near(got[sel].reshape(-1, 2, 64), want[sel], mass[sel], "f32", kind, top, 64, 48)


@pytest.mark.parametrize("starts", [[0, 9, -4, 2], [6, 3, 100, 1], [0, 6, 0, 6], [2 ** 31 - 1, 0, -2 ** 31, 6]])
def test_row_starts_out_of_order_stay_inside(pkg, starts):
    """What they compute is nobody's; what lies around the buffers stays as it is."""
    B = pm.Batch(8, [40, 10, 20], [2, 2, 2], 1, 64, 16, weights=True)
    fill_new(B)
    cache, _, _ = on_gpu(pkg, B, "f32")
    before = torch.nan_to_num(cache.k, nan=5.0).clone()
    need = pkg.op_paged_attention_scratch(cache, 6, 6, 2, True).numel()
    scratch = torch.full((need + 4096,), 0x5a, dtype=torch.uint8, device="cuda")
    out = torch.full((8, 128), 3.0, device="cuda")
    q = torch.randn(6, 128, device="cuda")
    pkg.op_paged_attention(cache, q, dev(np.array(starts, np.int32)), 6, 2, 0.125, accumulate=True, scratch=scratch[:need], out=out[:6])
    torch.cuda.synchronize()
    assert torch.all(out[6:] == 3.0) and torch.all(scratch[need:] == 0x5a)
    assert torch.equal(torch.nan_to_num(cache.k, nan=5.0), before)


@pytest.mark.parametrize("act,kind", TYPES)
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_values_that_are_not_finite_reach_only_rows_that_see_them(pkg, act, kind, bad):
    heads, dim = 4, 64
    for window, first, at in ((0, 0, 42), (8, 1, 0), (8, 1, 35)):   # the third row's own token; one that all see; one left behind
        B = pm.Batch(9, [40], [4], 2, dim, 16)
        fill_new(B)
        p, i = B.slot(0, at)
        B.v[p, 1, i, 5] = bad
        q64, q = held(B.rng.standard_normal((4, heads * dim)), act)
        cache, k64, v64 = on_gpu(pkg, B, kind)
        got = pkg.op_paged_attention(cache, q, dev(B.row_start), 4, heads, 0.125, window=window, first=first).double().cpu().numpy()
        want, _, _, _ = pm.attend(B, q64.reshape(4, heads, dim), k64, v64, heads, 0.125, window, first)
        want = want.reshape(4, -1)
        assert np.array_equal(np.isfinite(got), np.isfinite(want))
        ok = np.isfinite(want)
        assert np.all(np.abs(got[ok] - want[ok]) <= (2 ** -6 if act == "bf16" else 1e-5))


@pytest.mark.parametrize("act,kind", TYPES)
def test_extreme_scores(pkg, act, kind):
    """Scores of thousands, equal scores, and keys of the type's largest value against queries that are zero"""
    B = pm.Batch(10, [60, 60, 60], [1, 1, 1], 1, 64, 16)
    fill_new(B)
    B.k[B.table[0, 0], 0, 3] *= 60.0
    B.k[B.table[2, 1], 0, 5] = 60000.0
    q = B.rng.standard_normal((3, 64)) * 20.0
    q[1] = 0.0
    q[2] = 0.0
    q64, qt = held(q, act)
    cache, k64, v64 = on_gpu(pkg, B, kind)
    got = pkg.op_paged_attention(cache, qt, dev(B.row_start), 1, 1, 1.0).double().cpu().numpy()
    want, _, mass, top = pm.attend(B, q64.reshape(3, 1, 64), k64, v64, 1, 1.0)
    near(got.reshape(3, 1, 64), want, mass, act, kind, top, 64, 61)


# ---- append ---------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("act,kind", TYPES)
@pytest.mark.parametrize("heads,kv,dim,rot,page,lens,rows,pos", [
    (12, 2, 128, 128, 16, [200, 0, 15], [1, 3, 2], None),
    (7, 1, 64, 32, 32, [31, 64], [2, 1], [100, 3]),
    (4, 4, 72, 72, 16, [0], [40], None),
    (2, 1, 256, 0, 64, [63, 5, 9], [2, 0, 4], None),
    (3, 3, 8, 8, 16, [1], [1], [0]),
])
def test_append(pkg, act, kind, heads, kv, dim, rot, page, lens, rows, pos):
    B = pm.Batch(11, lens, rows, kv, dim, page, weights=True)
    cache, _, _ = on_gpu(pkg, B, kind)
    n, extra = B.total, 3
    fused = B.rng.standard_normal((n + extra, (heads + 2 * kv) * dim))
    f64, ft = held(fused, act)
    q, k, v = ft[:, :heads * dim], ft[:, heads * dim:(heads + kv) * dim], ft[:, (heads + kv) * dim:]
    sin, cos = (pkg.op_rope_table(512, rot, 1e4) if rot else (None, None))
    before_k, before_v = cache.k.clone(), cache.v.clone()
    out = torch.full((n + extra, heads * dim), 9.0, dtype=q.dtype, device="cuda")
    pkg.op_paged_append(cache, q, k, v, dev(B.row_start), sin, cos, pos=None if pos is None else dev(np.array(pos, np.int32)), out=out)
    torch.cuda.synchronize()
    sn, cs = (sin.cpu().numpy(), cos.cpu().numpy()) if rot else (None, None)
    got_q, got_k, got_v, got_w = (t.double().cpu().numpy() for t in (out, cache.k, cache.v, cache.weight))
    assert np.all(got_q[n:] == 9.0)
    want_k, want_v, want_w = before_k.double().cpu().numpy(), before_v.double().cpu().numpy(), B.weight.astype(np.float32).astype(float)

    def close(got, want, size, kind):   # two products and a sum in f32, then one rounding to the type; f16's smallest step
        assert np.all(np.abs(got - want) <= pm.HALF[kind] * np.abs(want) * 1.01 + 3 * 2.0 ** -24 * size + 2.0 ** -25 * (kind == "f16"))

    for b, base in enumerate(B.lens):
        for j in range(B.rows[b]):
            r, at = B.row_start[b] + j, (base if pos is None else pos[b]) + j
            x = f64[r].reshape(-1, dim)
            big = np.abs(x).max()
            close(got_q[r].reshape(heads, dim), pm.rotate(x[:heads], at, rot, sn, cs), big, act)
            p, i = B.slot(b, base + j)
            close(got_k[p, :, i], pm.rotate(x[heads:heads + kv], at, rot, sn, cs), big, kind)
            close(got_v[p, :, i], x[heads + kv:], 0.0, kind)
            assert np.all(got_w[p, :, i] == 0.0)
            want_k[p, :, i], want_v[p, :, i], want_w[p, :, i] = got_k[p, :, i], got_v[p, :, i], 0.0
    for got, want in ((got_k, want_k), (got_v, want_v), (got_w, want_w)):   # and nothing else was touched
        assert np.array_equal(got, want, equal_nan=True)


def test_append_leaves_out_what_has_no_place(pkg):
    B = pm.Batch(12, [14, 30, 5], [4, 4, 3], 1, 64, 16, table_ld=2)
    cache, _, _ = on_gpu(pkg, B, "f32")
    B.table[0, 1] = B.n_pages                      # rows 2 and 3 of the first sequence
    cache.table.copy_(dev(B.table))                # the second sequence's last two rows lie behind the table
    cache.length[1] = 30
    q, k, v = (torch.randn(11, 64, device="cuda") for _ in range(3))
    sin, cos = pkg.op_rope_table(40, 64, 1e4)
    pos = dev(np.array([0, 0, 38], np.int32))      # the third sequence's last row is past the rotation tables
    out = torch.full((11, 64), 9.0, device="cuda")
    before = torch.nan_to_num(cache.v, nan=-1.0)
    pkg.op_paged_append(cache, q, k, v, dev(B.row_start), sin, cos, pos=pos, out=out)
    after = torch.nan_to_num(cache.v, nan=-1.0)
    want = before.clone()
    for b, j, t in ((0, 0, 14), (0, 1, 15), (1, 0, 30), (1, 1, 31), (2, 0, 5), (2, 1, 6)):
        p, i = B.slot(b, t)
        want[p, 0, i] = v[B.row_start[b] + j]
    assert torch.equal(after, want)
    assert torch.all(out[10] == 9.0) and not torch.any(out[:10] == 9.0)


def test_append_in_place_and_keys_alone(pkg):
    B = pm.Batch(13, [3], [2], 2, 64, 16)
    cache, _, _ = on_gpu(pkg, B, "bf16")
    sin, cos = pkg.op_rope_table(64, 64, 1e4)
    q, k, v = (torch.randn(2, 128, device="cuda") for _ in range(3))
    want = pkg.op_paged_append(cache, q, k, v, dev(B.row_start), sin, cos)
    same = pkg.op_paged_append(cache, q, k, v, dev(B.row_start), sin, cos, out=q)
    assert same.data_ptr() == q.data_ptr() and torch.equal(same, want)


# ---- evict ----------------------------------------------------------------------------------------------------------------

def spare_cache(pkg, B, budget, kind, page=None):
    page = page or B.page
    room = -(-budget // page)
    table = np.random.default_rng(5).permutation(len(B.lens) * room + 2)[:len(B.lens) * room].reshape(len(B.lens), room).astype(np.int32)
    shape = (len(B.lens) * room + 2, B.kv, page)
    full = lambda *s: torch.full(s, 0.25, dtype=TORCH[kind], device="cuda")  # noqa: E731
    return table, pkg.PagedCache(full(*shape, B.dim), full(*shape, B.dim), dev(table), torch.zeros(len(B.lens), dtype=torch.int32, device="cuda"),
                                 torch.full(shape, 0.25, device="cuda"))


def check_evict(pkg, B, kind, budget, first, recent, page=None):
    cache, k64, v64 = on_gpu(pkg, B, kind)
    table, to = spare_cache(pkg, B, budget, kind, page)
    got = pkg.op_paged_evict(cache, to, budget, first, recent).cpu().numpy()
    weight = B.weight.astype(np.float32)
    kept = pm.evict(B, k64, v64, weight, budget, first, recent)
    assert np.array_equal(got, kept)
    assert to.length.tolist() == [min(max(n, 0), budget) for n in B.lens]
    want = [np.full(t.shape, 0.25) for t in (to.k, to.v, to.weight)]
    for b in range(len(B.lens)):
        for g in range(B.kv):
            for i, t in enumerate(x for x in kept[b, g] if x >= 0):
                dst = (table[b, i // to.k.shape[2]], g, i % to.k.shape[2])
                p, s = B.slot(b, t)
                there = B.there(b, t)
                want[0][dst], want[1][dst], want[2][dst] = (k64[p, g, s], v64[p, g, s], weight[p, g, s]) if there else (0, 0, 0)
    for t, w in zip((to.k, to.v, to.weight), want):
        assert np.array_equal(t.double().cpu().numpy(), w, equal_nan=True)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kv,dim,page,lens,budget,first,recent", [
    (2, 128, 16, [100, 64, 65, 63, 0, 1], 64, 4, 16),
    (1, 64, 32, [1500, 2049], 300, 0, 0),
    (3, 72, 16, [90], 1, 0, 0),
    (1, 256, 64, [200, 130], 128, 100, 28),      # nothing but the first and the last
    (2, 8, 16, [40, 300], 33, 0, 33),
])
def test_evict(pkg, kind, kv, dim, page, lens, budget, first, recent):
    check_evict(pkg, pm.Batch(14, lens, [0] * len(lens), kv, dim, page, weights=True), kind, budget, first, recent)


def test_evict_from_a_table_for_very_long_sequences(pkg):
    """More slots than the selection holds in LDS"""
    B = pm.Batch(29, [3000, 700], [0, 0], 1, 8, 64, weights=True, table_ld=600)
    check_evict(pkg, B, "bf16", 900, 5, 100)


def test_evict_equal_weights_and_odd_ones(pkg):
    B = pm.Batch(15, [500, 400, 300, 2500], [0] * 4, 1, 64, 16, weights=True)
    pick = np.array([0.0, -0.0, 1.0, 1.0, 2.0, -3.0, np.inf, -np.inf, 1e-40, np.nan])
    B.weight = np.where(np.isnan(B.weight), np.nan, B.rng.choice(pick, B.weight.shape))
    B.weight[B.table[3, 20:40]] = 1.0
    check_evict(pkg, B, "bf16", 128, 3, 17)
    B.weight = np.zeros_like(B.weight)
    check_evict(pkg, B, "f32", 100, 0, 10, page=64)


def test_evict_with_pages_that_are_not_there(pkg):
    B = pm.Batch(16, [200, 100], [0, 0], 2, 64, 16, weights=True)
    B.table[0, 2], B.table[1, 0] = -1, B.n_pages + 3
    check_evict(pkg, B, "bf16", 64, 2, 60)


# ---- verification ---------------------------------------------------------------------------------------------------------

def drafted(rng, rows, V, draft, std=2.0):
    """Logits, tokens of which many will be accepted, and the numbers"""
    starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    n = int(starts[-1])
    logits = (rng.standard_normal((n, V)) * std).astype(np.float32)
    other = (logits + rng.standard_normal((n, V)) * 0.7).astype(np.float32) if draft else None
    tokens = rng.integers(0, V, n)
    for b in range(len(rows)):
        for r in range(starts[b], starts[b + 1] - 1):
            tokens[r + 1] = np.argmax((other if draft else logits * 1.5)[r] + rng.gumbel(size=V))
    return starts, logits, other, tokens, rng.random(n, dtype=np.float32), rng.random(len(rows), dtype=np.float32)


def check_verify(pkg, starts, logits, other, tokens, uniform, choice, temperature, max_rows=None, want=None, **kw):
    length = torch.full((len(starts) - 1,), 100, dtype=torch.int32, device="cuda")
    lt = kw.get("lt", dev(logits))
    count, token = pkg.op_verify_drafts(lt, dev(starts), max_rows or max(1, int(np.diff(starts).max())), dev(tokens), dev(uniform), dev(choice),
                                        temperature, draft=None if other is None else kw.get("dt", dev(other)), length=length)
    a, b = want or pm.verify(logits, starts, tokens, uniform, choice, temperature, other)
    assert count.tolist() == a.tolist() and token.tolist() == b.tolist()
    assert length.tolist() == (100 + a).tolist()


@pytest.mark.parametrize("V", [1, 2, 63, 1000, 4096, 4097, 20001])
@pytest.mark.parametrize("temperature", [0.0, 0.3, 1.0, 2.5])
@pytest.mark.parametrize("draft", [False, True])
def test_verify(pkg, V, temperature, draft):
    rng = np.random.default_rng(17 + V)
    rows = [1, 5, 0, 3, 8, 2, 1, 11, 0]
    check_verify(pkg, *drafted(rng, rows, V, draft), temperature)


def test_verify_large_vocabulary(pkg):
    rng = np.random.default_rng(18)
    check_verify(pkg, *drafted(rng, [5, 3, 8], 151936, True), 1.0)
    check_verify(pkg, *drafted(rng, [5, 2], 152064, False, std=0.3), 0.8)


def test_verify_keeps_the_target_distribution(pkg):
    """Many sequences of one drafted token each: the first emitted token is distributed as the target's, whatever the draft."""
    rng, n, V = np.random.default_rng(19), 20000, 5
    p, q = np.array([0.4, 0.3, 0.2, 0.1, 0.0]), np.array([0.1, 0.1, 0.1, 0.3, 0.4])
    starts = (2 * np.arange(n + 1)).astype(np.int32)
    with np.errstate(divide="ignore"):
        logits, other = (np.tile(np.log(x).astype(np.float32), (2 * n, 1)) for x in (p, q))
    tokens = np.zeros(2 * n, np.int64)
    tokens[1::2] = rng.choice(V, n, p=q)
    uniform, choice = rng.random(2 * n, dtype=np.float32), rng.random(n, dtype=np.float32)
    count, token = pkg.op_verify_drafts(dev(logits), dev(starts), 2, dev(tokens), dev(uniform), dev(choice), 1.0, draft=dev(other))
    first = torch.where(count == 2, dev(tokens[1::2]), token).cpu().numpy()
    got = np.bincount(first, minlength=V) / n
    assert got[4] == 0.0
    assert np.all(np.abs(got - p) <= 5 * np.sqrt(p * (1 - p) / n))   # five standard deviations of a share of n draws


def test_verify_odd_logits(pkg):
    rng = np.random.default_rng(20)
    starts, logits, other, tokens, uniform, choice = drafted(rng, [2] * 10, 700, False)
    logits[0, :] = -np.inf                  # no distribution
    logits[2, 5] = np.nan
    logits[4, 7] = np.inf
    logits[6, :699] = -np.inf               # one token alone
    tokens[7] = 699
    logits[7, :] = -np.inf
    tokens[9] = 700                         # no such token
    tokens[11] = -1
    logits[12, tokens[13]] = -np.inf        # a token that cannot be
    logits[14, 20:] = -np.inf
    logits[16] *= 1e36                      # one token is all there is
    logits[18] = 0.0                        # all alike
    want = pm.verify(logits, starts, tokens, uniform, choice, 1.0)
    assert want[1][:4].tolist() == [-1, -1, -1, -1] and want[0][:4].tolist() == [1, 1, 1, 2]
    check_verify(pkg, starts, logits, None, tokens, uniform, choice, 1.0)
    clean = np.where(np.isnan(logits), -np.inf, logits)
    check_verify(pkg, starts, clean, None, tokens, uniform, choice, 0.0)
    same = clean.copy()                     # draft and target alike: all is accepted, and a refusal has nothing left but p
    same[0], same[4] = 0.0, 1.0
    same[7] = 2.0
    check_verify(pkg, starts, same, same, tokens, uniform, choice, 1.0)


@pytest.mark.parametrize("temperature", [1e-2, 1e-6, 1e-12, 1e-20, 1e-38])
def test_verify_low_temperatures(pkg, temperature):
    """All that is left are the largest logits, each as likely as the other"""
    rng = np.random.default_rng(23)
    starts, logits, other, tokens, uniform, choice = drafted(rng, [2, 3] * 12, 5000, False)
    for r in range(len(logits)):
        at = rng.choice(5000, int(rng.integers(1, 5)), replace=False)
        logits[r, at] = np.float32(37.3) + r
        if r + 1 < len(tokens):
            tokens[r + 1] = rng.choice(at)
    check_verify(pkg, starts, logits, None, tokens, uniform, choice, temperature)
    check_verify(pkg, starts, logits, np.roll(logits, 1, 0), tokens, uniform, choice, temperature)


def test_verify_of_rows_in_wider_tensors(pkg):
    rng = np.random.default_rng(21)
    starts, logits, other, tokens, uniform, choice = drafted(rng, [3, 1, 4], 1001, True)
    wide = torch.full((8, 2051), float("nan"), device="cuda")
    wide[:, 3:1004], wide[:, 1010:2011] = dev(logits), dev(other)
    check_verify(pkg, starts, logits, other, tokens, uniform, choice, 1.0, lt=wide[:, 3:1004], dt=wide[:, 1010:2011])


def test_verify_numbers_at_the_ends(pkg):
    rng = np.random.default_rng(22)
    starts, logits, other, tokens, uniform, choice = drafted(rng, [2, 2, 2, 2], 5000, True)
    logits[:, 0] = logits[:, 4999] = -np.inf
    uniform[:], choice[:2], choice[2:] = 0.0, 0.0, np.float32(1 - 2.0 ** -24)
    check_verify(pkg, starts, logits, other, tokens, uniform, choice, 1.0)
    uniform[:] = np.float32(1 - 2.0 ** -24)
    check_verify(pkg, starts, logits, other, tokens, uniform, choice, 1.0)


# ---- together -------------------------------------------------------------------------------------------------------------

def torch_rope(pkg, n, dim):
    return pkg.op_rope_table(n, dim, 1e4)


@pytest.mark.parametrize("act,kind", TYPES)
def test_a_run_of_steps(pkg, act, kind):
    """Append, attend with weights, evict to other pages, then append at the true positions and attend again."""
    heads, kv, dim, page = 6, 2, 64, 16
    B = pm.Batch(23, [70, 33], [2, 3], kv, dim, page, weights=True)
    cache, k64, v64 = on_gpu(pkg, B, kind)
    sin, cos = torch_rope(pkg, 256, dim)
    starts = dev(B.row_start)

    def step(B, cache, pos):
        q, k, v = (torch.randn(B.total, n * dim, device="cuda").to(TORCH[act]) for n in (heads, kv, kv))
        turned = pkg.op_paged_append(cache, q, k, v, starts, sin, cos, pos=None if pos is None else dev(np.array(pos, np.int32)))
        k64, v64 = cache.k.double().cpu().numpy(), cache.v.double().cpu().numpy()
        weight = cache.weight.double().cpu().numpy()
        out = pkg.op_paged_attention(cache, turned, starts, 3, heads, dim ** -0.5, accumulate=True)
        q64 = turned.double().cpu().numpy().reshape(-1, heads, dim)
        want, added, mass, top = pm.attend(B, q64, k64, v64, heads, dim ** -0.5)
        near(out.double().cpu().numpy().reshape(-1, heads, dim), want, mass, act, kind, top, dim, 80)
        got = cache.weight.double().cpu().numpy()
        ok = ~np.isnan(weight)
        assert np.allclose(got[ok], (weight + added)[ok], rtol=2e-5, atol=1e-6)

    step(B, cache, None)
    cache.length += dev(np.array(B.rows, np.int32))
    B.lens = [a + b for a, b in zip(B.lens, B.rows)]
    true = list(B.lens)
    B.weight = cache.weight.double().cpu().numpy()
    table, to = spare_cache(pkg, B, 48, kind)
    kept = pkg.op_paged_evict(cache, to, 40, 2, 8)
    assert np.array_equal(kept.cpu().numpy(), pm.evict(B, None, None, B.weight, 40, 2, 8))
    B.table, B.lens, B.ld, B.n_pages = table, [min(n, 40) for n in true], table.shape[1], to.k.shape[0]
    assert to.length.tolist() == B.lens
    step(B, to, true)


def test_other_streams_and_graphs_at_other_lengths(pkg):
    """A captured step serves lengths, tables and rows that change between its replays; eager work stands in between."""
    heads, kv, dim, page, seqs = 6, 2, 128, 16, 3
    B = pm.Batch(24, [300, 20, 0], [2, 2, 2], kv, dim, page, table_ld=24)
    k, v = (torch.randn(B.n_pages + 40, kv, page, dim, device="cuda").to(torch.bfloat16) for _ in range(2))
    order = np.random.default_rng(6).permutation(B.n_pages + 40)[:3 * 20].reshape(3, 20)
    table = torch.full((3, 24), -1, dtype=torch.int32, device="cuda")
    table[:, :20] = dev(order.astype(np.int32))
    weight = torch.zeros(k.shape[:3], device="cuda")
    length = torch.zeros(3, dtype=torch.int32, device="cuda")
    cache = pkg.PagedCache(k, v, table, length, weight)
    starts = dev(B.row_start)
    q, kn, vn = (torch.empty(6, n * dim, device="cuda") for n in (heads, kv, kv))
    sin, cos = pkg.op_rope_table(512, dim, 1e4)
    logits, draft = torch.empty(6, 5003, device="cuda"), torch.empty(6, 5003, device="cuda")
    uniform, choice = torch.empty(6, device="cuda"), torch.empty(3, device="cuda")
    tokens = torch.zeros(6, dtype=torch.int64, device="cuda")
    scratch = pkg.op_paged_attention_scratch(cache, 6, 2, heads, True)
    vscratch = pkg.op_verify_drafts_scratch(6, 5003, 3)
    to = pkg.PagedCache(torch.zeros_like(k), torch.zeros_like(v), table, torch.zeros_like(length), torch.zeros_like(weight))

    def step():
        turned = pkg.op_paged_append(cache, q, kn, vn, starts, sin, cos)
        out = pkg.op_paged_attention(cache, turned, starts, 2, heads, dim ** -0.5, window=200, first=4, accumulate=True, scratch=scratch)
        kept = pkg.op_paged_evict(cache, to, 32, 4, 8)
        count, token = pkg.op_verify_drafts(logits, starts, 2, tokens, uniform, choice, 1.0, draft=draft, length=length, scratch=vscratch)
        return out, kept, count, token

    def inputs(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        for t in (q, kn, vn, logits):
            t.normal_(generator=g)
        draft.copy_(logits + 0.3)
        draft[:, ::2] -= 0.5
        for t in (uniform, choice):
            t.uniform_(generator=g)
        tokens.random_(0, 5003, generator=g)
        length.copy_(torch.tensor([[250, 20, 0], [5, 310, 64], [0, 0, 0], [17, 100, 300]][seed % 4], dtype=torch.int32))
        weight.zero_()
        to.k.zero_()

    side = torch.cuda.Stream()
    inputs(0)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    side.synchronize()
    inputs(0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        held_out = step()
    for seed in (1, 2, 3, 0, 1):
        inputs(seed)
        want = [t.clone() for t in step()] + [weight.clone(), length.clone(), to.k.clone(), to.length.clone()]
        torch.cuda.synchronize()
        inputs(seed)
        for t in held_out:
            t.fill_(3)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip([*held_out, weight, length, to.k, to.length], want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("act,kind", [("bf16", "bf16"), ("f32", "f16")])
def test_a_captured_portion_of_prompts(pkg, act, kind):
    """Buffers for 700 rows of three sequences, of which every replay finds other numbers; the graph and eager calls share their
    scratch memory in turn."""
    heads, kv, dim, page = 8, 4, 128, 32
    B = pm.Batch(29, [700, 700, 700], [0, 0, 0], kv, dim, page)
    cache, _, _ = on_gpu(pkg, B, kind)
    q = torch.randn(700, heads * dim, device="cuda").to(torch.bfloat16 if act == "bf16" else torch.float32)
    starts, out = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.empty_like(q)
    scratch = pkg.op_paged_attention_scratch(cache, 700, 600, heads)

    def step(out):
        return pkg.op_paged_attention(cache, q, starts, 600, heads, 0.1, scratch=scratch, out=out)

    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        step(out)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(out)
    for lens, rows in (([100, 0, 30], [600, 99, 1]), ([0, 5, 0], [2, 0, 1]), ([690, 0, 10], [4, 590, 50]), ([0, 0, 0], [0, 0, 0]),
                       ([100, 0, 30], [600, 99, 1])):
        starts.copy_(torch.tensor(np.concatenate([[0], np.cumsum(rows)]), dtype=torch.int32))
        cache.length.copy_(torch.tensor(lens, dtype=torch.int32))
        want = step(torch.full_like(q, 3.0)).clone()
        out.fill_(3.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert bool((want[sum(rows):] == 3.0).all()) and not bool((want[:sum(rows)] == 3.0).all(1).any())


@pytest.mark.parametrize("rows", [[2, 3], [600, 300]])
def test_most_rows_of_any_number(pkg, rows):
    B = pm.Batch(30, [40, 70], rows, 4, 64, 16)
    fill_new(B)
    q64, q = held(B.rng.standard_normal((B.total, 8 * 64)), "f32")
    cache, k64, v64 = on_gpu(pkg, B, "bf16")
    outs = [pkg.op_paged_attention(cache, q, dev(B.row_start), most, 8, 0.125) for most in (max(rows), 2 ** 31 - 1)]
    want = pm.attend(B, q64.reshape(-1, 8, 64), k64, v64, 8, 0.125)[0].reshape(B.total, -1)
    for out in outs:
        assert np.all(np.abs(out.double().cpu().numpy() - want) <= 1e-5)


def test_sequences_that_share_a_prompts_pages(pkg):
    """Two sequences read the same pages and append to pages of their own, on two streams at once with the same step alone"""
    heads, kv, dim, page = 8, 2, 64, 16
    B = pm.Batch(31, [64, 64, 64], [3, 2, 0], kv, dim, page)
    B.table[1, :4] = B.table[0, :4]
    fill_new(B)
    q64, q = held(B.rng.standard_normal((B.total, heads * dim)), "f32")
    cache, k64, v64 = on_gpu(pkg, B, "f16")
    want = pm.attend(B, q64.reshape(-1, heads, dim), k64, v64, heads, 0.125)[0].reshape(B.total, -1)
    starts, outs = dev(B.row_start), [torch.empty_like(q) for _ in range(2)]
    scratch = [pkg.op_paged_attention_scratch(cache, B.total, 3, heads) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, o, w in zip(streams, outs, scratch):
            with torch.cuda.stream(s):
                pkg.op_paged_attention(cache, q, starts, 3, heads, 0.125, scratch=w, out=o)
    torch.cuda.synchronize()
    for o in outs:
        assert np.all(np.abs(o.double().cpu().numpy() - want) <= 1e-5)
    assert torch.equal(*outs)


def test_more_rows_than_the_join_has_workgroups(pkg):
    """5000 sequences of 4 rows and 64 heads: 1.3 million rows of heads, each shared by several workgroups or not"""
    n, rows, heads, dim, length = 5000, 4, 64, 8, 150
    g = torch.Generator(device="cuda").manual_seed(5)
    pages = (length + rows + 15) // 16
    k, v = (torch.randn(n * pages, 1, 16, dim, device="cuda", generator=g) for _ in range(2))
    q = torch.randn(n * rows, heads * dim, device="cuda", generator=g)
    table = torch.arange(n * pages, dtype=torch.int32, device="cuda").reshape(n, pages)
    cache = pkg.PagedCache(k, v, table, torch.full((n,), length, dtype=torch.int32, device="cuda"))
    starts = torch.arange(n + 1, dtype=torch.int32, device="cuda") * rows
    got = pkg.op_paged_attention(cache, q, starts, rows, heads, 0.3).reshape(n, rows * heads, dim)
    seen = torch.arange(pages * 16, device="cuda")[None] <= length + torch.arange(rows, device="cuda")[:, None].repeat_interleave(heads, 0)
    for b in range(0, n, 500):
        kk, vv, qq = (x.double() for x in (k.reshape(n, -1, dim)[b:b + 500], v.reshape(n, -1, dim)[b:b + 500],
                                           q.reshape(n, rows * heads, dim)[b:b + 500]))
        s = torch.matmul(qq, kk.transpose(1, 2).contiguous()) * 0.3
        want = torch.matmul(torch.softmax(s.masked_fill(~seen, float("-inf")), -1), vv)
        assert bool(((got[b:b + 500] - want).abs() <= 1e-5).all())


@pytest.mark.parametrize("act,kind", TYPES)
def test_many_short_sequences(pkg, act, kind):
    """More sequences than workgroups, of up to eight tiles each: none is shared"""
    rng = np.random.default_rng(6)
    n = 650
    B = pm.Batch(35, rng.integers(0, 60, n).tolist(), rng.integers(0, 4, n).tolist(), 2, 16, 16, table_ld=4, weights=True)
    fill_new(B)
    run_attention(pkg, B, act, kind, 6)
    run_attention(pkg, B, act, kind, 6, accumulate=True)


def test_refused_tensors(pkg):
    B = pm.Batch(32, [40], [2], 2, 64, 16)
    fill_new(B)
    cache, _, _ = on_gpu(pkg, B, "f32")
    q, starts = torch.randn(2, 256, device="cuda"), dev(B.row_start)
    scratch = pkg.op_paged_attention_scratch(cache, 2, 2, 4)
    good = dict(q=q, row_start=starts, max_rows=2, heads=4, scale=0.1, scratch=scratch)
    for bad in (dict(q=q.cpu()), dict(q=q.half()), dict(q=q[:, ::2]), dict(q=q[0]), dict(q=q[:, :128]), dict(row_start=starts.long()),
                dict(row_start=starts.cpu()), dict(row_start=starts[:1]), dict(scratch=scratch.cpu()), dict(scratch=scratch[:64]),
                dict(window=2 ** 31), dict(first=2 ** 32), dict(window=-1), dict(scale=float("inf")), dict(out=q[:1].clone()),
                dict(out=torch.empty_like(q).bfloat16()), dict(heads=3), dict(heads=0), dict(max_rows=0)):
        with pytest.raises((pkg.W4A32Error, IndexError)):
            pkg.op_paged_attention(cache, **{**good, **bad})
    pkg.op_paged_attention(cache, **good)
    k, v, table, length = cache.k, cache.v, cache.table, cache.length
    for bad in ((k.cpu(), v, table, length), (k, v[:-1], table, length), (k, v.half(), table, length), (k, v, table.long(), length),
                (k, v, table, length.cpu()), (k, v, table[0], length), (k.double(), v.double(), table, length),
                (k.transpose(1, 2), v, table, length), (k, v, table, length, torch.zeros(3, device="cuda"))):
        with pytest.raises(pkg.W4A32Error):
            pkg.PagedCache(*bad)
    weight = torch.zeros(k.shape[:3], device="cuda")
    one = pkg.PagedCache(k, v, table, length, weight)
    two = pkg.PagedCache(k.clone(), v.clone(), table, length.clone(), weight.clone())
    for bad in (dict(to=one), dict(to=cache), dict(budget=0), dict(budget=2 ** 31), dict(first=2 ** 32), dict(recent=9),
                dict(scratch=torch.empty(10 ** 4)), dict(to=pkg.PagedCache(k, v, table, length.clone(), weight.clone()))):
        with pytest.raises(pkg.W4A32Error):
            pkg.op_paged_evict(one, **{**dict(to=two, budget=8), **bad})
    logits, tokens = torch.randn(2, 50, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    u, c = torch.rand(2, device="cuda"), torch.rand(1, device="cuda")
    good = dict(logits=logits, row_start=starts, max_rows=2, tokens=tokens, uniform=u, choice=c, temperature=1.0)
    for bad in (dict(logits=logits.half()), dict(logits=logits.t()), dict(tokens=tokens.int()), dict(tokens=tokens[:1]), dict(uniform=None),
                dict(choice=None), dict(uniform=u.double()), dict(choice=c.cpu()), dict(temperature=-0.5), dict(draft=logits[:, :49]),
                dict(scratch=torch.empty(10 ** 5)), dict(length=torch.zeros(2, dtype=torch.int32, device="cuda"))):
        with pytest.raises(pkg.W4A32Error):
            pkg.op_verify_drafts(**{**good, **bad})
    count, token = pkg.op_verify_drafts(**{**good, "uniform": None, "choice": None, "temperature": 0.0})
    assert count.tolist()[0] in (1, 2) and int(token) == int(logits[int(count) - 1].argmax())


def test_pages_beyond_32_bits_of_the_pools(pkg):
    """Pools of 4.5 thousand million elements, of which the last pages are used: the same bits as from small ones"""
    heads, kv, dim, page, far, few = 16, 8, 256, 128, 17100, 12
    assert (far - few) * kv * page * dim > 2 ** 32
    small = [torch.randn(few, kv, page, dim, device="cuda").bfloat16() for _ in range(2)]
    large = [torch.empty(far, kv, page, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    weight = torch.rand(few, kv, page, device="cuda")
    far_weight = torch.empty(far, kv, page, device="cuda")
    for a, b in zip((*small, weight), (*large, far_weight)):
        b[far - few:] = a
    table = torch.tensor([[3, 0, 7, 5], [1, 6, 2, 4]], dtype=torch.int32, device="cuda")
    length = torch.tensor([300, 30], dtype=torch.int32, device="cuda")
    caches = [pkg.PagedCache(*small, table, length, weight), pkg.PagedCache(*large, table + (far - few), length, far_weight)]
    others = torch.tensor([[8, 9], [10, 11]], dtype=torch.int32, device="cuda")
    sin, cos = pkg.op_rope_table(600, dim, 1e4)
    for rows in ([2, 1], [200, 300]):
        starts = torch.tensor([0, rows[0], sum(rows)], dtype=torch.int32, device="cuda")
        q, k, v = (torch.randn(sum(rows), n * dim, device="cuda").bfloat16() for n in (heads, kv, kv))
        outs = []
        for cache in caches:
            turned = pkg.op_paged_append(cache, q, k, v, starts, sin, cos)
            outs.append([turned, pkg.op_paged_attention(cache, turned, starts, max(rows), heads, dim ** -0.5),
                         pkg.op_paged_attention(cache, turned, starts, max(rows), heads, dim ** -0.5, window=40, first=2, accumulate=True)])
        for a, b in zip(*outs):
            assert torch.equal(a, b) and bool(a.isfinite().all())
        for a, b in zip((*small, weight), (*large, far_weight)):
            assert torch.equal(a, b[far - few:])
    tos = [pkg.PagedCache(c.k, c.v, others + shift, torch.zeros_like(length), c.weight) for c, shift in zip(caches, (0, far - few))]
    kept = [pkg.op_paged_evict(c, to, 100, 4, 20) for c, to in zip(caches, tos)]
    assert torch.equal(*kept) and torch.equal(tos[0].length, tos[1].length)
    for a, b in zip((*small, weight), (*large, far_weight)):
        assert torch.equal(a, b[far - few:])
