"""Attention of sequences that share prefixes in groups, against the definition in 64 bits: each sequence alone, with its prefix where it has it."""
import numpy as np
import pytest
import torch

import paged_model as pm
from test_gpu_paged import TYPES, dev, fill_new, held, near, on_gpu

pytestmark = pytest.mark.gpu


class Groups(pm.Batch):
    """Sequences in groups: counts[g] of them have prefix[g] tokens in the pages of the first, and own[b] of their own behind. Where the others'
    tables have room for the prefix they name the first one's pages; the page in which it ends is each one's own, with NaN in the prefix's
    places of all but the first: nobody reads them."""

    def __init__(self, seed, counts, prefix, own, rows, kv, dim, page, table_ld=None):
        self.counts, self.prefix = list(counts), list(prefix)
        group = [g for g, n in enumerate(counts) for _ in range(n)]
        super().__init__(seed, [prefix[g] + n for g, n in zip(group, own)], rows, kv, dim, page, table_ld=table_ld)
        self.group_start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.alone = self.table.copy()   # what a sequence sees, were it alone: its prefix's tokens are its first one's
        for b, g in enumerate(group):
            first, P = self.group_start[g], prefix[g]
            for i in range(min(P // page, self.ld)):
                self.table[b, i] = self.alone[b, i] = self.table[first, i]

    def definition(self, q, k, v, heads, scale):
        """attend() of the batch, with every sequence's part of the page in which the prefix ends filled from the first one's"""
        k, v = k.copy(), v.copy()
        for g, P in enumerate(self.prefix):
            a, e = self.group_start[g:g + 2]
            for b in range(a + 1, e):
                for t in range(P // self.page * self.page, P):
                    if self.there(a, t) and self.there(b, t):
                        (p, i), (o, _) = self.slot(b, t), self.slot(a, t)
                        k[p, :, i], v[p, :, i] = k[o, :, i], v[o, :, i]
        return pm.attend(self, q, k, v, heads, scale)

    def hide(self):
        for g, P in enumerate(self.prefix):
            a, e = self.group_start[g:g + 2]
            for b in range(a + 1, e):
                for t in range(P // self.page * self.page, P):
                    if self.there(b, t):
                        p, i = self.slot(b, t)
                        self.k[p, :, i] = self.v[p, :, i] = np.nan


def run(pkg, B, act, kind, heads, pad=0, stride=0, scale=None, scratch=None, max_rows=None, cut=None):
    fill_new(B)
    B.hide()
    q = B.rng.standard_normal((max(1, B.total) + pad, heads * B.dim + stride)) * 2.0
    q64, qt = held(q, act)
    q64 = q64[:, :heads * B.dim].reshape(-1, heads, B.dim)[:B.total]
    qt = qt[:, :heads * B.dim]
    cache, k64, v64 = on_gpu(pkg, B, kind)
    scale = B.dim ** -0.5 if scale is None else scale
    out = torch.full((max(1, B.total) + pad, heads * B.dim), 7.5, dtype=qt.dtype, device="cuda")
    most = max_rows or max(1, max(B.rows))
    if scratch is None:
        scratch = pkg.op_paged_prefix_attention_scratch(cache, out.shape[0], most, heads, len(B.counts))
        scratch.fill_(0xFF)   # NaN
    got = pkg.op_paged_prefix_attention(cache, qt, dev(B.row_start), most, heads, scale, dev(B.group_start),
                                        dev(np.array(B.prefix if cut is None else cut, np.int32)), scratch=scratch, out=out)
    torch.cuda.synchronize()
    want, _, mass, top = B.definition(q64, k64, v64, heads, scale)
    got = got.double().cpu().numpy()
    assert np.all(got[B.total:] == 7.5)
    near(got[:B.total].reshape(-1, heads, B.dim), want, mass, act, kind, top, B.dim, max(n + r for n, r in zip(B.lens, B.rows)))
    return got


SHAPES = [
    # heads, kv, dim, page, sequences of groups, prefixes, own tokens, rows
    (12, 2, 128, 16, [4], [200], [0, 40, 7, 16], [1, 1, 1, 1]),
    (7, 1, 128, 32, [3, 1, 2], [100, 64, 33], [5, 31, 32, 33, 0, 1], [1, 2, 1, 3, 1, 0]),       # a group of one, and one with rows of one alone
    (8, 8, 64, 64, [2], [129], [0, 3], [1, 2]),                                               # a head of its own for every query head
    (6, 2, 80, 16, [2, 3], [47, 0], [1, 10, 20, 3, 0], [3, 1, 1, 1, 5]),                      # a prefix of none
    (4, 2, 256, 128, [5], [300], [17, 0, 255, 1, 128], [1, 4, 1, 2, 1]),
    (34, 2, 72, 32, [2, 2], [70, 31], [2, 9, 0, 64], [2, 1, 1, 6]),
    (4, 1, 8, 16, [3], [1], [0, 0, 1], [1, 1, 1]),
    (6, 2, 96, 16, [6], [65], [0, 60, 3, 0, 0, 9], [37, 0, 21, 1, 0, 2]),                     # prompts behind a prefix, sequences without rows
    (28, 4, 128, 16, [20], [515], [i % 23 for i in range(20)], [1] * 20),                     # a workgroup of 256 rows, not all there
    (14, 2, 64, 16, [9, 8], [333, 260], list(range(17)), [3 + i % 3 for i in range(17)]),
    (16, 2, 256, 32, [10], [130], list(range(10)), [2] * 10),
    (12, 2, 64, 16, [3, 2], [100, 31], [5, 0, 70, 0, 1], [50, 3, 130, 22, 21]),                # prompts of more rows than a workgroup has, and fewer
    (12, 2, 128, 16, [2], [77], [0, 3], [64, 90]),                                            # and no others
    (4, 2, 256, 32, [3], [130], [100, 0, 40], [90, 1, 65]),
    (7, 1, 72, 16, [2, 2], [40, 0], [13, 0, 0, 50], [40, 19, 18, 60]),
    (12, 1, 128, 64, [30], [700], [3 * i for i in range(30)], [1 + i % 2 for i in range(30)]),
]


@pytest.mark.parametrize("act,kind", TYPES)
@pytest.mark.parametrize("heads,kv,dim,page,counts,prefix,own,rows", SHAPES)
def test_prefix_attention(pkg, act, kind, heads, kv, dim, page, counts, prefix, own, rows):
    run(pkg, Groups(1, counts, prefix, own, rows, kv, dim, page), act, kind, heads)


@pytest.mark.parametrize("act,kind", TYPES)
def test_strides_and_a_padded_batch(pkg, act, kind):
    run(pkg, Groups(2, [3, 4], [75, 130], [1, 2, 3, 4, 5, 6, 7], [2, 1, 0, 3, 1, 1, 1], 2, 64, 16), act, kind, 8, pad=5, stride=24)


@pytest.mark.parametrize("act,kind", TYPES)
@pytest.mark.parametrize("scale", [0.0, -0.3, 1e-40])
def test_scales(pkg, act, kind, scale):
    run(pkg, Groups(3, [3], [90], [0, 1, 30], [1, 2, 1], 2, 64, 16), act, kind, 6, scale=scale)


@pytest.mark.parametrize("act,kind", TYPES)
def test_one_sequence_and_many(pkg, act, kind):
    run(pkg, Groups(4, [1], [50], [3], [2], 2, 64, 16), act, kind, 6)
    counts = [3] * 50   # more than a wavefront's lanes of groups and sequences
    run(pkg, Groups(5, counts, [16 + 3 * i for i in range(50)], [i % 20 for i in range(150)], [(i * 7) % 3 for i in range(150)], 2, 64, 16), act, kind, 6)
    for n in (64, 65):   # one wavefront's lanes of sequences, and more
        run(pkg, Groups(5, [n - 7, 4, 3], [50, 0, 33], [i % 20 for i in range(n)], [i % 3 for i in range(n)], 2, 64, 16), act, kind, 6)
    for n in (8, 9, 16, 17):   # as many groups as are gone through one by one, and more
        run(pkg, Groups(5, [2] * n, [20 + i for i in range(n)], [i % 20 for i in range(2 * n)], [1 + i % 3 for i in range(2 * n)], 2, 64, 16), act, kind, 6)
    run(pkg, Groups(5, [40, 40], [50, 33], [i % 20 for i in range(80)], [70 if i % 9 == 0 else 1 for i in range(80)], 1, 64, 16), act, kind, 2)
    run(pkg, Groups(6, [1] * 70 + [70], [20] * 71, [i % 5 for i in range(140)], [1] * 140, 1, 64, 16), act, kind, 2)


@pytest.mark.parametrize("act,kind", TYPES)
def test_prefixes_that_pass_lengths_and_tables(pkg, act, kind):
    """A prefix is cut to what the sequences with rows have; a table may end inside it; negative ones are none"""
    B = Groups(7, [3, 2], [64, 32], [0, 16, 40, 0, 9], [1, 1, 2, 1, 1], 2, 64, 16)
    run(pkg, B, act, kind, 6, cut=[1 << 30, 40])
    run(pkg, Groups(7, [3, 2], [64, 32], [0, 16, 40, 0, 9], [1, 1, 2, 1, 1], 2, 64, 16), act, kind, 6, cut=[-5, -(1 << 31)])
    run(pkg, Groups(8, [3], [100], [5, 60, 0], [1, 3, 1], 2, 64, 16, table_ld=4), act, kind, 6)   # rows behind the table's end
    run(pkg, Groups(8, [3], [100], [5, 60, 0], [1, 3, 1], 2, 64, 16, table_ld=7), act, kind, 6)


@pytest.mark.parametrize("act,kind", TYPES)
def test_pages_that_are_not_there(pkg, act, kind):
    """Holes in the prefix and behind it; a row that sees nothing at all gets zeros"""
    B = Groups(9, [3, 2], [96, 48], [20, 0, 40, 0, 0], [1, 1, 2, 1, 1], 2, 64, 16)
    B.table[:3, 2] = -1
    B.table[:3, 4] = B.n_pages + 3
    B.table[1, 6] = -1          # the only page of its own
    B.table[3:, :] = -1
    got = run(pkg, B, act, kind, 6)
    assert np.all(got[4:6] == 0)


@pytest.mark.parametrize("act,kind", TYPES)
def test_lowest_and_infinite_values_where_nobody_sees_them(pkg, act, kind):
    B = Groups(10, [4], [61], [0, 5, 30, 1], [1, 2, 1, 1], 2, 64, 32)
    fill_new(B)
    B.hide()
    bad = np.isnan(B.k)
    lowest = float(torch.finfo({"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[kind]).min)
    for x in (np.inf, -np.inf, lowest):
        B.k[bad] = B.v[bad] = x
        B.hide = lambda: None
        cache_free = B
        run(pkg, cache_free, act, kind, 6)


@pytest.mark.parametrize("act,kind", TYPES)
@pytest.mark.parametrize("n,rows", [(2, 1), (24, 1), (2, 40)])
def test_values_that_are_not_finite(pkg, act, kind, n, rows):
    """An infinite or NaN value of the prefix reaches all rows of the group and none of another, one behind it its sequence alone"""
    B = Groups(11, [n, 2], [150, 40], [9] * n + [3, 3], [rows] * (n + 2), 2, 64, 16)
    heads = 12
    fill_new(B)
    p, i = B.slot(0, 77)
    B.v[p, 0, i, 5] = np.inf
    p, i = B.slot(0, 149)
    B.v[p, 1, i, 6] = np.nan
    p, i = B.slot(1, 155)
    B.v[p, 0, i, 7] = -np.inf
    fills = B.k, B.v
    q = B.rng.standard_normal((B.total, heads * 64)) * 2.0
    q64, qt = held(q, act)
    cache, k64, v64 = on_gpu(pkg, B, kind)
    out = pkg.op_paged_prefix_attention(cache, qt, dev(B.row_start), rows, heads, 0.125, dev(B.group_start), dev(np.array(B.prefix, np.int32)))
    torch.cuda.synchronize()
    got = out.double().cpu().numpy().reshape(-1, heads, 64)
    with np.errstate(invalid="ignore"):
        want, *_ = B.definition(q64.reshape(-1, heads, 64), k64, v64, heads, 0.125)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isinf(got), np.isinf(want))
    inf = np.isinf(want)
    assert inf.any() and np.array_equal(got[inf], want[inf])
    ok = np.isfinite(want)
    assert np.abs(got[ok] - want[ok]).max() < (0.05 if act == "bf16" else 1e-4)
    assert fills is not None


def test_a_row_of_nan(pkg):
    """q of NaN makes its own row NaN, whatever the others are"""
    for act, kind in TYPES:
        B = Groups(12, [5], [100], [3] * 5, [1] * 5, 2, 64, 16)
        fill_new(B)
        q = B.rng.standard_normal((B.total, 6 * 64))
        _, qt = held(q, act)
        cache, *_ = on_gpu(pkg, B, kind)
        args = (dev(B.row_start), 1, 6, 0.125, dev(B.group_start), dev(np.array(B.prefix, np.int32)))
        clean = pkg.op_paged_prefix_attention(cache, qt, *args)
        qt[2, 64:128] = float("nan")
        got = pkg.op_paged_prefix_attention(cache, qt, *args)
        assert torch.isnan(got[2, 64:128]).all()
        got[2, 64:128] = clean[2, 64:128]
        assert torch.equal(got, clean)


def test_rows_beyond_their_most(pkg):
    """Rows behind a sequence's max_rows are left as they are"""
    B = Groups(13, [3], [64], [0, 5, 9], [2, 4, 1], 2, 64, 16)
    fill_new(B)
    q64, qt = held(B.rng.standard_normal((B.total, 6 * 64)), "f32")
    cache, k64, v64 = on_gpu(pkg, B, "f32")
    out = torch.full_like(qt, 7.5)
    pkg.op_paged_prefix_attention(cache, qt, dev(B.row_start), 2, 6, 0.125, dev(B.group_start), dev(np.array([64], np.int32)), out=out)
    want, _, mass, top = B.definition(q64.reshape(-1, 6, 64), k64, v64, 6, 0.125)
    got = out.double().cpu().numpy().reshape(-1, 6, 64)
    there = [0, 1, 2, 3, 6]
    near(got[there], want[there], mass[there], "f32", "f32", top, 64, 80)
    assert np.all(got[[4, 5]] == 7.5)


@pytest.mark.parametrize("act,kind", TYPES)
def test_the_same_call_gives_the_same_bits_and_what_attention_alone_gives(pkg, act, kind):
    B = Groups(14, [8, 8], [512, 256], [5 * i for i in range(16)], [1 + i % 3 for i in range(16)], 2, 128, 16)
    fill_new(B)
    _, qt = held(B.rng.standard_normal((B.total, 12 * 128)), act)
    cache, *_ = on_gpu(pkg, B, kind)
    args = (dev(B.row_start), 3, 12, 0.09, dev(B.group_start), dev(np.array(B.prefix, np.int32)))
    one, two = (pkg.op_paged_prefix_attention(cache, qt, *args) for _ in range(2))
    alone = pkg.op_paged_attention(cache, qt, dev(B.row_start), 3, 12, 0.09)
    assert torch.equal(one, two)
    # both are off by 600 half steps of f32 sums at most, and bf16 rows by a rounding of weights and of results each
    tol = 2.0 ** -7 * 6 if act == "bf16" else 2 * 600 * 2.0 ** -24 * 6
    assert (one.double() - alone.double()).abs().max() <= tol


def test_captured(pkg):
    """One graph serves lengths, prefixes and groups that change between its replays"""
    B = Groups(15, [4, 4], [256, 128], [30] * 8, [1] * 8, 2, 64, 16)
    fill_new(B)
    _, qt = held(B.rng.standard_normal((8, 12 * 64)), "bf16")
    cache, *_ = on_gpu(pkg, B, "bf16")
    row_start, group_start, prefix = dev(B.row_start), dev(B.group_start), dev(np.array(B.prefix, np.int32))
    scratch = pkg.op_paged_prefix_attention_scratch(cache, 8, 1, 12, 2)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        pkg.op_paged_prefix_attention(cache, qt, row_start, 1, 12, 0.125, group_start, prefix, scratch=scratch)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = pkg.op_paged_prefix_attention(cache, qt, row_start, 1, 12, 0.125, group_start, prefix, scratch=scratch)
        for lens, starts, shared in (([286] * 4 + [158] * 4, [0, 4, 8], [256, 128]), ([270] * 4 + [128, 129, 130, 140], [0, 4, 8], [240, 128]),
                                     ([280] * 4 + [150] * 4, [0, 4, 8], [0, 16]), ([260, 261, 262, 263] + [130] * 4, [0, 2, 4], [64, 256])):
            cache.length.copy_(dev(np.array(lens, np.int32)))
            group_start.copy_(dev(np.array(starts, np.int32)))
            prefix.copy_(dev(np.array(shared, np.int32)))
            qt.mul_(-1.0)
            graph.replay()
            stream.synchronize()
            got = out.clone()
            scratch_too = pkg.op_paged_prefix_attention(cache, qt, row_start, 1, 12, 0.125, group_start, prefix)   # eager work between
            alone = pkg.op_paged_attention(cache, qt, row_start, 1, 12, 0.125)
            stream.synchronize()
            assert torch.equal(got, scratch_too)
            assert (got.double() - alone.double()).abs().max() <= 2.0 ** -7 * 5


def test_two_streams(pkg):
    """Two batches at once, each with scratch memory of its own"""
    both = []
    for i in range(2):
        B = Groups(16 + i, [5, 9], [300, 170], [7 * j for j in range(14)], [1 + (i + j) % 2 for j in range(14)], 2, 128, 16)
        fill_new(B)
        _, qt = held(B.rng.standard_normal((B.total, 12 * 128)), "bf16")
        cache, *_ = on_gpu(pkg, B, "bf16")
        args = (cache, qt, dev(B.row_start), 2, 12, 0.09, dev(B.group_start), dev(np.array(B.prefix, np.int32)))
        both.append((args, pkg.op_paged_prefix_attention(*args), torch.cuda.Stream()))
    torch.cuda.synchronize()
    for rep in range(5):
        out = []
        for args, _, stream in both:
            with torch.cuda.stream(stream):
                out.append(pkg.op_paged_prefix_attention(*args))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, (_, b, _) in zip(out, both))


@pytest.mark.parametrize("act,kind", TYPES)
def test_groups_that_overlap_stay_inside_the_arrays(pkg, act, kind):
    """Group starts that decrease or pass the batch: what the rows get is unspecified, what lies around them is left as it is"""
    B = Groups(18, [4, 4], [64, 48], [3, 0, 9, 20, 1, 1, 30, 2], [1, 2, 0, 3, 1, 1, 2, 1], 2, 64, 16)
    fill_new(B)
    _, qt = held(B.rng.standard_normal((B.total + 3, 6 * 64)), act)
    cache, *_ = on_gpu(pkg, B, kind)
    for starts in ([0, 6, 2], [5, 1, 8], [-7, 4, 1 << 30], [8, 0, 8], [0, 0, 0]):
        out = torch.full_like(qt, 7.5)
        pkg.op_paged_prefix_attention(cache, qt, dev(B.row_start), 3, 6, 0.125, dev(np.array(starts, np.int32)), dev(np.array(B.prefix, np.int32)), out=out)
        torch.cuda.synchronize()
        assert bool((out[B.total:] == 7.5).all())
