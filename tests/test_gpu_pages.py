"""Forking, copying and compacting the pages of a paged cache against plain Python."""
import numpy as np
import pytest
import torch

import pages_model as model

pytestmark = pytest.mark.gpu


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def cache_of(pkg, table, lens, page, n_pages, kv=1, dim=8, dtype=torch.bfloat16, fill=None, weight=False):
    shape = (n_pages, kv, page, dim)
    k, v = (torch.zeros(shape, dtype=dtype, device="cuda") if fill is None else fill(shape).to(dtype) for _ in range(2))
    w = fill(shape[:3]) if weight else None
    return pkg.PagedCache(k, v, dev(table), dev(lens), w)


def starts(rows):
    return np.concatenate([[0], np.cumsum(rows)])


def run_fork(pkg, table, lens, refs, page, parent=None, keep=None, rows=None, pad=0, scratch=None, max_rows=None):
    cache, r = cache_of(pkg, table, lens, page, len(refs)), dev(refs)
    total = 0 if rows is None else max(1, int(sum(rows)) + pad)
    if scratch is None:   # of any contents
        scratch = pkg.op_paged_fork_scratch(cache, total)
        scratch.fill_(0xA5)
    moves, counts = pkg.op_paged_fork(cache, r, parent=None if parent is None else dev(parent), keep=None if keep is None else dev(keep),
                                      row_start=None if rows is None else dev(starts(rows)), rows=total,
                                      max_rows=max_rows if max_rows or rows is None else max(1, max(rows)), scratch=scratch)
    torch.cuda.synchronize()
    return cache, r, moves.cpu().numpy(), counts.cpu().numpy()


def check_fork(pkg, table, lens, refs, page, parent=None, keep=None, rows=None, pad=0):
    want_table, want_lens, want_refs, pairs, missing = model.fork(table, lens, refs, page, parent, keep, rows)
    cache, r, moves, counts = run_fork(pkg, table, lens, refs, page, parent, keep, rows, pad)
    assert counts.tolist() == [len(pairs), missing]
    assert np.array_equal(cache.table.cpu().numpy(), want_table)
    assert np.array_equal(cache.length.cpu().numpy(), want_lens)
    assert np.array_equal(r.cpu().numpy(), refs if missing else want_refs)
    assert moves.tolist() == [list(p) for p in pairs] + [[-1, -1]] * (len(table) - len(pairs))
    return want_table, want_lens, want_refs, pairs


def test_one_prompt_and_its_answers(pkg):
    """A prompt of 37 tokens in pages of 16 becomes four answers: three copies of its last page, the last one keeps the page itself"""
    table = np.full((4, 4), -1)
    table[0, :3] = [5, 2, 7]
    got, _, refs, pairs = check_fork(pkg, table, [37, 0, 0, 0], model.count(table, 9), 16, parent=[0, 0, 0, 0], rows=[1, 1, 1, 1])
    assert got[:, :3].tolist() == [[5, 2, 0], [5, 2, 1], [5, 2, 3], [5, 2, 7]]
    assert pairs == [(7, 0), (7, 1), (7, 3)] and refs.tolist() == [1, 1, 4, 1, 0, 4, 0, 1, 0]


def test_where_a_page_ends(pkg):
    """No copy where the tokens fill their pages; a row more than a page has room for takes two"""
    table = np.array([[3, 1, -1, -1], [-1, -1, -1, -1]])
    got, *_, pairs = check_fork(pkg, table, [32, 0], model.count(table, 8), 16, parent=[0, 0], rows=[16, 17])
    assert got.tolist() == [[3, 1, 0, -1], [3, 1, 2, 4]] and not pairs


def test_a_new_and_an_ended_sequence(pkg):
    table = np.array([[0, 1], [2, 3], [4, -1]])
    check_fork(pkg, table, [20, 32, 7], model.count(table, 6), 16, parent=[-1, 2, 99], rows=[3, 1, 0])


def test_tokens_taken_back(pkg):
    """Pages behind what stays are free again, and rows get room once more"""
    table = np.array([[0, 1, 2, 3], [4, 5, 6, -1]])
    check_fork(pkg, table, [64, 40], model.count(table, 8), 16, keep=[17, 40], rows=[1, 2])
    check_fork(pkg, table, [64, 40], model.count(table, 8), 16, keep=[0, -5])
    check_fork(pkg, table, [64, 40], model.count(table, 8), 16, keep=[100, 33], rows=[0, 0])


def test_pages_of_someone_else(pkg):
    """A system prompt that no sequence owns: it is copied before it is written and never freed"""
    table = np.array([[2, 4, -1], [2, 4, -1], [-1, -1, -1]])
    refs = model.count(table, 8, held=[2, 4, 6])
    check_fork(pkg, table, [20, 32, 0], refs, 16, rows=[1, 1, 1])
    check_fork(pkg, table, [20, 32, 0], refs, 16, parent=[-1, -1, -1], rows=[1, 0, 40])


def test_too_few_pages_change_nothing(pkg):
    table = np.array([[0, 1, -1], [2, 3, -1], [4, -1, -1]])
    for n in (5, 6):
        check_fork(pkg, table, [32, 32, 16], model.count(table, n), 16, rows=[1, 1, 1])
    check_fork(pkg, table, [32, 32, 16], model.count(table, 8), 16, rows=[1, 1, 1])
    # pages that the same call frees are there
    check_fork(pkg, table, [32, 32, 16], model.count(table, 5), 16, parent=[0, -1, 2], rows=[1, 0, 1])


def test_places_that_are_not_there(pkg):
    """Holes, numbers outside the pool, lengths past the table and below zero"""
    table = np.array([[-1, 1, 9, -1], [3, 1 << 30, 2, -7], [4, 5, 6, 7], [-1, -1, -1, -1]])
    for lens in ([40, 40, 70, 0], [1, 30, -4, 3], [33, 1 << 30, 64, 5]):
        for rows in ([1, 1, 1, 1], [20, 0, 5, 70], None):
            check_fork(pkg, table, lens, model.count(table, 14), 16, rows=rows)
            check_fork(pkg, table, lens, model.count(table, 14), 16, parent=[1, 0, 3, 2], rows=rows)


@pytest.mark.parametrize("seed", range(40))
def test_fork(pkg, seed):
    rng = np.random.default_rng(seed)
    B, W, page = int(rng.integers(1, 40)), int(rng.integers(1, 30)), int(2 ** rng.integers(4, 8))
    n_pages = B * (W + 1) + int(rng.integers(0, 80))
    table, lens = model.pool(rng, B, W, page, n_pages, holes=0.1 if seed % 5 == 4 else 0.0)
    refs = model.count(table, n_pages, held=rng.choice(n_pages, int(rng.integers(0, 4)), replace=False))
    parent = [int(x) for x in rng.integers(-1, B + (seed % 3 == 0), B)] if seed % 4 else None
    keep = [int(x) for x in rng.integers(0, W * page + 1, B)] if seed % 3 == 1 else None
    rows = [int(x) for x in rng.integers(0, (4, 3 * page)[seed % 2], B)] if seed % 7 else None
    print(seed, B, W, page, n_pages, flush=True)
    check_fork(pkg, table, lens, refs, page, parent, keep, rows, pad=seed % 6)


@pytest.mark.parametrize("B,W,page,n_pages", [
    (1500, 5, 16, 12000),     # more sequences than the workgroup that settles them has threads
    (3, 20000, 16, 70000),    # long tables, many pages
    (300, 400, 16, 150000),
    (256, 64, 16, 18000),     # as many places as one workgroup takes of sequences that change, and more
    (257, 64, 16, 18000),
    (500, 1, 16, 700),        # a place each
    (512, 33, 32, 18000),
])
def test_large_forks(pkg, B, W, page, n_pages):
    rng = np.random.default_rng(B)
    table, lens = model.pool(rng, B, W, page, n_pages)
    parent = [int(x) for x in rng.integers(0, B, B)]
    check_fork(pkg, table, lens, model.count(table, n_pages), page, parent, None, [int(x) for x in rng.integers(0, 60, B)])
    check_fork(pkg, table, lens, model.count(table, n_pages), page, None, [int(n * rng.random()) for n in lens], [1] * B)


@pytest.mark.parametrize("B,W,n_pages", [(512, 64, 32768), (512, 61, 32000), (300, 109, 32768)])
def test_many_sequences_that_end(pkg, B, W, n_pages):
    """Some sequences have become shorter and give pages back, pages of others are shared: one workgroup, all that it has room for"""
    rng = np.random.default_rng(W)
    table, lens = model.pool(rng, B, W, 16, n_pages)
    lens = [int(n * rng.random()) if b % 3 == 0 else n for b, n in enumerate(lens)]
    table[7, :3], table[8, :3], lens[7], lens[8] = table[20, :3], table[20, :3], 40, 33
    check_fork(pkg, table, lens, model.count(table, n_pages), 16, None, None, [b % 3 for b in range(B)])


@pytest.mark.parametrize("B,W", [(3, 9), (40, 33), (1, 20000), (512, 64), (300, 200)])
@pytest.mark.parametrize("forked", [False, True])
def test_pages_behind_a_hole(pkg, B, W, forked):
    """A sequence that keeps nothing, or has no parent, gives up all of its pages, those behind places that name none too"""
    n_pages = B * W + 5
    table = np.random.default_rng(W).permutation(n_pages)[:B * W].reshape(B, W)
    table[:, :W // 2] = -1                       # pages that a window has left behind
    lens, rows, ends = [W * 16] * B, [b % 2 for b in range(B)], [b % 2 == 0 for b in range(B)]
    parent, keep = ([-1 if e else b for b, e in enumerate(ends)], None) if forked else (None, [0 if e else 1 << 30 for e in ends])
    check_fork(pkg, table, lens, model.count(table, n_pages), 16, parent, keep, rows)


def test_a_prompt_of_many_pages(pkg):
    table = np.full((2, 600), -1)
    table[1, :2] = [3, 4]
    check_fork(pkg, table, [0, 20], model.count(table, 1300), 16, rows=[9000, 7], pad=11)


def test_rows_beyond_their_most(pkg):
    """A sequence has room for max_rows rows at most, and none behind the buffers' rows"""
    table = np.full((3, 8), -1)
    cache, r, moves, counts = run_fork(pkg, table, [0, 0, 0], model.count(table, 30), 16, rows=[40, 3, 50], max_rows=17)
    assert (cache.table.cpu().numpy() >= 0).sum(1).tolist() == [2, 1, 2] and counts.tolist() == [0, 0]
    cache = cache_of(pkg, table, [0, 0, 0], 16, 30)
    pkg.op_paged_fork(cache, dev(model.count(table, 30)), row_start=dev([0, 40, 43, 93]), rows=41, max_rows=40)
    assert (cache.table.cpu().numpy() >= 0).sum(1).tolist() == [3, 1, 0]
    # row starts that decrease: nothing outside the arrays, whatever the rows get
    cache, refs = cache_of(pkg, table, [0, 0, 0], 16, 30), dev(model.count(table, 30))
    pkg.op_paged_fork(cache, refs, row_start=dev([0, 40, 0, 40]), rows=40, max_rows=40)
    got = cache.table.cpu().numpy()
    assert np.array_equal(model.count(got, 30), refs.cpu().numpy()) and refs.max() <= 1


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kv,dim,page,layers,weight", [(1, 8, 16, 1, False), (2, 72, 32, 3, True), (4, 128, 16, 37, True), (3, 256, 128, 2, False)])
def test_copy(pkg, dtype, kv, dim, page, layers, weight):
    gen = torch.Generator(device="cuda").manual_seed(dim)
    n_pages = 23

    def fill(shape):
        return torch.randn(shape, generator=gen, device="cuda")

    table = np.full((1, 1), -1)
    caches = [cache_of(pkg, table, [0], page, n_pages, kv, dim, dtype, fill, weight) for _ in range(layers)]
    before = [[x.clone() for x in (c.k, c.v, c.weight) if x is not None] for c in caches]
    pairs = [(3, 20), (3, 0), (22, 7), (-1, 5), (4, 23), (1 << 30, 6), (9, -2), (11, 21), (1, 2)]
    moves = dev(pairs)
    pkg.op_paged_copy(caches, moves, dev([len(pairs) - 1, 0]))   # the last pair is not counted
    torch.cuda.synchronize()
    for c, old in zip(caches, before):
        for x, o in zip([y for y in (c.k, c.v, c.weight) if y is not None], old):
            want = o.clone()
            for a, b in pairs[:-1]:
                if 0 <= a < n_pages and 0 <= b < n_pages:
                    want[b] = o[a]
            assert torch.equal(x, want)
    kept = [x.clone() for x in (caches[0].k, caches[0].v)]
    for n in (0, -3):
        pkg.op_paged_copy(caches[0], moves, dev([n]))
    pkg.op_paged_copy(caches[0], moves[:0], dev([0]))
    assert torch.equal(caches[0].k, kept[0]) and torch.equal(caches[0].v, kept[1])


def test_a_count_beyond_the_list(pkg):
    cache = cache_of(pkg, np.full((1, 1), -1), [0], 16, 6, fill=lambda s: torch.randn(s, device="cuda"))
    moves = dev([(0, 1), (2, 3), (4, 5)])
    old = cache.k.clone()
    pkg.op_paged_copy(cache, moves[:2], dev([1 << 30]))
    assert torch.equal(cache.k[3], old[2]) and torch.equal(cache.k[5], old[5])


def test_pools_beyond_32_bits(pkg):
    """Pages whose places pass 2^31 elements and 2^32 bytes of the pools"""
    n_pages, kv, page, dim = 270000, 8, 16, 128
    k = torch.empty((n_pages, kv, page, dim), dtype=torch.bfloat16, device="cuda")
    cache = pkg.PagedCache(k, torch.empty_like(k), dev(np.full((1, 1), -1)), dev([0]))
    for x in (cache.k, cache.v):
        x[1], x[n_pages - 1], x[135000] = 1.0, 2.0, 3.0
    pkg.op_paged_copy(cache, dev([(n_pages - 1, 0), (1, n_pages - 2), (135000, 200000)]), dev([3]))
    for x in (cache.k, cache.v):
        assert (x[0] == 2.0).all() and (x[n_pages - 2] == 1.0).all() and (x[200000] == 3.0).all()


def check_compact(pkg, table, refs):
    want_table, want_refs, pairs, end = model.compact(table, refs)
    cache, r = cache_of(pkg, table, [0] * len(table), 16, len(refs)), dev(refs)
    scratch = pkg.op_paged_compact_scratch(cache)
    scratch.fill_(0xA5)
    moves, counts = pkg.op_paged_compact(cache, r, scratch=scratch)
    torch.cuda.synchronize()
    assert counts.tolist() == [len(pairs), end]
    assert np.array_equal(cache.table.cpu().numpy(), want_table)
    assert np.array_equal(r.cpu().numpy(), want_refs)
    assert moves.tolist() == [list(p) for p in pairs] + [[-1, -1]] * (len(refs) // 2 - len(pairs))


@pytest.mark.parametrize("n_pages", [1, 2, 63, 64, 65, 129, 1000, 4096, 4097, 5000, 8192, 8193, 65536, 65537, 70000])
@pytest.mark.parametrize("held", [0, 3])
def test_compact(pkg, n_pages, held):
    rng = np.random.default_rng(n_pages + held)
    for used in sorted({0, 1, n_pages // 3, n_pages - 1, n_pages}):
        table = np.full((3, max(1, used)), -1)
        pages = rng.permutation(n_pages)[:used]
        table[1, :used] = pages
        table[0, :used // 2] = pages[:used // 2]   # shared
        table[2, 0] = n_pages + 5                  # nobody's
        refs = model.count(table, n_pages, held=rng.choice(n_pages, min(held, n_pages), replace=False))
        print(n_pages, held, used, flush=True)
        check_compact(pkg, table, refs)


def test_a_large_pool_is_compacted(pkg):
    rng = np.random.default_rng(0)
    n = 300000
    table = np.full((7, 30000), -1)
    table[:, :25000] = rng.permutation(n)[:7 * 25000].reshape(7, 25000)
    check_compact(pkg, table, model.count(table, n, held=[299999, 5]))


def test_captured(pkg):
    """Fork and copies in one graph, replayed on other lengths, with eager work between; two graphs share nothing"""
    page, n_pages, B, W = 16, 64, 4, 6
    gen = torch.Generator(device="cuda").manual_seed(0)

    def fill(shape):
        return torch.randn(shape, generator=gen, device="cuda")

    table = np.full((B, W), -1)
    table[0, :2] = [9, 4]
    cache, refs = cache_of(pkg, table, [20, 0, 0, 0], page, n_pages, 2, 64, torch.float32, fill), dev(model.count(table, n_pages))
    parent, row_start = dev([0, 0, 0, 0]), dev([0, 1, 2, 3, 4])
    scratch = pkg.op_paged_fork_scratch(cache, 4)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())

    def step():
        moves, counts = pkg.op_paged_fork(cache, refs, parent=parent, row_start=row_start, rows=4, max_rows=1, scratch=scratch)
        pkg.op_paged_copy(cache, moves, counts)
        return moves, counts

    with torch.cuda.stream(stream):
        saved = [x.clone() for x in (cache.table, cache.length, refs)]
        step()
        stream.synchronize()
        for x, y in zip((cache.table, cache.length, refs), saved):
            x.copy_(y)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            moves, counts = step()
        rng = np.random.default_rng(1)
        for i in range(6):
            before = [x.cpu().numpy() for x in (cache.table, cache.length, refs)]
            k = cache.k.clone()
            graph.replay()
            stream.synchronize()
            t, n, r, pairs, missing = model.fork(*before, page, parent=parent.cpu().numpy(), rows=[1] * B)
            assert not missing and counts.tolist() == [len(pairs), 0] and moves.tolist()[:len(pairs)] == [list(p) for p in pairs]
            for x, y in zip((cache.table, cache.length, refs), (t, n, r)):
                assert np.array_equal(x.cpu().numpy(), y)
            for a, b in pairs:
                k[b] = k[a]
            assert torch.equal(cache.k, k)
            cache.length.add_(1)   # eager work between the replays
            parent.copy_(dev(rng.integers(0, B, B)))
            stream.synchronize()


def test_on_another_stream_beside_another_call(pkg):
    """Two batches at once, each with scratch memory of its own"""
    rng = np.random.default_rng(5)
    both = []
    for i in range(2):
        table, lens = model.pool(rng, 20, 50, 16, 1500)
        refs = model.count(table, 1500)
        both.append((table, lens, refs, cache_of(pkg, table, lens, 16, 1500), dev(refs), dev(starts([3] * 20)), torch.cuda.Stream()))
    torch.cuda.synchronize()
    out = []
    for *_, cache, refs, row_start, stream in both:
        with torch.cuda.stream(stream):
            out.append(pkg.op_paged_fork(cache, refs, row_start=row_start, rows=60, max_rows=3))
    torch.cuda.synchronize()
    for (table, lens, refs, cache, r, *_), (moves, counts) in zip(both, out):
        t, n, c, pairs, missing = model.fork(table, lens, refs, 16, rows=[3] * 20)
        assert counts.tolist() == [len(pairs), missing] and np.array_equal(cache.table.cpu().numpy(), t) and np.array_equal(r.cpu().numpy(), c)


@pytest.mark.parametrize("n_pages", [200, 9000])
def test_compaction_captured(pkg, n_pages):
    """One graph, replayed on other tables with eager work between"""
    rng = np.random.default_rng(n_pages)
    cache = cache_of(pkg, np.full((4, n_pages // 4), -1), [0] * 4, 16, n_pages)
    refs, scratch = dev(np.zeros(n_pages)), pkg.op_paged_compact_scratch(cache)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        pkg.op_paged_compact(cache, refs, scratch=scratch)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            moves, counts = pkg.op_paged_compact(cache, refs, scratch=scratch)
        for i in range(4):
            table = np.full((4, n_pages // 4), -1)
            table.ravel()[:n_pages // 3] = rng.permutation(n_pages)[:n_pages // 3]
            before = model.count(table, n_pages)
            cache.table.copy_(dev(table))
            refs.copy_(dev(before))
            graph.replay()
            stream.synchronize()
            want, after, pairs, end = model.compact(table, before)
            assert counts.tolist() == [len(pairs), end] and np.array_equal(cache.table.cpu().numpy(), want) and np.array_equal(refs.cpu().numpy(), after)
            assert moves.tolist()[:len(pairs)] == [list(p) for p in pairs]
