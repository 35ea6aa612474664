"""Sequences that go on with all of their tokens and have pages behind a place without one, as a length that was made smaller by hand can leave them: they
keep those, whichever way a fork of that size goes and whatever the other sequences do."""
import numpy as np
import pytest

import pages_model as model
from test_gpu_pages import run_fork

pytestmark = pytest.mark.gpu

PAGE = 16


@pytest.mark.parametrize("B,W,n_pages", [
    (4, 9, 60),           # one workgroup, a step that shares nothing
    (40, 33, 1500),
    (40, 33, 40000),      # a pool of more pages than one workgroup has room for
    (20, 2000, 41000),    # more places
    (600, 12, 8000),      # more sequences
])
@pytest.mark.parametrize("form", ["alone", "beside a shared page", "with kept lengths", "as its own parent"])
def test_pages_behind_a_hole_stay(pkg, B, W, n_pages, form):
    rng = np.random.default_rng(B + W)
    table = rng.permutation(n_pages)[:B * W].reshape(B, W)
    lens = [int(x) for x in rng.integers(0, (W // 2) * PAGE, B)]
    rows = [int(x) for x in rng.integers(0, 3, B)]
    need = [-(-(n + r) // PAGE) for n, r in zip(lens, rows)]
    for b in range(B):
        if b % 3 == 2:
            table[b, need[b]:] = -1                                  # an ordinary sequence
        else:
            table[b, need[b]:need[b] + 1 + b % 2] = -1               # the hole, and pages behind it
        if b % 5 == 1 and need[b]:
            table[b, need[b] - 1] = -1 if lens[b] <= (need[b] - 1) * PAGE else table[b, need[b] - 1]   # a place that wants a page
    if form == "beside a shared page":
        lens[-1], lens[-2], rows[-1], rows[-2] = 20, 24, 1, 1
        table[-2:], table[-1, :2] = -1, table[0, -2:]
        table[-2, :2] = table[-1, :2]
        need[-2:] = [2, 2]
        table[0, -2:] = -1
    parent = list(range(B)) if form == "as its own parent" else None
    keep = [n + b % 2 * 5 for b, n in enumerate(lens)] if form == "with kept lengths" else None
    refs = model.count(table, n_pages)
    visible = table.copy()
    for b in range(B):
        visible[b, need[b]:] = -1
    want, want_lens, _, pairs, missing = model.fork(visible, lens, refs, PAGE, parent, keep, rows)
    assert not missing
    for b in range(B):
        want[b, need[b]:] = table[b, need[b]:]
    assert (want[:, W // 2 + 2:] >= 0).any()
    cache, r, moves, counts = run_fork(pkg, table, lens, refs, PAGE, parent, keep, rows)
    assert counts.tolist() == [len(pairs), 0] and moves[:len(pairs)].tolist() == [list(p) for p in pairs]
    assert np.array_equal(cache.table.cpu().numpy(), want)
    assert np.array_equal(cache.length.cpu().numpy(), want_lens)
    assert np.array_equal(r.cpu().numpy(), model.count(want, n_pages))


@pytest.mark.parametrize("W,n_pages", [(12, 60), (12, 40000)])
def test_and_are_given_back_with_tokens(pkg, W, n_pages):
    """A kept length that ends in an earlier page, another parent or none gives them back"""
    table = np.full((4, W), -1)
    table[0], table[1], table[2], table[3, 0] = np.arange(12), np.arange(12, 24), np.arange(24, 36), 40
    table[:3, 3] = -1
    lens, refs = [40, 40, 40, 7], model.count(table, n_pages)
    for parent, keep in ((None, [32, 33, 0, 100]), ([-1, 3, 0, 3], None)):
        want, want_lens, want_refs, _, _ = model.fork(table, lens, refs, PAGE, parent, keep, None)
        if keep:
            want[1, 3:] = table[1, 3:]   # its tokens' places are the same
            want_refs = model.count(want, n_pages)
        cache, r, *_ = run_fork(pkg, table, lens, refs, PAGE, parent, keep, None)
        assert np.array_equal(cache.table.cpu().numpy(), want) and np.array_equal(cache.length.cpu().numpy(), want_lens)
        assert np.array_equal(r.cpu().numpy(), want_refs)
