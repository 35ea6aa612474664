"""The pages of a paged cache, place by place in plain Python: what fork and compaction are held to."""
import numpy as np


def fork(table, lens, refs, page, parent=None, keep=None, rows=None):
    """-> table, lengths, refs, (from, to) pairs, pages missing"""
    B, W, n = len(table), len(table[0]), len(refs)
    old = [list(map(int, r)) for r in table]
    refs = list(map(int, refs))
    there = lambda p: 0 <= p < n  # noqa: E731
    new, length, wanted = [], [], []   # wanted: (sequence, place, whether it has tokens), of the places that rows write
    for b in range(B):
        p = b if parent is None else int(parent[b])
        known = 0 <= p < B
        t = max(0, int(lens[p])) if known else 0
        if keep is not None:
            t = min(t, max(0, int(keep[b])))
        r = 0 if rows is None else int(rows[b])
        kept = min(-(-t // page), W)
        need = max(kept, min(-(-(t + r) // page), W)) if r else kept
        new.append([(old[p][i] if i < kept else old[b][i] if p == b and i < need else -1) for i in range(W)])
        length.append(t)
        if r:
            wanted += [(b, i, i < kept) for i in range(t // page, need)]
    for which, step in ((old, -1), (new, 1)):
        for row in which:
            for p in row:
                if there(p) and refs[p] >= 0:
                    refs[p] += step
    who = {}
    for b, i, _ in wanted:
        p = new[b][i]
        if there(p) and refs[p] != 1:
            who.setdefault(p, []).append((b, i))
    leave = set()
    for p, writers in who.items():
        leave |= set(writers[:-1] if refs[p] == len(writers) else writers)
    for b, i in leave:
        if refs[new[b][i]] >= 0:
            refs[new[b][i]] -= 1
    fresh = [(b, i, full) for b, i, full in wanted if (b, i) in leave or (not there(new[b][i]) and not full)]
    free = [p for p in range(n) if refs[p] == 0]
    if len(fresh) > len(free):
        return table, lens, None, [], len(fresh) - len(free)
    pairs = []
    for (b, i, full), p in zip(fresh, free):
        if full:
            pairs.append((new[b][i], p))
        new[b][i] = p
        refs[p] = 1
    return np.array(new, np.int32), np.array(length, np.int32), np.array(refs, np.int32), pairs, 0


def compact(table, refs):
    """-> table, refs, (from, to) pairs, the number behind the last page in use"""
    refs = list(map(int, refs))
    used = sum(r != 0 for r in refs)
    pairs = list(zip([p for p in range(used, len(refs)) if refs[p] > 0], [p for p in range(used) if refs[p] == 0]))
    name = dict(pairs)
    for a, b in pairs:
        refs[b], refs[a] = refs[a], 0
    return (np.array([[name.get(int(p), int(p)) for p in row] for row in table], np.int32), np.array(refs, np.int32), pairs,
            max([p + 1 for p, r in enumerate(refs) if r], default=0))


def count(table, n_pages, held=()):
    """What refs says of a table"""
    refs = np.bincount(table[(table >= 0) & (table < n_pages)].ravel(), minlength=n_pages).astype(np.int32)
    refs[list(held)] = -1
    return refs


def pool(rng, B, W, page, n_pages, lens=None, share=0.5, holes=0.0, room=0.3):
    """A table of sequences that share some of their pages with earlier ones, some with room behind their tokens"""
    lens = [int(rng.integers(0, W * page + 1)) for _ in range(B)] if lens is None else lens
    table = np.full((B, W), -1, np.int32)
    free = list(rng.permutation(n_pages))
    for b, n in enumerate(lens):
        places = min(-(-max(0, n) // page), W)
        first = 0
        if b and rng.random() < share:
            other = int(rng.integers(0, b))
            first = int(rng.integers(0, min(places, -(-min(max(lens[other], 0), W * page) // page)) + 1))
            table[b, :first] = table[other, :first]
        for i in range(first, places):
            table[b, i] = free.pop()
        if places < W and rng.random() < room:
            table[b, places] = free.pop()
    table[(rng.random((B, W)) < holes) & (table >= 0)] = -1
    return table, lens
