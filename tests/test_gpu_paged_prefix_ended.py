"""Attention behind shared prefixes in groups whose first sequences have ended, as a fork without a parent leaves them: no tokens, no pages."""
import numpy as np
import pytest
import torch

import paged_model as pm
from test_gpu_beams import VOCAB, Beams, alone, weights
from test_gpu_paged import TYPES, dev, fill_new, held, near, on_gpu

pytestmark = pytest.mark.gpu


def grouped(seed, counts, prefix, own, rows, kv, dim, page, ended=(), shorter=()):
    """(batch, group starts): counts[g] sequences have the same prefix[g] tokens, in the same pages but for the one in which the prefix ends, of which each
    has a copy, as forks leave them. `ended` have nothing, `shorter` (sequence: tokens) have given some of theirs back; neither has rows."""
    starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    of = [g for g, n in enumerate(counts) for _ in range(n)]
    B = pm.Batch(seed, [prefix[g] + n for g, n in zip(of, own)], rows, kv, dim, page)
    fill_new(B)
    for b, g in enumerate(of):
        full = prefix[g] // page
        B.table[b, :full] = B.table[starts[g], :full]
        for t in range(full * page, prefix[g]):
            (p, i), (o, _) = B.slot(b, t), B.slot(starts[g], t)
            B.k[p, :, i], B.v[p, :, i] = B.k[o, :, i], B.v[o, :, i]
    for b in ended:
        assert rows[b] == 0
        B.table[b], B.lens[b] = -1, 0
    for b, n in dict(shorter).items():
        assert rows[b] == 0
        B.table[b, -(-n // page):], B.lens[b] = -1, n
    return B, starts


def run(pkg, B, starts, prefix, act, kind, heads):
    q64, q = held(B.rng.standard_normal((B.total, heads * B.dim)) * 2.0, act)
    cache, k64, v64 = on_gpu(pkg, B, kind)
    scale, most = B.dim ** -0.5, max(B.rows)
    got = pkg.op_paged_prefix_attention(cache, q, dev(B.row_start), most, heads, scale, dev(starts), dev(np.array(prefix, np.int32)))
    torch.cuda.synchronize()
    want, _, mass, top = pm.attend(B, q64.reshape(-1, heads, B.dim), k64, v64, heads, scale)
    near(got.double().cpu().numpy().reshape(-1, heads, B.dim), want, mass, act, kind, top, B.dim, max(n + r for n, r in zip(B.lens, B.rows)))


# sequences of groups, prefixes, own tokens, rows, ended, with fewer tokens than the prefix
CASES = [
    ([5], [50], [0, 3, 0, 9, 1], [0, 1, 0, 1, 0], [0, 2, 4], {}),
    ([4], [130], [5, 0, 40, 7], [0, 0, 2, 3], [0], {1: 129}),                                      # the first that has the prefix is the third
    ([4], [130], [5, 0, 40, 7], [0, 0, 2, 3], [], {0: 16, 1: 130}),                                # the second has just as much, and no rows
    ([3, 4], [64, 200], [1, 2, 3, 4, 5, 6, 7], [0, 1, 1, 0, 0, 4, 1], [0, 3, 4], {}),
    ([3], [100], [0, 5, 9], [0, 40, 70], [0], {}),                                                 # prompts
    ([70], [90], [i % 20 for i in range(70)], [0] * 66 + [1, 0, 2, 1], range(66), {}),            # dealt by a launch in front, over 64 in front of the first
    ([66, 3], [33, 80], [i % 9 for i in range(69)], [0] + [1] * 65 + [0, 2, 1], [0, 66], {}),
    ([3] * 10, [20 + 9 * g for g in range(10)], [i % 7 for i in range(30)], [0, 1, 2] * 10, range(0, 30, 3), {}),   # more groups than are gone through one by one
]


@pytest.mark.parametrize("act,kind", TYPES)
@pytest.mark.parametrize("counts,prefix,own,rows,ended,shorter", CASES)
def test_first_sequences_without_the_prefix(pkg, act, kind, counts, prefix, own, rows, ended, shorter):
    B, starts = grouped(20, counts, prefix, own, rows, 2, 64, 16, ended, shorter)
    run(pkg, B, starts, prefix, act, kind, 6)


def test_answers_go_on_when_others_have_ended(pkg):
    """Five answers to one prompt, of which the first, third and fifth end: the others' log probabilities are those of their tokens alone"""
    rng = np.random.default_rng(1)
    w = weights(rng)
    prompt = list(rng.integers(0, VOCAB, 50))
    B = Beams(pkg, w, [prompt], 5, 40, 160)
    B.step(prompt, [50, 0, 0, 0, 0])
    B.prefix.fill_(50)
    answers = [[int(t)] for t in rng.integers(0, VOCAB, 5)]
    B.step([a[0] for a in answers], [1] * 5, parent=[0] * 5)
    parent = [-1, 1, -1, 3, -1]
    for step in range(3):
        for b in (1, 3):
            answers[b].append(int(rng.integers(0, VOCAB)))
        *_, ids, lps = B.step([answers[1][-1], answers[3][-1]], [0, 1, 0, 1, 0], parent=parent if step == 0 else None, top=20)
        ids, lps = ids.cpu().numpy(), lps.double().cpu().numpy()
        for r, b in enumerate((1, 3)):
            # f32 rows of 48 to 384 products in two layers: some 1e-6 of each logit, of which the largest is about 10
            assert np.abs(lps[r] - alone(w, prompt + answers[b])[ids[r]]).max() < 1e-4, (step, b)
