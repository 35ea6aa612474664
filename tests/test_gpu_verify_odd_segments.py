"""Verification of drafted tokens where a row's NaN stands in a part of the vocabulary that has nothing else."""
import numpy as np
import pytest

from test_gpu_paged import check_verify, drafted

pytestmark = pytest.mark.gpu

INF, NAN = np.inf, np.nan


def spoil(row, how):
    if how == "behind":          # the last logit, by itself behind 4096 others
        row[4096] = NAN
    elif how == "masked":        # among logits of -infinity
        row[4096:8192] = -INF
        row[5003] = NAN
    elif how == "all":           # nothing else for 4096 logits
        row[4096:8192] = NAN
    elif how == "whole":         # nothing else at all
        row[:] = NAN
    else:                        # two parts of -infinity, a NaN in one of them
        row[:8192] = -INF
        row[0] = NAN


@pytest.mark.parametrize("how,V", [("behind", 4097), ("masked", 12300), ("all", 12300), ("whole", 8200), ("parts", 300001)])
@pytest.mark.parametrize("draft", [False, True])
def test_a_nan_leaves_no_distribution(pkg, how, V, draft):
    """Sequences 0 to 2: the NaN in the row that judges the first token, in the row behind an accepted token, in the last row;
    3: none; 4: in the draft model's row. The tokens in front are the target's and the draft's most probable by far."""
    rng = np.random.default_rng(40)
    starts, logits, other, tokens, uniform, choice = drafted(rng, [2, 3, 2, 2, 2], V, draft)
    at = 17   # of a sequence's tokens
    for x in (logits, other) if draft else (logits,):
        x[:, at] = 60.0
    tokens[:] = at
    for r in (0, 3, 6):
        spoil(logits[r], how)
    counts, nexts = [1, 2, 2, 2, 2], [-1, -1, -1, at, at]
    if draft:
        spoil(other[9], how)
        counts[4], nexts[4] = 1, -1
    want = np.array(counts, np.int32), np.array(nexts, np.int64)
    check_verify(pkg, starts, logits, other, tokens, uniform, choice, 1.0, want=want)
    check_verify(pkg, starts, logits, other, tokens, uniform, choice, 0.2, want=want)
