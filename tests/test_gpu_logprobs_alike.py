"""Log probabilities and entropies of rows in which all logits but a few are alike: whatever is rounded off one of them is rounded off all."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def definition(values, counts, T):
    """of `counts` logits of each value -> (log probabilities of the values, entropy) in long doubles"""
    d = (values.astype(np.longdouble) - values.max()) / np.longdouble(T)
    e = np.exp(d) * counts
    return d - np.log(e.sum()), np.log(e.sum()) - (e * d).sum() / e.sum()


@pytest.mark.parametrize("V", [1000, 32000, 151936, 1000000])
@pytest.mark.parametrize("everywhere", [False, True])
def test_roundings_that_add_up(pkg, V, everywhere):
    """One larger logit, or one in each block. With x the others' exponent: the difference of two logits, its product with 1 / T and the sum of that are off by
    half a step each, 2^-24 of x and 2 * 2^-20 of the power of two (x below 22 where it matters), an exponential by a step, a sum by half a step of each
    of its 22 additions: 1.3e-6 + 1.3e-6 + 1.2e-7 + 1.3e-6 of a logarithm. An entropy has x p (1 - p), 3.5 for a million tokens, times the first three
    and x p times the sums' of both its terms."""
    rng = np.random.default_rng(V + everywhere)
    for trial in range(40):
        T = float(rng.choice([1.0, 0.7, 1.3, rng.uniform(0.2, 3.0)]))
        z = np.full(V, rng.normal() * 5, np.float32)
        z[::1024 if everywhere else V] += np.float32(rng.uniform(0, 1.2 * np.log(V)) * T)
        values, counts = np.unique(z, return_counts=True)
        lps, entropy = definition(values, counts, T)
        tokens = torch.tensor([0, 1], device="cuda")
        lp, rank, ent, *_ = pkg.op_token_logprobs(torch.from_numpy(z).cuda().repeat(2, 1), tokens, temperature=T)
        want = [float(lps[values == z[t]][0]) for t in (0, 1)]
        assert np.all(np.abs(lp.double().cpu().numpy() - want) <= 4e-6 + 2.0 ** -24 * np.abs(want)), (trial, T)
        assert np.all(np.abs(ent.double().cpu().numpy() - float(entropy)) <= 3e-5 + 2.0 ** -24 * float(entropy)), (trial, T)
        assert rank.tolist() == [0, int(z[0] > z[1]) * len(z[::1024 if everywhere else V]) + (z[0] == z[1])]
