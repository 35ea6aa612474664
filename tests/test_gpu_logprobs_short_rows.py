"""Log probabilities over vocabularies of a few tokens, whose rows are shorter than one load of 16 bytes."""
import pytest
import torch

from test_gpu_logprobs import TYPES, check, logits_of, some_tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("V", list(range(1, 10)))
def test_few_tokens(pkg, kind, V):
    """Rows on 16 bytes and off them, with places for more tokens than there are"""
    x = logits_of(1, 4096, kind, V)
    for at in (4096 - V, (4096 - V) // 16 * 16):   # off 16 bytes and on them
        for top in (0, 1, V, 20):
            check(pkg, x[:, at:at + V], some_tokens(1, V, V), top, 1.0)
    check(pkg, logits_of(3, V, kind, V), some_tokens(3, V, V), V, 0.7)
