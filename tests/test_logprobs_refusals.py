"""What log probabilities of tokens refuse, on the host alone: no call here gets past its checks."""
import ctypes

import pytest

EINVAL, ESHAPE = -1, -2
P = 1 << 20   # an address on 16 bytes: nothing reads it


def call(pkg, scratch=P, size=1 << 50, **kw):
    base = dict(d_logits=P, d_tokens=P, d_logprob=P, d_rank=P, d_entropy=P, d_top_token=P, d_top_logprob=P, rows=3, vocab=100, ldl=100, dtype=1, top=5,
                temperature=1.0)
    a = pkg.LogprobsArgs(**{**base, **kw})
    return pkg.lib().w4a32_op_token_logprobs(ctypes.byref(a), scratch, size, None)


@pytest.mark.parametrize("bad", [
    dict(d_logits=None), dict(rows=0), dict(vocab=0), dict(top=-1), dict(ldl=99), dict(dtype=0), dict(dtype=4), dict(temperature=0.0), dict(temperature=-1.0),
    dict(temperature=float("nan")), dict(temperature=float("inf")), dict(temperature=1e-31), dict(temperature=1e31), dict(d_tokens=None),
    dict(d_top_token=None), dict(d_top_logprob=None), dict(d_logits=P + 2), dict(d_logits=P + 1, dtype=3), dict(d_tokens=P + 4), dict(d_logprob=P + 2),
    dict(d_rank=P + 1), dict(d_entropy=P + 2), dict(d_top_token=P + 4), dict(d_top_logprob=P + 2), dict(scratch=None), dict(scratch=P + 8), dict(size=0)])
def test_arguments(pkg, bad):
    assert call(pkg, **bad) == EINVAL


@pytest.mark.parametrize("bad", [dict(rows=1 << 24), dict(rows=1 << 20, vocab=1 << 16, ldl=1 << 16), dict(vocab=1 << 30, ldl=1 << 30), dict(top=1025),
                                 dict(rows=1 << 22)])
def test_sizes(pkg, bad):
    assert call(pkg, **bad) == ESHAPE
    sizes = {**dict(rows=3, vocab=100, top=5), **{k: v for k, v in bad.items() if k != "ldl"}}
    assert pkg.lib().w4a32_op_token_logprobs_scratch_bytes(sizes["rows"], sizes["vocab"], sizes["top"]) == 0


def test_room(pkg):
    need = pkg.lib().w4a32_op_token_logprobs_scratch_bytes(3, 100, 5)
    assert need > 0 and call(pkg, size=need - 1) == EINVAL
    for bad in ((0, 100, 5), (3, 0, 5), (3, 100, -1)):
        assert pkg.lib().w4a32_op_token_logprobs_scratch_bytes(*bad) == 0
