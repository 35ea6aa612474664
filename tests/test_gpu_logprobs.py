"""Log probabilities, ranks, entropies and the most probable tokens of rows of logits against their definitions in 64 bits."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def definition(z, tokens, top, T):
    """z f64 [rows][vocab] -> the operator's five outputs"""
    rows, V = z.shape
    lp, rank, ent = np.full(rows, np.nan), np.full(rows, -1), np.full(rows, np.nan)
    ids, lps = np.full((rows, top), -1), np.full((rows, top), np.nan)
    for r in range(rows):
        x = z[r]
        if np.isnan(x).any() or x.max() == np.inf or x.max() == -np.inf:
            continue
        with np.errstate(divide="ignore", invalid="ignore"):
            d = (x - x.max()) / T
            e = np.exp(d)
            logp = d - np.log(e.sum())
            p = e / e.sum()
            ent[r] = -np.sum(np.where(p > 0, p * logp, 0.0))
        t = int(tokens[r]) if tokens is not None else -1
        lp[r] = logp[t] if 0 <= t < V else -np.inf
        if 0 <= t < V:
            rank[r] = (x > x[t]).sum() + (x[:t] == x[t]).sum()
        order = np.lexsort((np.arange(V), -x))[:top]
        order = order[x[order] > -np.inf]
        ids[r, :len(order)] = order
        lps[r] = -np.inf
        lps[r, :len(order)] = logp[order]
    return lp, rank, ent, ids, lps


def near(got, want, what):
    """f32 sums of at most 1024 exponentials, each off by 2^-22 or so of its own: a logarithm is off by 2^-21 at most, an entropy, which
    has the mean of the exponents (below 2^4 for the logits here, each off by 2^-23 of it), by 2^-19; and the result is rounded."""
    got = got.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isinf(got), np.isinf(want)), what
    ok = np.isfinite(want)
    tol = (2.0 ** -19 if what == "entropy" else 2.0 ** -21) + 2.0 ** -23 * np.abs(want[ok])
    d = np.abs(got[ok] - want[ok])
    assert np.all(d <= tol), f"{what}: off by {(d - tol).max()} more than allowed"


def check(pkg, logits, tokens, top, T, scratch=None):
    if scratch is None:
        scratch = pkg.op_token_logprobs_scratch(*logits.shape, top)
        scratch.fill_(0xA5)
    got = pkg.op_token_logprobs(logits, tokens, top=top, temperature=T, scratch=scratch)
    torch.cuda.synchronize()
    want = definition(logits.double().cpu().numpy(), None if tokens is None else tokens.cpu().numpy(), top, T)
    near(got[2], want[2], "entropy")
    if tokens is None:
        assert got[0] is None and got[1] is None
    else:
        near(got[0], want[0], "logprob")
        assert np.array_equal(got[1].cpu().numpy(), want[1])
    if top == 0:
        assert got[3] is None and got[4] is None
    else:
        assert np.array_equal(got[3].cpu().numpy(), want[3])
        near(got[4], want[4], "top")


def logits_of(rows, V, kind, seed=0, std=2.5):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(rows, V, generator=gen, device="cuda") * std).to(TYPES[kind])


def some_tokens(rows, V, seed=0):
    return torch.from_numpy(np.random.default_rng(seed).integers(0, V, rows)).cuda()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,V", [(1, 1), (2, 2), (3, 63), (5, 1000), (2, 1024), (3, 1025), (4, 4095), (2, 4096), (7, 12289), (3, 32000), (2, 151936),
                                    (3, 152064)])
@pytest.mark.parametrize("top,T", [(0, 1.0), (1, 0.7), (5, 1.3), (64, 1.0)])
def test_logprobs(pkg, kind, rows, V, top, T):
    check(pkg, logits_of(rows, V, kind, V), some_tokens(rows, V, V), top, T)


@pytest.mark.parametrize("top", [0, 20])
def test_many_rows(pkg, top):
    check(pkg, logits_of(333, 5003, "f32"), some_tokens(333, 5003), top, 1.0)


@pytest.mark.parametrize("kind", TYPES)
def test_rows_apart(pkg, kind):
    """Rows of a wider buffer, on 16 bytes and off them"""
    wide = logits_of(6, 9000, kind)
    for lo, hi in ((0, 8192), (8, 8200), (1, 8001), (3, 3)):
        if hi > lo:
            check(pkg, wide[:, lo:hi], some_tokens(6, hi - lo), 7, 1.0)


def test_no_token_is_given(pkg):
    check(pkg, logits_of(4, 700, "f32"), None, 3, 1.0)
    check(pkg, logits_of(4, 700, "f32"), None, 0, 1.0)


@pytest.mark.parametrize("kind", TYPES)
def test_tokens_outside_the_vocabulary(pkg, kind):
    tokens = torch.tensor([-1, 3000, 1 << 40, -(1 << 62), 2999], device="cuda")
    check(pkg, logits_of(5, 3000, kind), tokens, 2, 1.0)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("V", [40, 5000, 70001])
def test_values_that_are_not_finite(pkg, kind, V):
    x = logits_of(9, V, kind)
    x[0, 7] = float("nan")
    x[1, V - 1] = float("inf")
    x[2] = float("-inf")
    x[3, : V - 1] = float("-inf")              # one token is certain
    x[4, 1:-1] = float("-inf")                 # two tokens
    x[5, ::2] = float("-inf")
    x[6] = torch.finfo(TYPES[kind]).min        # all masked by the lowest value: all the same
    x[7] = torch.finfo(TYPES[kind]).min
    x[7, 5] = 1.0
    x[8] = float("-inf")
    x[8, 1] = float("nan")                     # in a block that has nothing else
    check(pkg, x, torch.full((9,), V - 1, device="cuda"), 8, 1.0)
    check(pkg, x, torch.full((9,), 5, device="cuda"), 0, 0.5)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("V", [1000, 3000, 40000, 152064])
def test_equal_logits(pkg, kind, V):
    """Ties go by index, also where more reach the bound than are put in order by counting"""
    x = torch.zeros(6, V, device="cuda")
    x[1] = (torch.arange(V, device="cuda") % 3).float()
    x[2] = -(torch.arange(V, device="cuda") // 700).float()
    x[3, -3:] = 1.0
    x[4] = (torch.arange(V, device="cuda") % 1000 == 999).float()
    x[5] = torch.where(torch.arange(V, device="cuda") % 2 == 0, 0.0, -0.0)
    for top in (1, 20, 64, 1000):
        check(pkg, x.to(TYPES[kind]), some_tokens(6, V), top, 1.0)


def test_more_than_there_are(pkg):
    check(pkg, logits_of(3, 5, "f32"), some_tokens(3, 5), 9, 1.0)
    check(pkg, logits_of(3, 1500, "bf16"), some_tokens(3, 1500), 1024, 1.0)


def test_a_vocabulary_of_more_than_a_million(pkg):
    """More blocks than maxima that are compared"""
    V = 1024 * 1024 + 12345
    check(pkg, logits_of(2, V, "f32"), some_tokens(2, V), 33, 1.0)
    check(pkg, torch.zeros(1, V, dtype=torch.bfloat16, device="cuda"), some_tokens(1, V), 10, 1.0)


@pytest.mark.parametrize("T", [1e-30, 1e-3, 0.1, 100.0, 1e30])
def test_temperatures(pkg, T):
    x = logits_of(4, 3001, "f32")
    got = pkg.op_token_logprobs(x, some_tokens(4, 3001), top=4, temperature=T)
    want = definition(x.double().cpu().numpy(), some_tokens(4, 3001).cpu().numpy(), 4, T)
    for g, w in ((got[0], want[0]), (got[2], want[2]), (got[4], want[4])):   # a quotient's rounding, on top
        g = g.double().cpu().numpy()
        assert np.all(np.abs(g - w) <= 2.0 ** -19 + 2.0 ** -22 * np.abs(w)), (T, g, w)
    assert np.array_equal(got[1].cpu().numpy(), want[1]) and np.array_equal(got[3].cpu().numpy(), want[3])


@pytest.mark.parametrize("T", [1e-30, 1e-8, 1e30])
def test_masked_logits_at_any_temperature(pkg, T):
    """Differences that pass f32 once they are divided leave nothing, and no NaN"""
    x = logits_of(5, 1500, "f32")
    x[:, 100:900] = float("-inf")
    x[1, 50] = -3e38
    x[2, 7] = 3e38
    tokens = torch.tensor([3, 50, 7, 500, 1499], device="cuda")
    got = [g.double().cpu().numpy() for g in pkg.op_token_logprobs(x, tokens, top=4, temperature=T)]
    want = definition(x.double().cpu().numpy(), tokens.cpu().numpy(), 4, T)
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[3], want[3])
    for g, w in ((got[0], want[0]), (got[2], want[2]), (got[4], want[4])):
        w = np.where(np.abs(w) > np.finfo(np.float32).max, np.sign(w) * np.inf, w)   # as f32 holds it
        ok = np.isfinite(w)
        assert np.array_equal(g[~ok], w[~ok]) and np.all(np.abs(g[ok] - w[ok]) <= 2.0 ** -19 + 2.0 ** -22 * np.abs(w[ok])), (T, g, w)


def test_large_logits(pkg):
    x = logits_of(3, 2000, "f32", std=1.0)
    check(pkg, x + 5e4, some_tokens(3, 2000), 3, 1.0)
    check(pkg, x - 3e6, some_tokens(3, 2000), 3, 1.0)
    x[:, 3] = 3e38
    x[:, 4] = -3e38
    check(pkg, x, torch.full((3,), 3, device="cuda"), 3, 1.0)


def test_a_sure_row_has_next_to_no_entropy(pkg):
    """Nothing cancels: an entropy of 2e-12 is right to the last bits"""
    x = torch.zeros(1, 2000, device="cuda")
    x[0, 77] = 38.0
    got = float(pkg.op_token_logprobs(x)[2])
    e = np.exp(-38.0) * 1999
    want = np.log1p(e) + 38.0 * e / (1 + e)
    assert abs(got - want) <= 2.0 ** -24 + 1e-6 * want


def test_captured(pkg):
    x, tokens = logits_of(5, 30000, "bf16"), some_tokens(5, 30000)
    scratch = pkg.op_token_logprobs_scratch(5, 30000, 10)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        pkg.op_token_logprobs(x, tokens, top=10, scratch=scratch)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = pkg.op_token_logprobs(x, tokens, top=10, scratch=scratch)
        for i in range(4):
            x.copy_(logits_of(5, 30000, "bf16", seed=10 + i))
            tokens.copy_(some_tokens(5, 30000, seed=i))
            graph.replay()
            stream.synchronize()
            eager = pkg.op_token_logprobs(x, tokens, top=10)
            stream.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, eager))


@pytest.mark.parametrize("kind", TYPES)
def test_nan_of_either_sign(pkg, kind):
    bits = torch.int32 if kind == "f32" else torch.int16
    x = logits_of(6, 2500, kind)
    minus = x[:, 0].clone().fill_(float("nan")).view(bits)
    minus |= torch.iinfo(bits).min
    for r, at in enumerate((0, 700, 1024, 2047, 2499)):
        x.view(bits)[r, at] = minus[r]
    assert bool(torch.signbit(x[:5][torch.isnan(x[:5])]).all()) and int(torch.isnan(x).sum()) == 5
    check(pkg, x, some_tokens(6, 2500), 4, 1.0)
    check(pkg, x, some_tokens(6, 2500), 0, 1.0)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("V", [262144, 262145, 524288, 524289])
def test_as_many_chunks_as_are_kept(pkg, kind, V):
    """Vocabularies whose chunks' maxima just have room in LDS, and larger ones"""
    for top in (1, 50):
        check(pkg, logits_of(3, V, kind, V), some_tokens(3, V), top, 0.8)
    check(pkg, (torch.arange(V, device="cuda") % 1000 == 999).to(TYPES[kind])[None], some_tokens(1, V), 700, 1.0)


@pytest.mark.parametrize("kind", TYPES)
def test_ranks_among_equal_logits(pkg, kind):
    """The given token at blocks' borders: equal ones in front of it come before it, those behind it do not"""
    V = 3500
    tokens = torch.tensor([0, 1, 1023, 1024, 1025, 2047, 2048, 3071, 3073, 3499, 63, 64], device="cuda")
    x = (torch.arange(V, device="cuda") % 2).to(TYPES[kind]).repeat(len(tokens), 1)
    check(pkg, x, tokens, 0, 1.0)
    check(pkg, x * 0, tokens, 2, 1.0)
    x[:, ::3] = float("-inf")
    check(pkg, x, tokens, 3, 1.0)
