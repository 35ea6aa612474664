"""Beams over two prompts with a small two-layer model on a paged cache: forked, copied, appended, attended behind the shared prompt, ranked by log
probabilities and, in between, compacted. Every step is held to the same hypotheses computed alone, from their tokens, in 64 bits."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

HEADS, KV, DIM, WIDTH, VOCAB, LAYERS, PAGE = 6, 2, 64, 48, 500, 2, 16


def weights(rng):
    w = {"embed": rng.standard_normal((VOCAB, WIDTH))}
    for i in range(LAYERS):
        for name, n in (("q", HEADS * DIM), ("k", KV * DIM), ("v", KV * DIM)):
            w[f"{name}{i}"] = rng.standard_normal((WIDTH, n)) * WIDTH ** -0.5
        w[f"o{i}"] = rng.standard_normal((HEADS * DIM, WIDTH)) * (HEADS * DIM) ** -0.5
    return {k: v.astype(np.float32) for k, v in w.items()}


def turned(x, pos, heads):
    """[tokens][heads * dim] at their positions, dimension i with i + dim / 2"""
    x = x.reshape(len(pos), heads, DIM)
    a = pos[:, None, None] * 1e4 ** (-np.arange(DIM // 2) * 2.0 / DIM)
    u, v = x[..., :DIM // 2], x[..., DIM // 2:]
    return np.concatenate([u * np.cos(a) - v * np.sin(a), v * np.cos(a) + u * np.sin(a)], -1)


def alone(w, tokens):
    """log probabilities of the token behind these, all in 64 bits"""
    w = {k: v.astype(np.float64) for k, v in w.items()}
    pos = np.arange(len(tokens), dtype=np.float64)
    x = w["embed"][tokens]
    for i in range(LAYERS):
        q, k = turned(x @ w[f"q{i}"], pos, HEADS), turned(x @ w[f"k{i}"], pos, KV)
        v = (x @ w[f"v{i}"]).reshape(-1, KV, DIM)
        out = np.zeros_like(q)
        for h in range(HEADS):
            z = q[:, h] @ k[:, h // (HEADS // KV)].T * DIM ** -0.5
            z[pos[:, None] < pos[None, :]] = -np.inf
            p = np.exp(z - z.max(1, keepdims=True))
            out[:, h] = p / p.sum(1, keepdims=True) @ v[:, h // (HEADS // KV)]
        x = x + out.reshape(len(tokens), -1) @ w[f"o{i}"]
    z = x[-1] @ w["embed"].T * WIDTH ** -0.5
    return z - z.max() - np.log(np.exp(z - z.max()).sum())


class Beams:
    def __init__(self, pkg, w, prompts, width, n_pages, room):
        self.pkg, self.w, self.width = pkg, {k: torch.from_numpy(v).cuda() for k, v in w.items()}, width
        self.n = n = len(prompts) * width
        self.table = torch.full((n, room // PAGE), -1, dtype=torch.int32, device="cuda")
        self.length, self.refs = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros(n_pages, dtype=torch.int32, device="cuda")
        pool = (n_pages, KV, PAGE, DIM)
        # values that would show if a page were read that nobody wrote
        self.caches = [pkg.PagedCache(torch.full(pool, 1e6, device="cuda"), torch.full(pool, 1e6, device="cuda"), self.table, self.length) for _ in range(LAYERS)]
        angle = torch.arange(room, dtype=torch.float64, device="cuda")[:, None] * 1e4 ** (torch.arange(DIM // 2, dtype=torch.float64, device="cuda") * -2.0 / DIM)
        self.sin, self.cos = angle.sin().float(), angle.cos().float()
        self.group_start = torch.arange(0, n + 1, width, dtype=torch.int32, device="cuda")
        self.prefix = torch.zeros(len(prompts), dtype=torch.int32, device="cuda")

    def ints(self, v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    def step(self, tokens, rows, parent=None, top=0):
        """Rows of tokens behind the parents', what follows each sequence's last row"""
        pkg, w = self.pkg, self.w
        starts = np.concatenate([[0], np.cumsum(rows)])
        row_start, total, most = self.ints(starts), len(tokens), max(rows)
        moves, counts = pkg.op_paged_fork(self.caches[0], self.refs, parent=None if parent is None else self.ints(parent), row_start=row_start, rows=total,
                                          max_rows=most)
        pkg.op_paged_copy(self.caches, moves, counts)
        assert counts[1] == 0
        x = w["embed"][torch.tensor(tokens, device="cuda")]
        for i, cache in enumerate(self.caches):
            q = pkg.op_paged_append(cache, x @ w[f"q{i}"], x @ w[f"k{i}"], x @ w[f"v{i}"], row_start, self.sin, self.cos, max_rows=most)
            o = pkg.op_paged_prefix_attention(cache, q, row_start, most, HEADS, DIM ** -0.5, self.group_start, self.prefix)
            x = x + o @ w[f"o{i}"]
        self.length += self.ints(rows)
        last = torch.tensor([e - 1 for b, e in zip(starts, starts[1:]) if e > b], device="cuda")
        logits = (x[last] @ w["embed"].T) * WIDTH ** -0.5
        return pkg.op_token_logprobs(logits, top=top)

    def compact(self):
        moves, counts = self.pkg.op_paged_compact(self.caches[0], self.refs)
        self.pkg.op_paged_copy(self.caches, moves, counts)
        used = int((self.refs > 0).sum())
        assert counts.tolist()[1] == used and bool((self.refs[used:] == 0).all())


def test_beams(pkg):
    rng = np.random.default_rng(0)
    w, width, steps = weights(rng), 4, 21
    prompts = [list(rng.integers(0, VOCAB, n)) for n in (37, 64)]
    B = Beams(pkg, w, prompts, width, 60, 160)
    # the prompts are read by the first beam of each
    rows = [len(p) if j == 0 else 0 for p in prompts for j in range(width)]
    _, _, entropy, ids, lps = B.step(sum(prompts, []), rows, top=width)
    ids, lps, entropy = ids.cpu().numpy(), lps.double().cpu().numpy(), entropy.double().cpu().numpy()
    for g, p in enumerate(prompts):
        want = alone(w, p)
        assert np.abs(entropy[g] + (np.exp(want) * want).sum()) < 1e-4
    B.prefix.copy_(B.ints([len(p) for p in prompts]))
    live = [(list(p), 0.0) for p in prompts for _ in range(width)]
    parent = [g * width for g in range(len(prompts)) for _ in range(width)]
    token = [int(ids[g, j]) for g in range(len(prompts)) for j in range(width)]
    score = [lps[g, j] for g in range(len(prompts)) for j in range(width)]
    shared = 0
    for step in range(steps):
        live = [(live[p][0] + [t], s) for p, t, s in zip(parent, token, score)]
        *_, ids, lps = B.step(token, [1] * B.n, parent=parent, top=width)
        ids, lps = ids.cpu().numpy(), lps.double().cpu().numpy()
        for b, (tokens, _) in enumerate(live):
            want = alone(w, tokens)
            # f32 rows of 48 to 384 products in two layers: some 1e-6 of each logit, of which the largest is about 10
            assert np.abs(lps[b] - want[ids[b]]).max() < 1e-4, (step, b)
            assert np.abs(lps[b] - np.sort(want)[::-1][:width]).max() < 1e-4
        # the best of a group's continuations
        parent, token, score = [], [], []
        for g in range(len(prompts)):
            every = sorted(((live[b][1] + lps[b, j], b, int(ids[b, j])) for b in range(g * width, (g + 1) * width) for j in range(width)), reverse=True)
            for s, b, t in every[:width]:
                parent.append(b)
                token.append(t)
                score.append(s)
        shared += len(set(parent)) < B.n
        if step % 8 == 5:
            B.compact()
    assert shared > 0   # some step dropped a beam and forked another
    names = B.table[B.table >= 0].long().cpu()
    assert torch.equal(torch.bincount(names, minlength=60).int(), B.refs.cpu())


def test_answers_that_end_give_their_pages_back(pkg):
    rng = np.random.default_rng(1)
    w = weights(rng)
    prompt = list(rng.integers(0, VOCAB, 50))
    B = Beams(pkg, w, [prompt], 5, 40, 160)
    B.step(prompt, [50, 0, 0, 0, 0])
    B.prefix.fill_(50)
    B.step(list(rng.integers(0, VOCAB, 5)), [1] * 5, parent=[0] * 5)
    assert int((B.refs > 0).sum()) == 3 + 5   # three full pages, and each its own fourth
    B.step(list(rng.integers(0, VOCAB, 2)), [0, 1, 0, 1, 0], parent=[-1, 1, -1, 3, -1])
    assert int((B.refs > 0).sum()) == 3 + 2 and B.length.tolist() == [0, 52, 0, 52, 0]
    pkg.op_paged_fork(B.caches[0], B.refs, parent=B.ints([-1] * 5))
    assert bool((B.refs == 0).all()) and bool((B.table == -1).all()) and bool((B.length == 0).all())
