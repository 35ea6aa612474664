"""A batch of sequences on a paged cache in plain numpy and 64 bits: what the paged operators are held to."""
import numpy as np

KINDS = {"f32": 4, "f16": 2, "bf16": 2}
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}   # half a step of each type, relative to the value


class Batch:
    """Pools of pages in an order of chance, with NaN wherever no token lies; page numbers behind a sequence's last page are -1."""

    def __init__(self, seed, lens, rows, kv, dim, page, spare=3, table_ld=None, weights=False, std_k=1.0):
        rng = self.rng = np.random.default_rng(seed)
        self.lens, self.rows, self.kv, self.dim, self.page = list(lens), list(rows), kv, dim, page
        need = [min(-(-(n + r) // page), table_ld or 1 << 30) for n, r in zip(lens, rows)]
        self.ld = table_ld or max(1, max(need))
        self.n_pages = sum(need) + spare
        order = rng.permutation(self.n_pages)
        self.table = np.full((len(lens), self.ld), -1, np.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        shape = (self.n_pages, kv, page)
        self.k, self.v = np.full((*shape, dim), np.nan), np.full((*shape, dim), np.nan)
        self.weight = np.full(shape, np.nan) if weights else None
        for b, n in enumerate(lens):
            for t in range(min(n, self.ld * page)):
                p, i = self.slot(b, t)
                self.k[p, :, i] = rng.standard_normal((kv, dim)) * std_k
                self.v[p, :, i] = rng.standard_normal((kv, dim))
                if weights:
                    self.weight[p, :, i] = rng.exponential(size=kv) ** 2
        self.row_start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        self.total = int(self.row_start[-1])

    def slot(self, b, t):
        return self.table[b, t // self.page], t % self.page

    def there(self, b, t):
        i = t // self.page
        return i < self.ld and 0 <= self.table[b, i] < self.n_pages


def rotate(x, pos, dims, sin, cos):
    """x [heads][dim] at one position, tables as the operator has them"""
    x = x.astype(np.float64)
    h = dims // 2
    if h == 0:
        return x
    s, c = sin[pos].astype(np.float64), cos[pos].astype(np.float64)
    a, b = x[:, :h], x[:, h:dims]
    return np.concatenate([a * c - b * s, b * c + a * s, x[:, dims:]], 1)


def attend(B, q, k, v, heads, scale, window=0, first=0):
    """q [rows][heads][dim], pools in 64 bits -> (out, weights added [pages][kv][page], sum of p |v|, largest score)"""
    out, mass = np.zeros((B.total, heads, B.dim)), np.zeros((B.total, heads, B.dim))
    added = np.zeros((B.n_pages, B.kv, B.page))
    G, top = heads // B.kv, 0.0
    for b, n in enumerate(B.lens):
        for j in range(B.rows[b]):
            s = n + j
            t = np.arange(min(s + 1, B.ld * B.page))
            page = B.table[b, t // B.page]
            seen = (page >= 0) & (page < B.n_pages)
            if window:
                seen &= (t > s - window) | (t < first)
            if not seen.any():
                continue
            pages, slots = page[seen], t[seen] % B.page
            for h in range(heads):
                kk, vv = k[pages, h // G, slots], v[pages, h // G, slots]
                with np.errstate(invalid="ignore", over="ignore"):
                    z = kk @ q[B.row_start[b] + j, h] * scale
                    top = max(top, np.abs(z[np.isfinite(z)]).max(initial=0.0))
                    p = np.exp(z - z.max())
                    p /= p.sum()
                    out[B.row_start[b] + j, h] = p @ vv
                    mass[B.row_start[b] + j, h] = p @ np.abs(vv)
                added[pages, h // G, slots] += p
    return out, added, mass, top


def evict(B, k, v, weight, budget, first, recent):
    """-> per sequence and head the slots that stay"""
    kept = np.full((len(B.lens), B.kv, budget), -1, np.int32)
    for b, n in enumerate(B.lens):
        for g in range(B.kv):
            w = np.array([weight[B.slot(b, t)[0], g, B.slot(b, t)[1]] if B.there(b, t) else 0.0 for t in range(n)])
            w = np.where(np.isnan(w), np.inf, w)
            safe = [t for t in range(n) if t < first or t >= n - recent]
            others = sorted((t for t in range(n) if first <= t < n - recent), key=lambda t: (-w[t], t))
            chosen = sorted(safe + others[:max(0, min(n, budget) - len(safe))])
            kept[b, g, :len(chosen)] = chosen
    return kept


def verify(logits, row_start, tokens, uniform, choice, temperature, draft=None):
    counts, nexts, near = [], [], []
    V = logits.shape[1]
    for b in range(len(row_start) - 1):
        accepted, token = 0, -1
        lo, hi = int(row_start[b]), int(row_start[b + 1])
        if lo == hi:
            counts.append(0)
            nexts.append(-1)
            continue
        for r in range(lo, hi):
            z = logits[r].astype(np.float64)
            t = int(tokens[r + 1]) if r + 1 < hi else None
            if temperature == 0:
                best = int(np.flatnonzero(z == np.nanmax(z))[0]) if np.nanmax(z, initial=-np.inf) > -np.inf else -1
                if t is not None and t == best and best >= 0:
                    accepted += 1
                    continue
                token = best
                break
            if not np.isfinite(z.max()):
                break
            with np.errstate(under="ignore"):
                p = np.exp((z - z.max()) / temperature)
                p /= p.sum()
                q = np.zeros(V)
                if t is not None and draft is not None:
                    y = draft[r].astype(np.float64)
                    q = np.exp((y - y.max()) / temperature)
                    q /= q.sum()
            if t is not None:
                known = 0 <= t < V
                if draft is None and known:
                    q[t] = 1.0
                a, c = float(uniform[r]) * (q[t] if known else 1.0), p[t] if known else 0.0
                if known and a < c:
                    accepted += 1
                    continue
                left = np.maximum(p - q, 0.0)
                if draft is None and known:
                    left[t] = 0.0
                p = left if left.sum() > 0 else p
            up = np.cumsum(p)
            mark = float(choice[b]) * up[-1]
            token = int(np.flatnonzero(up > mark)[0])
            break
        counts.append(accepted + 1)
        nexts.append(token)
    return np.array(counts, np.int32), np.array(nexts, np.int64)
