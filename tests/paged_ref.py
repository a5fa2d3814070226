"""Plain forms of the paged cache's operators: the book in Python lists, attention and adjusted logits in 64 bits on the host."""

import math

import torch

RANGE, PAGES, NO_TOKEN = 1, 2, 4


class Book:
    """table, lengths, refs, and what each sequence's rows hold (any values)."""

    def __init__(self, sequences, entries, pages, T):
        self.table = [[] for _ in range(sequences)]
        self.lengths, self.refs = [0] * sequences, [0] * pages
        self.entries, self.T = entries, T
        self.err = 0
        self.moves = []  # (source page, target page) copies of the last call

    def pages_of(self, rows):
        return -(-rows // self.T)

    def take(self):
        p = self.refs.index(0)
        self.refs[p] = 1
        return p

    def extend(self, counts, n):
        """positions, rows, starts"""
        c = []
        for s, x in enumerate(counts):
            ok = 0 <= x <= self.entries * self.T - self.lengths[s]
            c.append(x if ok else 0)
            self.err |= 0 if ok else RANGE
        free, needed = self.refs.count(0), 0
        for s, x in enumerate(c):
            need = self.pages_of(self.lengths[s] + x) - self.pages_of(self.lengths[s])
            needed += need
            if need and needed > free:
                c[s], self.err = 0, self.err | PAGES
        total = 0
        for s, x in enumerate(c):
            total += x
            if x and total > n:
                c[s], self.err = 0, self.err | RANGE
        positions, rows, starts = [], [], [0]
        for s, x in enumerate(c):
            for p in range(self.lengths[s], self.lengths[s] + x):
                if p % self.T == 0:
                    self.table[s].append(self.take())
                positions.append(p)
                rows.append(self.table[s][p // self.T] * self.T + p % self.T)
            self.lengths[s] += x
            starts.append(len(rows))
        behind = n - len(rows)
        return positions + [0] * behind, rows + [-1] * behind, starts

    def fork(self, sources, targets):
        self.moves, S = [], len(self.lengths)
        named, free, needed = set(), self.refs.count(0), 0
        before = list(self.lengths)
        for a, b in zip(sources, targets):
            ok = 0 <= a < S and 0 <= b < S and a != b and before[b] == 0 and b not in named
            if 0 <= b < S:
                named.add(b)
            if not ok:
                self.err |= RANGE
                continue
            whole, part = divmod(before[a], self.T)
            needed += part > 0
            if part and needed > free:
                self.err |= PAGES
                continue
            for p in self.table[a][:whole]:
                self.refs[p] += 1
            self.table[b] = self.table[a][:whole]
            if part:
                self.table[b].append(self.take())
                self.moves.append((self.table[a][whole], self.table[b][whole]))
            self.lengths[b] = before[a]

    def free(self, sequences, keep=None):
        refs, done = list(self.refs), set()
        for i, s in enumerate(sequences):
            if not 0 <= s < len(self.lengths):
                self.err |= RANGE
                continue
            left = 0 if keep is None else min(keep[i], self.lengths[s])
            if s in done:
                continue
            done.add(s)
            if left < 0 or left < self.lengths[s] and left % self.T and refs[self.table[s][left // self.T]] > 1:
                self.err |= RANGE
                continue
            for p in self.table[s][self.pages_of(left):]:
                self.refs[p] -= 1
            self.table[s], self.lengths[s] = self.table[s][:self.pages_of(left)], left

    def compact(self):
        used = sum(r > 0 for r in self.refs)
        self.moves = list(zip([p for p in range(used, len(self.refs)) if self.refs[p] > 0], [p for p in range(used) if self.refs[p] == 0]))
        name = dict(self.moves)
        for a, b in self.moves:
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.table = [[name.get(p, p) for p in row] for row in self.table]
        return used

    def rows(self, s):
        """Rows of the pool that sequence s has, in order."""
        return torch.tensor([self.table[s][j // self.T] * self.T + j % self.T for j in range(self.lengths[s])], dtype=torch.int64)

    def check(self, cache, err=None):
        assert cache.lengths.tolist() == self.lengths
        assert cache.refs.tolist() == self.refs
        for got, want in zip(cache.table.tolist(), self.table):
            assert got[:len(want)] == want
        if err is not None:
            assert int(err.item()) == self.err


def attention(q, K, V, new, scale=None):
    """q (Hq, c, D), K/V (Hkv, rows, D) of one sequence: the 64-bit result (c, Hq, D) and a bound on a kernel's distance from it.

    A weight is rounded to bf16, off by at most 2^-8 of itself, in the products and in their sum alike: 2 2^-8 sum_j p_j |v_j|. The result is
    rounded to bf16: 2^-8 |out|. Scores in fp32: D + 2 roundings of 2^-24 of sum_d |q_d k_d| scale in the exponent, on the weights, twice; and
    the exponential, sums over rows and the joins' factors, 2^-18 together."""
    Hq, c, D = q.shape
    Hkv, rows = K.shape[:2]
    scale = D ** -0.5 if scale is None else scale
    q, K, V = q.double().cpu(), K.double().cpu(), V.double().cpu()
    out, bound = torch.zeros(c, Hq, D, dtype=torch.float64), torch.zeros(c, Hq, D, dtype=torch.float64)
    pos = torch.arange(rows - c, rows)
    seen = torch.arange(rows)[None] <= pos[:, None]
    for h in range(Hq):
        k, v = K[h // (Hq // Hkv)], V[h // (Hq // Hkv)]
        if rows == 0:
            continue
        x = (q[h] @ k.t() * scale).masked_fill(~seen, -math.inf)
        p = torch.where(seen.any(1, keepdim=True), torch.softmax(x, 1), torch.zeros((), dtype=torch.float64))
        size = (q[h].abs() @ k.abs().t() * scale).masked_fill(~seen, 0.0).amax(1, keepdim=True)
        out[:, h] = p @ v
        a = p @ v.abs()
        bound[:, h] = (2 * 2.0 ** -8 + 2 * (D + 2) * 2.0 ** -24 * size + 2.0 ** -18) * a + 2.0 ** -8 * (p @ v).abs()
    return torch.nan_to_num(out), torch.nan_to_num(bound) + 1e-30


def adjusted(logits, prompt=None, generated=None, repetition=1.0, frequency=0.0, presence=0.0, bias=None, allowed=None):
    """The adjusted logits in the steps and roundings of the definition (fp32, each once), on the host, with loops over the tokens."""
    x = logits.float().cpu().clone()
    b, n = x.shape
    of = lambda v, i: (v[i].cpu() if isinstance(v, torch.Tensor) else torch.tensor(float(v))).float()  # noqa: E731
    for i in range(b):
        count = {}
        for t in [] if generated is None else generated[i].tolist():
            if 0 <= t < n:
                count[t] = count.get(t, 0) + 1
        known = set(count) | {t for t in ([] if prompt is None else prompt[i].tolist()) if 0 <= t < n}
        r, f, p = of(repetition, i), of(frequency, i), of(presence, i)
        for t in known:
            v = x[i, t]
            v = v / r if v > 0 else v * r
            if t in count:
                v = (v - f * torch.tensor(float(count[t]))) - p
            x[i, t] = v
        if bias is not None:
            x[i] += (bias if bias.dim() == 1 else bias[i if bias.shape[0] > 1 else 0]).cpu()
        if allowed is not None:
            w = (allowed if allowed.dim() == 1 else allowed[i if allowed.shape[0] > 1 else 0]).cpu()
            at = torch.arange(n)
            x[i, ((w[at // 32] >> (at % 32)) & 1) == 0] = -math.inf
    return x


# Launches of attention over a paged cache that reach every kernel form: heads, sequences (rows, new tokens), most, whether all rows together are told
# (and then the rows of a tile, whether they are split, their joins spread, the sequences more than 64).
_7B, _05B = (28, 4, 128), (14, 2, 64)
FORMS = [
    (_05B, [(64, 1)], 1, False),  # 16, 0, 0, 0
    (_05B, [(64, 1)] + [(40, 1)] * 64, 1, False),  # 16, 0, 0, 1
    (_05B, [(1500, 20)] + [(40, 20)] * 9, 20, True),  # 16, 1, 0, 0
    (_05B, [(1500, 3)] + [(40, 3)] * 64, 3, True),  # 16, 1, 0, 1
    (_05B, [(1500, 1)], 1, False),  # 16, 1, 1, 0
    (_05B, [(1500, 1)] + [(40, 1)] * 65, 1, False),  # 16, 1, 1, 1
    (_05B, [(300, 60)] + [(64, 60)] * 9, 60, False),  # 32, 0, 0, 0
    (_05B, [(100, 8)] * 2 + [(40, 8)] * 64, 8, False),  # 32, 0, 0, 1
    (_05B, [(2000, 8)] + [(40, 8)] * 19, 8, False),  # 32, 1, 0, 0
    (_05B, [(2000, 3)] + [(40, 3)] * 64, 3, False),  # 32, 1, 0, 1
    (_05B, [(2000, 60)] + [(40, 40)] * 2, 60, False),  # 32, 1, 1, 0
    (_05B, [(2000, 4)] + [(40, 1)] * 64, 4, False),  # 32, 1, 1, 1
    (_05B, [(64, 40)] + [(64, 40)] * 9, 40, False),  # 128, 0, 0, 0
    (_05B, [(2500, 8)] + [(40, 8)] * 29, 8, False),  # 128, 1, 0, 0
    (_05B, [(2500, 40)] + [(40, 40)] * 9, 40, False),  # 128, 1, 1, 0
    (_7B, [(64, 1)], 1, False),  # 16, 0, 0, 0
    (_7B, [(64, 1)] + [(40, 1)] * 64, 1, False),  # 16, 0, 0, 1
    (_7B, [(1500, 8)] + [(100, 8)] * 9, 8, True),  # 16, 1, 0, 0
    (_7B, [(1500, 2)] + [(40, 2)] * 65, 2, True),  # 16, 1, 0, 1
    (_7B, [(900, 1)], 1, False),  # 16, 1, 1, 0
    ((3, 1, 128), [(900, 1)] + [(40, 1)] * 64, 1, False),  # 16, 1, 1, 1
    (_7B, [(100, 100)] + [(40, 40)], 100, False),  # 32, 0, 0, 0
    (_7B, [(64, 3)] * 2 + [(40, 3)] * 63, 3, False),  # 32, 0, 0, 1
    (_7B, [(1500, 12)] + [(40, 12)] * 9, 12, True),  # 32, 1, 0, 0
    (_7B, [(1500, 3)] + [(40, 3)] * 64, 3, True),  # 32, 1, 0, 1
    (_7B, [(1500, 12)] + [(40, 12)] * 4, 12, False),  # 32, 1, 1, 0
    ((3, 1, 128), [(1500, 8)] + [(40, 8)] * 64, 8, False),  # 32, 1, 1, 1
    (_7B, [(64, 60)] * 2, 60, False),  # 128, 0, 0, 0
    (_7B, [(2000, 5)] + [(40, 5)] * 19, 5, False),  # 128, 1, 0, 0
    (_7B, [(2000, 12)] + [(40, 12)] * 9, 12, False),  # 128, 1, 1, 0
]
