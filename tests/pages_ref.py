"""Plain restatements of the paged cache's operators, for the tests: the bookkeeping step by step on Python lists, the attention in 64 bits."""
import numpy as np
import torch

F64 = torch.float64


class State:
    """Table, lengths and reference counts as lists; every method follows the documented rules entry by entry."""

    def __init__(self, S, M, P, page):
        self.table, self.lens, self.refs, self.page = [[-1] * M for _ in range(S)], [0] * S, [0] * P, page
        self.S, self.M, self.P = S, M, P

    def free(self, rows, begin=None, end=None):
        seen = set()
        for i, r in enumerate(rows):
            if not 0 <= r < self.S or r in seen:
                continue
            seen.add(r)
            n = self.lens[r]
            b = max(0, begin[i]) if begin else 0
            e = min(n, end[i]) if end else n
            for p in range(self.M):
                if p * self.page >= b and p * self.page < n and min((p + 1) * self.page, n) <= e and self.table[r][p] >= 0:
                    self.refs[self.table[r][p]] -= 1
                    self.table[r][p] = -1
            if e >= n:
                self.lens[r] = min(n, b)

    def fork(self, src, dst, tokens=None):
        before, out, seen = list(self.lens), [], set()
        rows = [list(t) for t in self.table]
        for i, (s, d) in enumerate(zip(src, dst)):
            if not 0 <= s < self.S or not 0 <= d < self.S or s == d or before[d] != 0 or d in seen:
                out.append(-1)
                seen.add(d)
                continue
            seen.add(d)
            n = before[s] if tokens is None else max(0, min(tokens[i], before[s]))
            for p in range(-(-n // self.page)):
                e = rows[s][p]
                self.table[d][p] = e
                if e >= 0:
                    self.refs[e] += 1
            if n:
                self.lens[d] = n
            out.append(n)
        return out

    def reserve(self, rows, counts):
        free = [p for p in range(self.P) if self.refs[p] == 0]
        refs = list(self.refs)
        used, positions, copies, seen = 0, [], [], set()
        for r, c in zip(rows, counts):
            known = 0 <= r < self.S and r not in seen
            seen.add(r)
            if not known or c < 0 or self.lens[r] + c > self.M * self.page:
                positions.append(-1)
                copies.append((-1, -1))
                continue
            n = self.lens[r]
            cols = list(range(-(-n // self.page), -(-(n + c) // self.page)))
            old = None
            if c > 0 and n % self.page:
                last = self.table[r][n // self.page]
                if last < 0 or refs[last] > 1:
                    cols.insert(0, n // self.page)
                    old = last
            used += len(cols)
            if cols and used > len(free):
                positions.append(-1)
                copies.append((-1, -1))
                continue
            pair = (-1, -1)
            for k, p in enumerate(cols):
                page = free[used - len(cols) + k]
                if k == 0 and old is not None and old >= 0:
                    pair = (old, page)
                    self.refs[old] -= 1
                self.table[r][p] = page
                self.refs[page] = 1
            self.lens[r] = n + c
            positions.append(n)
            copies.append(pair)
        return positions, copies

    def compact(self):
        live = [p for p in range(self.P) if self.refs[p] > 0]
        n = len(live)
        holes = [p for p in range(n) if self.refs[p] <= 0]
        remap = [p if self.refs[p] > 0 and p < n else -1 for p in range(self.P)]
        moves = []
        for p, h in zip([p for p in live if p >= n], holes):
            remap[p] = h
            moves.append((p, h))
            self.refs[h], self.refs[p] = self.refs[p], 0
        self.table = [[remap[e] if e >= 0 else -1 for e in row] for row in self.table]
        return remap, moves


def seen(n, window, sinks):
    return [t for t in range(n) if window <= 0 or t < sinks or t >= n - window]


def decode(q, k, v, scale, keep):
    """One query head: q [D], k / v [T, D] fp64 arrays, keep = visible rows.  Returns the output and p."""
    if len(keep) == 0:
        return np.zeros(v.shape[-1]), np.zeros(0)
    s = k[keep] @ q * scale
    p = np.exp(s - s.max())
    p /= p.sum()
    return p @ v[keep], p
