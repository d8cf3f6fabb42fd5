"""What the operators between two passes of a model do, written out on the host in 64 bits, one sequence and one entry at a time."""
import math

import numpy as np


def weights(row, tau):
    """P of a row of logits (largest: 1), all zero where there is nothing to choose."""
    row = np.where(np.isnan(row), -np.inf, row)
    top = row.max()
    if top == -np.inf:
        return np.zeros_like(row)
    if not tau > 0:
        p = np.zeros_like(row)
        p[int(row.argmax())] = 1.0
        return p
    if top == np.inf:
        return (row == np.inf).astype(np.float64)
    if tau == np.inf:
        return (row > -np.inf).astype(np.float64)
    return np.exp((row - top) / tau)


def pick(w, u):
    """The smallest place at which the running sum passes u of the whole; the last with any weight where none does."""
    if not w.sum() > 0:
        return -1
    run = np.cumsum(w)
    over = np.flatnonzero((run > u * run[-1]) & (w > 0))
    return int(over[0]) if len(over) else int(np.flatnonzero(w)[-1])


def walk(logits, tokens, parent, u_accept, u_next, tau, draft, max_path):
    """(path, next token) of one tree, by p <- norm(max(p - q, 0)) for every child that falls (not the running form of the kernel)."""
    n, vocabulary = logits.shape
    if n == 0:
        return [], -1
    path, node = [], 0
    while True:
        path.append(node)
        p = weights(logits[node], tau)
        if not p.sum() > 0:
            return path, -1
        p = p / p.sum()
        kept = p.copy()                                      # P without the tokens that fell
        q = None if draft is None or not tau > 0 else np.maximum(np.nan_to_num(draft[node], nan=0.0), 0.0)
        left, fallen, after = 1.0, set(), None
        for child in range(node + 1, n) if len(path) < max_path else ():
            if parent[child] != node:
                continue
            x = int(tokens[child])
            if not 0 <= x < vocabulary or x in fallen:
                continue
            u = float(u_accept[child])
            drawn = q is not None and q[x] > 0 and left > 0
            if u * (q[x] / left) < p[x] if drawn else u < p[x]:
                after = child
                break
            if drawn:
                p = np.maximum(p - q / left, 0.0)
                left -= q[x]
            fallen.add(x)
            kept[x] = 0.0
            p[list(fallen)] = 0.0
            if p.sum() > 0:
                p = p / p.sum()
        if after is None:
            for w in (p, kept, weights(logits[node], tau)):
                if w.sum() > 0:
                    return path, pick(w, float(u_next))
            return path, -1
        node = after


def verify(logits, tokens, parent, starts, u_accept, u_next, tau, draft, max_path):
    """(path, counts, next tokens) of a batch; all arguments numpy, tau one per sequence."""
    batch = len(starts) - 1
    path = np.full((batch, max_path), -1, dtype=np.int64)
    counts, following = np.zeros(batch, dtype=np.int64), np.zeros(batch, dtype=np.int64)
    for b in range(batch):
        s = slice(max(0, min(starts[b], len(tokens))), max(0, min(starts[b + 1], len(tokens))))
        nodes, following[b] = walk(logits[s], tokens[s], parent[s], u_accept[s], u_next[b], tau[b], None if draft is None else draft[s], max_path)
        path[b, :len(nodes)], counts[b] = nodes, len(nodes)
    return path, counts, following


class Server:
    """Page table, references, lengths and pools of a program, on the host: `pools` is a list of numpy arrays
    [pages, heads, page, ...] (bytes; rows and exponents alike)."""

    def __init__(self, table, refs, lens, pools, page):
        self.table, self.refs, self.lens, self.page = table.copy(), refs.copy(), lens.copy(), page
        self.pools = [p.copy() for p in pools]

    def named(self, p):
        return 0 <= p < len(self.refs)

    def copy_rows(self, old, new, rows):
        for p in self.pools:
            p[new, :, :rows] = p[old, :, :rows]

    def fit(self, lens):
        free = [i for i, r in enumerate(self.refs) if r <= 0]
        before, missing = self.refs.copy(), np.zeros(len(lens), dtype=np.int32)
        for b, n in enumerate(lens):
            n = min(max(int(n), 0), self.table.shape[1] * self.page)
            keep = math.ceil(n / self.page)
            for s in range(self.table.shape[1]):
                p = int(self.table[b, s])
                if s >= keep:
                    if self.named(p):
                        self.refs[p] -= 1
                    self.table[b, s] = -1
                elif not self.named(p):
                    self.table[b, s] = -1
                    if free:
                        self.table[b, s] = free.pop(0)
                        self.refs[self.table[b, s]] = 1
                    else:
                        missing[b] += 1
                elif s == keep - 1 and n % self.page and before[p] > 1:
                    if free:
                        self.table[b, s] = free.pop(0)
                        self.refs[self.table[b, s]] = 1
                        self.refs[p] -= 1
                        self.copy_rows(p, self.table[b, s], n % self.page)
                    else:
                        missing[b] += 1
        return missing

    def fork(self, sources, targets):
        free = [i for i, r in enumerate(self.refs) if r <= 0]
        table, lens, slots = self.table.copy(), self.lens.copy(), len(self.lens)
        missing, seen = np.zeros(len(sources), dtype=np.int32), set()
        for i, (a, t) in enumerate(zip(sources, targets)):
            if not (0 <= a < slots and 0 <= t < slots) or t in seen:
                continue
            seen.add(t)
            if a == t:
                continue
            n = min(max(int(lens[a]), 0), table.shape[1] * self.page)
            keep = math.ceil(n / self.page)
            row = [int(p) if s < keep and self.named(p) else -1 for s, p in enumerate(table[a])]
            for p in table[t]:
                if self.named(p):
                    self.refs[p] -= 1
            if n % self.page and row[keep - 1] >= 0:
                if free:
                    new = free.pop(0)
                    self.refs[new] = 1
                    self.copy_rows(row[keep - 1], new, n % self.page)
                    for p in row[:keep - 1]:
                        if p >= 0:
                            self.refs[p] += 1
                    row[keep - 1] = new
                else:
                    row, n, missing[i] = [-1] * len(row), 0, 1
            else:
                for p in row:
                    if p >= 0:
                        self.refs[p] += 1
            self.table[t], self.lens[t] = row, n
        return missing

    def compact(self, path, counts, lens, starts):
        out = np.zeros(len(lens), dtype=np.int32)
        for b, n in enumerate(lens):
            n = min(max(int(n), 0), self.table.shape[1] * self.page)
            fresh = min(max(int(starts[b + 1]) - int(starts[b]), 0), n)
            count = min(max(int(counts[b]), 0), fresh, path.shape[1])
            for i in range(count):
                p = int(path[b, i])
                if 0 <= p < fresh:
                    old, new = divmod(n - fresh + p, self.page), divmod(n - fresh + i, self.page)
                    a, c = int(self.table[b, old[0]]), int(self.table[b, new[0]])
                    if self.named(a) and self.named(c):
                        for x in self.pools:
                            x[c, :, new[1]] = x[a, :, old[1]]
            out[b] = n - fresh + count
        return out
