"""Requests that share pages, and draws from rows of logits, restated on the host."""
import math

import numpy as np

from tests.util_paged import PAGE, Pool

ONE = 1 << 44


class SharedPool(Pool):
    """A pool whose pages may have several holders.  ``bytes`` [pages]: what a page holds, as a number that copies take along."""

    def __init__(self, requests, pages, max_length):
        super().__init__(requests, pages, max_length)
        self.holders = [0] * pages
        self.bytes = list(range(pages))

    def plan(self, rows, counts, T, max_count):
        got = super().plan(rows, counts, T, max_count)
        for t in self.table:
            for p in t:
                self.holders[p] = max(self.holders[p], 1)
        return got

    def fork(self, rows, into):
        lengths, tables = list(self.lengths), [list(t) for t in self.table]
        status, named, wanted, n_free = [], set(), 0, len(self.free)
        for r, t in zip(rows, into):
            first = 0 <= t < self.requests and t not in named
            named.add(t)
            if not first or not 0 <= r < self.requests or lengths[t] != 0:
                status.append(3)
                continue
            whole, part = divmod(lengths[r], PAGE)
            wanted += part > 0
            if part and wanted > n_free:
                status.append(1)
                continue
            status.append(0)
            self.table[t], self.lengths[t] = tables[r][:whole], lengths[r]
            for p in self.table[t]:
                self.holders[p] += 1
            if part:
                p = self.free.pop()
                self.table[t].append(p)
                self.holders[p], self.bytes[p] = 1, self.bytes[tables[r][whole]]
        return status

    def truncate(self, rows, keep):
        """Decisions on the pool as it is before; then what is given back, in the order of the sequences, by the last of those that give a page back."""
        status, seen, cuts, wanted, n_free = [], set(), [], 0, len(self.free)
        holders, was = list(self.holders), list(self.bytes)
        for i, (r, k) in enumerate(zip(rows, keep)):
            status.append(0)
            if not 0 <= r < self.requests or r in seen:
                continue
            seen.add(r)
            if not 0 <= k < self.lengths[r]:
                continue
            copy = k % PAGE > 0 and holders[self.table[r][k // PAGE]] > 1
            wanted += copy
            if copy and wanted > n_free:
                status[i] = 1
                continue
            cuts.append((i, r, k, self.free.pop() if copy else None))
        given = []
        for i, r, k, new in cuts:
            first = k // PAGE if new is not None else -(-k // PAGE)
            given += [(i, p) for p in self.table[r][first:]]
            if new is not None:
                self.bytes[new] = was[self.table[r][first]]
            self.table[r] = self.table[r][:first] + ([new] if new is not None else [])
            self.lengths[r] = k
        latest = {p: i for i, p in given}
        back = []
        for i, p in given:
            self.holders[p] -= 1
        for i, r, k, new in cuts:
            if new is not None:
                self.holders[new] = 1
        for i, p in given:
            if self.holders[p] == 0 and latest[p] == i:
                back.append(p)
        self.free += back[::-1]
        return status

    def agrees(self, cache):
        super().agrees(cache)
        assert cache._shared[0].tolist() == [max(h - 1, 0) for h in self.holders]
        assert cache._shared[1].tolist() == [-1] * cache.pages


def drawn(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The token that a row of numbers comes to, by the definition, in whole numbers of any length."""
    x = np.asarray(logits, dtype=np.float64)
    settings = (u, temperature, top_p, min_p)
    if np.isnan(x).any() or any(math.isnan(s) for s in settings) or x.max() == -math.inf or not 0 <= u <= 1 or not 0 <= temperature < math.inf:
        return -1
    m = x.max()
    if temperature == 0:
        return int(np.argmax(x))
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.rint(np.exp(np.where(x == m, 0.0, (x - m) * (1.0 / temperature))) * ONE)
    w = np.where(np.isnan(w), 0, w).astype(object)
    w = np.array([int(v) for v in w], dtype=object)
    kept = np.ones(len(x), bool)
    if 1 <= top_k < len(x):
        kept &= x >= np.sort(x)[-top_k]
    if top_p < 1:
        want = top_p * float(sum(w[kept]))
        order = np.argsort(-x, kind="stable")
        total, border = 0, None
        for i in order:
            if border is not None and x[i] < border:
                break
            if kept[i]:
                total += w[i]
                if border is None and float(total) >= want and total > 0:
                    border = x[i]
        kept &= x >= border
    kept &= np.array([float(v) >= min(min_p, 1.0) * ONE for v in w])
    total = sum(w[kept])
    target = min(math.floor(u * float(total)), total - 1)
    running = 0
    for i in np.nonzero(kept)[0]:
        running += w[i]
        if running > target:
            return int(i)
    raise AssertionError("no token")
