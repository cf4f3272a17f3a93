"""The paged 4-bit cache restated on the host: the pool as lists, the rounding number by number, attention in 64 bits."""
import math

import torch

PAGE = 64


class Pool:
    """Pages and slots of requests, one after the other."""

    def __init__(self, requests, pages, max_length):
        self.requests, self.pages, self.max_length = requests, pages, max_length
        self.free = list(range(pages - 1, -1, -1))
        self.table = [[] for _ in range(requests)]
        self.lengths = [0] * requests

    def plan(self, rows, counts, T, max_count):
        starts, ends, status, positions, slots = [0], [], [], [-1] * T, [-1] * T
        at, seen, dry = 0, set(), False
        wanted, n_free = 0, len(self.free)
        for row, count in zip(rows, counts):
            n, s = max(count, 0), 0
            named = 0 <= row < self.requests
            if count < 0 or (n > 0 and (not named or row in seen)):
                s = 3
            elif at + n > T:
                s = 4
            elif n > max_count or self.lengths[row if named else 0] * named + n > self.max_length:
                s = 2
            if n > 0 and named:
                seen.add(row)
            if s == 0 and n > 0:
                need = -(-(self.lengths[row] + n) // PAGE) - len(self.table[row])
                wanted += need
                if need > 0 and wanted > n_free:
                    s = 1
                else:
                    for _ in range(need):
                        self.table[row].append(self.free.pop())
                    for r in range(n):
                        p = self.lengths[row] + r
                        positions[at + r], slots[at + r] = p, self.table[row][p // PAGE] * PAGE + p % PAGE
                    self.lengths[row] += n
            status.append(s)
            ends.append(row if s == 0 and named else None)
            at += n
            starts.append(min(at, T))
        ends = [0 if row is None else self.lengths[row] for row in ends]
        return dict(starts=starts, ends=ends, status=status, positions=positions, slots=slots)

    def truncate(self, rows, keep):
        back, seen = [], set()
        for row, k in zip(rows, keep):
            if not 0 <= row < self.requests or row in seen:
                continue
            seen.add(row)
            if 0 <= k < self.lengths[row]:
                first = -(-k // PAGE)
                back += self.table[row][first:]
                self.table[row] = self.table[row][:first]
                self.lengths[row] = k
        self.free += back[::-1]

    def agrees(self, cache):
        width = cache.width
        table = [t + [-1] * (width - len(t)) for t in self.table]
        n = int(cache.n_free)
        assert n == len(self.free)
        assert cache.free[:n].tolist() == self.free
        assert cache.table.tolist() == table
        assert cache.lengths.tolist() == self.lengths


def held_as(x, group):
    """What the cache holds for ``x [..., D]`` of its type, in fp32 steps as the definition has them; the value in 64 bits."""
    g = x.float().unflatten(-1, (-1, group))
    lo, hi = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
    s = ((hi - lo) * torch.tensor(1.0 / 15.0, dtype=torch.float32)).to(x.dtype).float()
    c = torch.where(s > 0, ((g - lo) / torch.where(s > 0, s, torch.ones_like(s))).round().clamp(0, 15), torch.zeros_like(g))
    bad = ~torch.isfinite(g).all(-1, keepdim=True) | ~torch.isfinite(s)
    v = c.double() * s.double() + lo.double()
    return torch.where(bad, math.nan, v).flatten(-2)


def turned(x, positions, rope):
    """Pairs of neighbours turned in fp32, each product and sum rounded, and rounded to the type of ``x``."""
    cs = rope[positions.long()][:, None]
    a, b = x.float()[..., 0::2], x.float()[..., 1::2]
    c, s = cs[..., 0], cs[..., 1]
    return torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2).to(x.dtype)


def attention(q, k, v, first, scale):
    """``q [n, H, D]`` at positions first .. over ``k, v [L, G, D]``, in 64 bits: outputs, and what an error of the weights and of the scores is multiplied
    by: sum w |v| and, per head, the largest sum of |q| |k| over a query's keys."""
    n, H, D = q.shape
    L, G = k.shape[:2]
    q, k, v = q.double(), k.double().repeat_interleave(H // G, 1), v.double().repeat_interleave(H // G, 1)
    s = torch.einsum("nhd,lhd->hnl", q, k) * scale
    mag = torch.einsum("nhd,lhd->hnl", q.abs(), k.abs()) * abs(scale)
    seen = torch.arange(L)[None] <= first + torch.arange(n)[:, None]
    w = s.masked_fill(~seen, -math.inf).softmax(-1)
    y = torch.einsum("hnl,lhd->nhd", w, v)
    size = torch.einsum("hnl,lhd->nhd", w, v.abs())
    return y, size, mag.masked_fill(~seen, 0).amax(-1).T[..., None]
