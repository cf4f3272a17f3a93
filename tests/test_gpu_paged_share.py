"""Requests of the paged 4-bit cache that share pages: forks and cuts against lists on the host, pages' bytes, attention over shared pages against 64 bits."""
import random

import pytest
import torch

from tests.util_paged import PAGE, attention, held_as
from tests.util_share import SharedPool

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16


def _cache(*a, **k):
    from lit_llama.paged_cache import PagedCache4

    return PagedCache4(*a, **k, share=True)


@pytest.mark.parametrize("requests, pages, max_length, seed", [(2, 3, 64, 0), (5, 12, 200, 1), (40, 90, 400, 2), (40, 30, 400, 5), (300, 900, 300, 7), (1500, 2500, 300, 3)])
def test_forks_and_cuts(requests, pages, max_length, seed):
    """Steps, forks and cuts one after the other, some refused, mistakes among them: the same pages, holders, reasons and bytes as on the host."""
    rng = random.Random(seed)
    cache, pool = _cache(3, 2, 32, group=32, pages=pages, requests=requests, max_length=max_length), SharedPool(requests, pages, max_length)
    first = torch.arange(pages, device=DEV, dtype=torch.int32)
    cache.blocks.copy_((first[None, :, None, None] * 7 + torch.arange(3, device=DEV)[:, None, None, None] * 31 + torch.arange(cache.blocks.shape[3], device=DEV)) % 251)
    start = cache.blocks.clone()
    seen = set()
    some = lambda n: rng.randrange(1, n + 1)  # noqa: E731
    for step in range(14):
        if step % 3 == 0:
            rows = rng.sample(range(requests), some(requests))
            counts = [rng.choice([0, 1, 64, some(max_length)]) for _ in rows]
            plan = cache.plan(rows, counts, sum(counts), max_count=max_length)
            assert plan.status.tolist() == pool.plan(rows, counts, sum(counts), min(max_length, sum(counts)))["status"]
        pool.agrees(cache)
        n = some(requests)
        rows, into = [rng.randrange(requests) for _ in range(n)], [rng.randrange(requests) for _ in range(n)]
        if step % 4 != 1:                                     # (else a few of them are empty)
            empty = [r for r in range(requests) if pool.lengths[r] == 0]
            into = [rng.choice(empty) if empty else r for r in into]
        if step % 4 == 3:
            rows[rng.randrange(n)] = rng.choice([-1, requests, 1 << 30])
            into[rng.randrange(n)] = rng.choice([-1, requests, -(1 << 31)])
        got, want = cache.fork(rows, into).tolist(), pool.fork(rows, into)
        assert got == want
        seen |= set(got)
        pool.agrees(cache)
        rows = [rng.randrange(-1, requests + 1) for _ in range(some(requests))]
        keep = [rng.choice([0, 0, 1, PAGE, rng.randrange(max_length), rng.randrange(max_length), -1]) for _ in rows]
        got, want = cache.truncate(rows, keep).tolist(), pool.truncate(rows, keep)
        assert got == want
        seen |= {10 + s for s in got}
        pool.agrees(cache)
        assert torch.equal(cache.blocks, start[:, torch.tensor(pool.bytes, device=DEV)])
    assert {0, 3} <= seen and (pages > 2 * requests or requests < 40 or {1, 11} <= seen)
    cache.reset()
    SharedPool(requests, pages, max_length).agrees(cache)


def test_calls_that_are_refused():
    from lit_llama.paged_cache import PagedCache4

    plain = PagedCache4(1, 2, 32, group=32, pages=4, requests=3, max_length=100)
    with pytest.raises(RuntimeError):
        plain.fork([0], [1])
    assert plain.truncate([0], [0]) is None
    cache = _cache(1, 2, 32, group=32, pages=4, requests=3, max_length=100)
    for rows, into in (([0], [1, 2]), ([], []), (torch.tensor([0], device=DEV), torch.tensor([1], device=DEV)), (torch.tensor([0], dtype=torch.int32), [1]),
                       (torch.zeros(1, 1, dtype=torch.int32, device=DEV), [1])):
        with pytest.raises(RuntimeError):
            cache.fork(rows, into)
    plan = cache.plan([0], [1], 1)
    cache.fork([0], [1])
    with pytest.raises(RuntimeError):                         # a fork ends the plans before it
        cache.attend(0, plan, torch.zeros(1, 2, 32, dtype=BF, device=DEV))


# ---------------------------------------------------------------------------------------------------------------- attention over shared pages
def _filled(H, G, D, group, dtype, held, copies, more, seed, order=None):
    """A cache of prompts and their copies with some tokens of their own, a step's last tokens planned again; queries, and every copy's keys and values.
    ``copies[i]``: how many of prompt i; ``more``: tokens of a copy's own, the last ``new`` of them the step's (pairs)."""
    gen = torch.Generator().manual_seed(seed)
    n, total = len(held), sum(copies)
    loud = torch.where(torch.rand(G, D, generator=gen) < 0.05, 6.0, 1.0)
    make = lambda rows, by: (torch.randn(rows, G, D, generator=gen) * by).to(dtype)  # noqa: E731
    prompts = [(make(h, loud), make(h, 1.0)) for h in held]
    parts = [(make(m, loud), make(m, 1.0)) for m, _ in more]
    T = sum(new for _, new in more)
    q = make_q = torch.randn(T, H, D, generator=gen).to(dtype)
    pages = sum(-(-h // PAGE) for h in held) + sum(h // PAGE * 0 + -(-(h % PAGE + m) // PAGE) for h, (m, _) in zip([h for h, c in zip(held, copies) for _ in range(c)], more)) + 2
    longest = max(h for h in held) + max(m for m, _ in more)
    cache = _cache(2, H, D, n_kv_head=G, group=group, pages=pages, requests=n + total, max_length=longest, dtype=dtype)
    source = [i for i, c in enumerate(copies) for _ in range(c)]
    into = list(range(n, n + total))
    cache.append(1, cache.plan(list(range(n)), held, sum(held)), None, torch.cat([k for k, _ in prompts]).to(DEV), torch.cat([v for _, v in prompts]).to(DEV))
    assert cache.fork(source, into).tolist() == [0] * total
    order = list(range(total)) if order is None else order
    rows = [into[i] for i in order]
    counts = [more[i][0] for i in order]
    plan = cache.plan(rows, counts, sum(counts))
    plan.check()
    cache.append(1, plan, None, torch.cat([parts[i][0] for i in order]).to(DEV), torch.cat([parts[i][1] for i in order]).to(DEV))
    ends = [held[source[i]] + more[i][0] for i in order]
    assert cache.truncate(rows, [e - more[i][1] for e, i in zip(ends, order)]).tolist() == [0] * total
    keys = [tuple(torch.cat([held_as(a, group), held_as(b, group)]) for a, b in zip(prompts[source[i]], parts[i])) for i in order]
    return cache, rows, [more[i][1] for i in order], q, keys


def _held_parts(x, group):
    """|code * scale| + |lowest value|: what a value that the cache holds is made of."""
    g = x.float().unflatten(-1, (-1, group))
    lo = g.min(-1, keepdim=True).values.double()
    return ((held_as(x, group).unflatten(-1, (-1, group)) - lo).abs() + lo.abs()).flatten(-2)


def _near(y, q, keys, counts, dtype, scale, parts=None):
    """The tolerance: half a step of the result, weights of 11 bits and values and keys of a bf16 cache's prompts rounded to 11 bits (each 2^-11 of
    sum w |v| at most, with the scores' 2^-11 of sum |q| |k| scaled), once more for sums.  ``parts``: the sums run over w s c and w lo apart, and weights
    of 11 bits meet the first alone: where a number far below its group's others makes these c s + lo of two large terms, an error of a weight is
    multiplied by |c s|, not by |v|, so that sum w (|c s| + |lo|) takes the place of sum w |v|."""
    at = 0
    for i, ((k, v), n) in enumerate(zip(keys, counts)):
        if n == 0:
            continue
        want, size, mag = attention(q[at:at + n], k, v, k.shape[0] - n, scale)
        if parts is not None:
            size = attention(q[at:at + n], k, parts[i], k.shape[0] - n, scale)[1]
        tol = want.abs() * torch.finfo(dtype).eps / 2 + size * (3 * 2.0**-11 + mag * 2.0**-11 * 2)
        got = y[at:at + n].cpu().double()
        assert bool(((got - want).abs() <= tol).all()), float(((got - want).abs() / tol).max())
        at += n


GROUPS = [
    ([200], [3], [(5, 1)] * 3),
    ([300], [4], [(40, 1), (1, 1), (64, 1), (20, 1)]),
    ([64], [2], [(1, 1)] * 2),                                       # one shared page, which is full
    ([63], [5], [(2, 1)] * 5),                                       # none
    ([1], [2], [(1, 1)] * 2),
    ([1000, 1, 130], [3, 2, 9], [(1 + i % 7, 1) for i in range(14)]),
    ([2048], [64], [(1 + 3 * i, 1) for i in range(64)]),
    ([700], [300], [(1 + i % 90, 1) for i in range(300)]),
    ([500, 640], [6, 5], [(30, 4)] * 11),                            # drafts
    ([900, 400], [3, 4], [(60, 1), (60, 50), (8, 1), (300, 300), (4, 2), (1, 1), (64, 33)]),      # prompts' parts beside them
]


@pytest.mark.parametrize("H, G, D, group, dtype", [(4, 4, 64, 64, BF), (8, 2, 128, 32, HF), (6, 2, 128, 128, BF), (8, 8, 32, 32, HF), (4, 1, 64, 32, BF), (5, 1, 128, 64, HF)], ids=str)
@pytest.mark.parametrize("held, copies, more", GROUPS, ids=range(len(GROUPS)))
def test_attention_of_copies(held, copies, more, H, G, D, group, dtype):
    cache, rows, counts, q, keys = _filled(H, G, D, group, dtype, held, copies, more, seed=len(more))
    plan = cache.plan(rows, counts, sum(counts))
    y = cache.attend(1, plan, q.to(DEV))
    _near(y, q, keys, counts, dtype, D ** -0.5)
    assert torch.equal(y, cache.attend(1, plan, q.to(DEV)))          # the same bits


@pytest.mark.parametrize("H, G, D, group, dtype, held, copies", [(2, 1, 64, 64, BF, 20000, 3), (1, 1, 64, 64, BF, 20000, 40), (4, 1, 128, 32, HF, 9000, 20), (8, 2, 128, 128, BF, 5003, 2)],
                         ids=str)
def test_long_shared_prompts(H, G, D, group, dtype, held, copies):
    """Walks of shared pages in more parts than a warp joins, of few columns and of many."""
    more = [(1 + i % 5, 1) for i in range(copies)]
    cache, rows, counts, q, keys = _filled(H, G, D, group, dtype, [held], [copies], more, seed=copies)
    plan = cache.plan(rows, counts, sum(counts), max_count=1)
    y = cache.attend(1, plan, q.to(DEV))
    _near(y, q, keys, counts, dtype, D ** -0.5)
    assert torch.equal(y, cache.attend(1, plan, q.to(DEV)))


@pytest.mark.parametrize("H, G, new, dtype", [(2, 2, 1, BF), (8, 2, 1, HF), (2, 2, 3, BF), (8, 2, 2, BF)], ids=str)
def test_shared_pages_of_large_values(H, G, new, dtype):
    """Shared pages with numbers that fp16 operands do not hold: their tiles are left to the walk of few columns.  And values that are no numbers in a copy's own
    page, which are its own."""
    D, held, copies = 64, 700, 40
    gen = torch.Generator().manual_seed(1)
    make = lambda n: torch.randn(n, G, D, generator=gen)  # noqa: E731
    k, v = make(held), make(held)
    v[::50, :, 3] = 3e4
    v[130, :, 40] = -6e4 if dtype == HF else -1e6
    k, v = k.to(dtype), v.to(dtype)
    cache = _cache(1, H, D, n_kv_head=G, group=64, pages=11 + 2 * copies, requests=1 + copies, max_length=held + 60, dtype=dtype)
    cache.append(0, cache.plan([0], [held], held), None, k.to(DEV), v.to(DEV))
    into = list(range(1, 1 + copies))
    assert cache.fork([0] * copies, into).tolist() == [0] * copies
    pk, pv = make(copies * new).to(dtype), make(copies * new).to(dtype)
    pv[5 * new] = float("nan")
    plan = cache.plan(into, [new] * copies, copies * new, max_count=new)
    cache.append(0, plan, None, pk.to(DEV), pv.to(DEV))
    q = torch.randn(copies * new, H, D, generator=gen).to(dtype)
    y = cache.attend(0, plan, q.to(DEV))
    assert bool(y[5 * new:6 * new].isnan().all()) and bool(torch.isfinite(torch.cat([y[:5 * new], y[6 * new:]])).all())
    keys = [tuple(torch.cat([held_as(a, 64), held_as(b[i * new:(i + 1) * new], 64)]) for a, b in ((k, pk), (v, pv))) for i in range(copies)]
    there = [i for i in range(copies) if i != 5]
    at = torch.cat([torch.arange(i * new, (i + 1) * new) for i in there])
    parts = [torch.cat([_held_parts(v, 64), _held_parts(pv[i * new:(i + 1) * new], 64)]) for i in there]
    _near(y.cpu()[at], q[at], [keys[i] for i in there], [new] * len(there), dtype, D ** -0.5, parts)


def test_copies_in_any_order():
    """Copies of several prompts one after the other in turn, idle and refused sequences between them, and rows behind the last token."""
    held, copies = [400, 200, 777], [5, 5, 5]
    more = [(1 + i, 1) for i in range(15)]
    order = [i // 3 + 5 * (i % 3) for i in range(15)]
    cache, rows, counts, q, keys = _filled(4, 2, 64, 64, BF, held, copies, more, 3, order)
    idle, refused = [2, 8], [5, 11]
    for i in idle:
        counts[i] = 0
    rows = [(1 << 20) if i in refused else r for i, r in enumerate(rows)]
    T = sum(counts) + 3
    q = torch.randn(T, 4, 64, generator=torch.Generator().manual_seed(5)).to(BF)
    plan = cache.plan(rows, counts, T, max_count=1)
    out = torch.full((T, 4, 64), 7.0, dtype=BF, device=DEV)
    cache.attend(1, plan, q.to(DEV), out=out)
    assert bool((out[-3:] == 7).all())
    at = 0
    for i, n in enumerate(counts):
        if n == 0:
            continue
        if i in refused:
            assert bool(out[at].isnan().all())
        else:
            _near(out[at:at + 1], q[at:at + 1], [(keys[i][0], keys[i][1])], [1], BF, 64 ** -0.5)
        at += n


def test_captured_steps_over_forks():
    """A captured step serves requests that are forked, cut and go on after the capture, next to the same steps called one by one."""
    H, D = 4, 64
    graphed, eager = (_cache(1, H, D, pages=60, requests=12, max_length=600) for _ in range(2))
    rows = torch.arange(12, dtype=torch.int32, device=DEV)
    live = torch.zeros(12, dtype=torch.int32, device=DEV)
    q, k, v = (torch.zeros(12, H, D, dtype=BF, device=DEV) for _ in range(3))

    def step(cache):
        plan = cache.plan(rows, live, 12, max_count=1)
        cache.append(0, plan, None, k, v)
        return cache.attend(0, plan, q)

    step(graphed)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(graphed)
    gen = torch.Generator().manual_seed(1)
    new = lambda n: (torch.randn(n, H, D, generator=gen) * 2).to(BF).to(DEV)  # noqa: E731
    pk, pv = new(230), new(230)
    for c in (graphed, eager):
        c.append(0, c.plan([0, 1], [200, 30], 230), None, pk, pv)
        assert c.fork([0, 0, 0, 1, 1], [2, 3, 4, 5, 6]).tolist() == [0] * 5
    live[:7] = 1
    for i in range(80):
        for t in (q, k, v):
            t.copy_(new(12))
        if i == 20:
            for c in (graphed, eager):
                c.truncate([2, 3, 5], [100, 128, 0])
                c.fork([4, 2], [5, 7])
            live[7] = 1
        if i == 50:
            live[3] = 0
        g.replay()
        want = step(eager)
        n = int(live.sum())
        assert torch.equal(out[:n], want[:n]) and not bool(want[:n].isnan().any())
    assert torch.equal(graphed.table, eager.table) and torch.equal(graphed.lengths, eager.lengths)
