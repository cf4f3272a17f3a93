"""The paged 4-bit cache: pages and slots against lists on the host, rounding and attention against 64 bits."""
import math
import random

import pytest
import torch

from tests.util_paged import PAGE, Pool, attention, held_as, turned

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16


def _cache(*a, **k):
    from lit_llama.paged_cache import PagedCache4

    return PagedCache4(*a, **k)


def _rope(n, D):
    theta = 1.0 / 10000 ** (torch.arange(0, D, 2, dtype=torch.float64) / D)
    angle = torch.arange(n, dtype=torch.float64)[:, None] * theta
    return torch.stack((angle.cos(), angle.sin()), -1).float()


# ---------------------------------------------------------------------------------------------------------------- pages and slots
def _same_plan(plan, want):
    for name, w in want.items():
        assert getattr(plan, name).tolist() == w, name


@pytest.mark.parametrize("requests, pages, max_length, seed", [(1, 1, 64, 0), (3, 7, 100, 1), (40, 90, 400, 2), (40, 30, 400, 5), (1500, 2500, 300, 3), (1500, 700, 300, 6), (2300, 4000, 130, 4)])
def test_steps_get_their_pages(requests, pages, max_length, seed):
    """Steps of unequal requests, some idle, some of them refused: the same pages, slots and reasons as one after the other on the host."""
    rng = random.Random(seed)
    cache, pool = _cache(1, 1, 32, group=32, pages=pages, requests=requests, max_length=max_length), Pool(requests, pages, max_length)
    seen = set()
    for step in range(12):
        B = rng.randrange(1, requests + 1) if step % 3 else requests
        rows = rng.sample(range(requests), B)
        counts = [rng.choice([0, 1, 1, 1, rng.randrange(1, 80), rng.randrange(1, max_length + 1)]) for _ in rows]
        if step % 4 == 3:                                    # mistakes among them
            for _ in range(1 + B // 5):
                i = rng.randrange(B)
                kind = rng.randrange(4)
                if kind == 0:
                    rows[i] = rng.choice([-1, requests, 1 << 30, -(1 << 31)])
                elif kind == 1:
                    rows[i] = rows[rng.randrange(B)]
                elif kind == 2:
                    counts[i] = -rng.randrange(1, 5)
                else:
                    counts[i] = max_length + 1
        total = sum(max(c, 0) for c in counts)
        T = total if step % 5 else max(0, total - rng.randrange(0, 9)) + (step % 2) * 7
        most = max_length if step % 2 else 70
        plan = cache.plan(rows, counts, T, max_count=most)
        _same_plan(plan, pool.plan(rows, counts, T, min(most, T)))
        seen |= set(plan.status.tolist())
        pool.agrees(cache)
        ended = [rng.randrange(-1, requests + 1) for _ in range(rng.randrange(1, requests + 1))]
        keep = [rng.choice([0, 0, 1, PAGE, rng.randrange(max_length), -1]) for _ in ended]
        cache.truncate(ended, keep)
        pool.truncate(ended, keep)
        pool.agrees(cache)
    assert 0 in seen and (requests < 40 or {2, 3, 4} <= seen) and (pages >= requests or 1 in seen)


def test_reasons():
    cache = _cache(1, 1, 32, group=32, pages=3, requests=4, max_length=150)
    cache.plan([0, 1], [64, 65], 129).check()
    for rows, counts, T, word in (([2], [1], 1, "pages"), ([0], [100], 100, "longer"), ([4], [1], 1, "no such"), ([1, 1], [1, 1], 2, "no such"),
                                  ([0], [-1], 1, "negative"), ([1], [2], 1, "behind")):
        with pytest.raises(RuntimeError, match=word):
            cache.plan(rows, counts, T).check()
    cache.truncate([1], [64])
    cache.plan([2], [1], 1).check()
    cache.reset()
    assert cache.lengths.tolist() == [0] * 4 and int(cache.n_free) == 3
    cache.plan([3], [150], 150).check()


def test_a_step_of_nothing():
    cache = _cache(1, 2, 64, pages=3, requests=4, max_length=150)
    plan = cache.plan([0, 1], [0, 0], 0)
    q = torch.empty((0, 2, 64), dtype=BF, device=DEV)
    assert cache.append(0, plan, q, q, q).shape == (0, 2, 64) and cache.attend(0, plan, q).shape == (0, 2, 64)
    assert plan.starts.tolist() == [0, 0, 0] and int(cache.n_free) == 3


# ---------------------------------------------------------------------------------------------------------------- rounding
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D, group", [(32, 32), (64, 32), (64, 64), (128, 32), (128, 64), (128, 128)])
@pytest.mark.parametrize("turn", [False, True])
def test_append_rounds_as_defined(D, group, dtype, turn):
    """Every value that the cache stands for, bit by bit; odd counts, so that pairs of slots and pages end inside requests; rows of a wider matrix."""
    torch.manual_seed(D + group)
    H, G, counts = 6, 3, [1, 70, 0, 33, 129]
    T = sum(counts)
    cache = _cache(2, H, D, n_kv_head=G, group=group, dtype=dtype, pages=9, requests=5, max_length=200)
    cache.free.copy_(torch.randperm(9))
    cache.blocks.fill_(255)
    start = [3, 0, 5, 64, 60]
    cache.plan(range(5), start, sum(start)).check()
    plan = cache.plan(range(5), counts, T)
    plan.check()
    rows = torch.randn(T, (H + 2 * G) * D + 8)
    rows[:, D:2 * D] *= 30.0
    rows[1, H * D:] = 2.5                                # groups of one value
    rows[2, H * D:] = 0.0
    rows[3, H * D:] *= 1e-6
    rows[4, H * D:] *= 2000.0
    rows = rows.to(dtype).to(DEV)
    q, k, v = (rows[:, a * D:b * D].unflatten(1, (-1, D)) for a, b in ((0, H), (H, H + G), (H + G, H + 2 * G)))
    rope = _rope(200, D).to(DEV) if turn else None
    out = cache.append(1, plan, q, k, v, rope=rope)
    pos = plan.positions.cpu()
    want_q, want_k = (turned(x.cpu(), pos, rope.cpu()) if turn else x.cpu() for x in (q, k))
    assert torch.equal(out.cpu(), want_q)
    got_k, got_v = cache.read(1, plan.slots)
    # a value is one product, exact in 32 bits (4 by at most 11), one sum rounded to 32 bits and one rounding to the type
    for got, x in ((got_k, want_k), (got_v, v.cpu())):
        want = held_as(x, group).float().to(dtype)
        assert torch.equal(got.cpu(), want)
    assert bool((cache.blocks[0] == 255).all())


@pytest.mark.parametrize("dtype", [BF, HF])
def test_groups_that_are_no_numbers(dtype):
    D, group = 64, 32
    cache = _cache(1, 1, D, group=group, dtype=dtype, pages=1, requests=1, max_length=64)
    x = torch.randn(6, 1, D)
    x[0, 0, 3], x[1, 0, 40], x[2, 0, 0], x[3, 0, 63] = math.nan, math.inf, -math.inf, math.nan
    x[4, 0, 0], x[4, 0, 1] = torch.finfo(dtype).max, -torch.finfo(dtype).max        # fp16: a range that its scale holds; bf16: none
    x = x.to(dtype)
    plan = cache.plan([0], [6], 6)
    cache.append(0, plan, None, x.to(DEV), x.to(DEV))
    for got in cache.read(0, plan.slots):
        want = held_as(x, group).float().to(dtype)
        assert torch.equal(got.cpu().isnan(), want.isnan())
        assert torch.equal(got.cpu().nan_to_num(7.0), want.nan_to_num(7.0))
    assert cache.read(0, torch.tensor([-1, 64, 1 << 30], dtype=torch.int32, device=DEV))[0].isnan().all()


# ---------------------------------------------------------------------------------------------------------------- attention
def _filled(held, counts, H, G, D, group, dtype, *, seed=0, spare=3, loud=True):
    """A cache (page tails and free pages hold bytes that are no numbers) whose requests have brought held + counts tokens, the plan of the last
    counts, and the values it stands for."""
    torch.manual_seed(seed)
    n = len(held)
    total = [a + b for a, b in zip(held, counts)]
    pages = sum(-(-t // PAGE) for t in total) + spare
    cache = _cache(1, H, D, n_kv_head=G, group=group, dtype=dtype, pages=pages, requests=n + 2, max_length=max(total) + 5)
    cache.free.copy_(torch.randperm(pages))
    cache.blocks.fill_(255)
    rows = torch.randperm(n + 2)[:n].tolist()
    k, v = torch.randn(sum(total), G, D), torch.randn(sum(total), G, D)
    if loud:
        k[..., torch.randperm(D)[:3]] *= 6
        v += torch.randn(G, D)
    k, v = cache.brought = k.to(dtype), v.to(dtype)
    plan = cache.plan(rows, total, sum(total))
    plan.check()
    cache.append(0, plan, None, k.to(DEV), v.to(DEV))
    cache.truncate(rows, held)
    plan = cache.plan(rows, counts, sum(counts), max_count=max(counts))
    plan.check()
    q = torch.randn(sum(counts), H, D).to(dtype)
    return cache, plan, q, held_as(k, group), held_as(v, group)


def _near(got, q, k, v, held, counts, dtype, scale):
    """Against 64 bits.  The weights are rounded to fp16 (half a place, 2^-11) or for whole prompts to 16 bits, their sum is of the unrounded ones or of the rounded ones: twice that.
    Prompts' kernels see keys and values rounded to the cache's type, the others exactly: a score is off by the sum of |q| |k| times half a place (and 2^-18 of that sum for
    fp32 sums and the exponential), a weight by twice that; the result is rounded once."""
    half = torch.finfo(dtype).eps / 2
    at = first = 0
    for h, c in zip(held, counts):
        if c == 0:
            at += h
            continue
        y, size, mag = attention(q[first:first + c], k[at:at + h + c], v[at:at + h + c], h, scale)
        tol = y.abs() * half + size * (2 * 2.0 ** -11 + half + 2 * mag * (half + 2.0 ** -18)) + 1e-7
        g = got[first:first + c].double().cpu()
        assert bool(((g - y).abs() <= tol).all()), (h, c, float(((g - y).abs() / tol).max()))
        # and on the whole: roundings of unequal sign leave far less than their bounds
        assert float((g - y).norm() / y.norm()) <= 2 * half + 2.0 ** -10
        at, first = at + h + c, first + c


SHAPES = [
    # held, counts, heads, key heads
    ([0], [1], 1, 1),
    ([63], [1], 3, 3),
    ([64], [1], 4, 1),
    ([0, 5, 700, 64, 127], [1, 1, 1, 1, 1], 8, 2),
    ([0, 10, 700, 0], [1, 0, 1, 0], 4, 4),
    ([3000], [1], 2, 2),
    ([2500, 3], [1, 1], 12, 1),
    ([0, 63, 64, 200], [4, 3, 5, 1], 4, 4),
    ([100, 0], [17, 2], 8, 1),
    ([0], [64], 2, 2),
    ([0], [65], 4, 2),
    ([1], [300], 3, 3),
    ([500, 0, 3, 900], [130, 257, 1, 1], 4, 1),
    ([129, 64], [1, 383], 2, 2),
]


@pytest.mark.parametrize("held, counts, H, G", SHAPES)
@pytest.mark.parametrize("D, group, dtype", [(128, 64, BF), (128, 32, HF), (64, 64, BF), (32, 32, BF)])
@torch.no_grad()
def test_attention(held, counts, H, G, D, group, dtype):
    cache, plan, q, k, v = _filled(held, counts, H, G, D, group, dtype)
    got = cache.attend(0, plan, q.to(DEV))
    _near(got, q, k, v, held, counts, dtype, D ** -0.5)


@pytest.mark.parametrize("D, group, dtype", [(128, 128, BF), (128, 128, HF), (128, 32, BF), (64, 32, BF), (64, 32, HF), (64, 64, HF), (32, 32, HF)])
@pytest.mark.parametrize("held, counts", [([300, 20], [1, 1]), ([77, 0], [3, 9]), ([0, 33], [200, 70])])
@torch.no_grad()
def test_attention_of_every_form(held, counts, D, group, dtype):
    cache, plan, q, k, v = _filled(held, counts, 4, 2, D, group, dtype, seed=1)
    _near(cache.attend(0, plan, q.to(DEV), scale=0.3), q, k, v, held, counts, dtype, 0.3)


@pytest.mark.parametrize("counts", [[1, 1, 1, 1], [3, 2, 9, 1], [90, 70, 128, 66]])
@torch.no_grad()
def test_refused_sequences_and_rows_behind_the_last(counts):
    """Tokens of refused sequences are no numbers and leave the others alone; rows behind the last token stay as they are."""
    held, H, G, D, dtype = [100, 60, 0, 30], 4, 2, 64, BF
    cache, plan, q, k, v = _filled(held, counts, H, G, D, 32, dtype, spare=0)
    rows = plan.request.tolist()
    cache.truncate(rows, held)
    T = sum(counts) + 37
    q = torch.cat([q, torch.randn(37, H, D).to(dtype)])
    wrong = list(rows)
    wrong[1] = wrong[0]                                       # the second names the first's request
    plan = cache.plan(wrong, counts, T)
    assert plan.status.tolist() == [0, 3, 0, 0]
    out = torch.full((T, H, D), 7.0, dtype=dtype, device=DEV)
    at = [sum(held[:i]) + sum(counts[:i]) for i in range(5)]
    step = [torch.cat([x[at[i] + held[i]:at[i + 1]] for i in range(4)] + [torch.full((37, G, D), math.nan, dtype=dtype)]).to(DEV) for x in cache.brought]
    held_before = cache.read(0, torch.arange(cache.pages * PAGE, dtype=torch.int32, device=DEV))
    assert cache.append(0, plan, None, *step) is None
    s = plan.starts.tolist()
    mine = torch.zeros(cache.pages * PAGE, dtype=torch.bool)
    mine[plan.slots[plan.slots >= 0].long().cpu()] = True
    assert int(mine.sum()) == sum(counts) - counts[1] and bool((plan.slots[s[1]:s[2]] == -1).all()) and bool((plan.slots[s[4]:] == -1).all())
    for x, y in zip(held_before, cache.read(0, torch.arange(cache.pages * PAGE, dtype=torch.int32, device=DEV))):
        assert torch.equal(x[~mine].nan_to_num(9.0), y[~mine].nan_to_num(9.0))              # every other slot is as it was
    y = cache.attend(0, plan, q.to(DEV), out=out)
    assert y is out
    assert y[s[1]:s[2]].isnan().all() and bool((y[s[4]:] == 7.0).all())
    for i in (0, 2, 3):
        _near(y[s[i]:s[i + 1]], q[s[i]:s[i + 1]], k[at[i]:at[i + 1]], v[at[i]:at[i + 1]], [held[i]], [counts[i]], dtype, D ** -0.5)


@torch.no_grad()
def test_values_and_keys_of_very_unequal_size():
    """Groups of one head's values 2^20 apart, queries and keys with large numbers in a few dimensions, scores far apart."""
    D, group, dtype = 128, 32, BF
    torch.manual_seed(3)
    cache = _cache(1, 2, D, group=group, dtype=dtype, pages=20, requests=1, max_length=1000)
    k, v, q = torch.randn(900, 2, D), torch.randn(900, 2, D), torch.randn(1, 2, D)
    v[..., :32] *= 2.0 ** 20
    v[..., 32:64] *= 2.0 ** -20
    k[..., 5] *= 100
    q[..., 7] *= 2.0 ** 12
    k[..., 7] *= 2.0 ** -12
    k, v, q = k.to(dtype), v.to(dtype), q.to(dtype)
    cache.plan([0], [899], 899)
    for n in (899, 1):
        if n == 1:
            plan = cache.plan([0], [1], 1)
        else:
            cache.truncate([0], [0])
            plan = cache.plan([0], [899], 899)
        part = slice(0, 899) if n > 1 else slice(899, 900)
        cache.append(0, plan, None, k[part].to(DEV), v[part].to(DEV))
    got = cache.attend(0, plan, q.to(DEV))
    K, V = held_as(k, group), held_as(v, group)
    y, size, mag = attention(q, K, V, 899, D ** -0.5)
    half = torch.finfo(dtype).eps / 2
    tol = y.abs() * half + size * (2 * 2.0 ** -11 + 2 * mag * 2.0 ** -18)
    assert bool(((got.double().cpu() - y).abs() <= tol).all())


@torch.no_grad()
def test_keys_that_are_no_numbers():
    """A key that is none in sight: its queries' outputs are none.  Behind a query, or in another request: no trace of it."""
    D, dtype = 64, BF
    for counts in ([1], [3], [100]):
        held = [40]
        cache, plan, q, k, v = _filled(held, counts, 2, 2, D, 32, dtype)
        n = counts[0]
        bad = torch.randn(n, 2, D).to(dtype)
        bad[n - 1, 1, 2] = math.nan                              # the last token's second head
        cache.append(0, plan, None, bad.to(DEV), bad.to(DEV))
        y = cache.attend(0, plan, q.to(DEV)).cpu()
        assert y[n - 1, 1].isnan().all() and not y[:n - 1].isnan().any() and not y[:, 0].isnan().any()


@torch.no_grad()
def test_a_cache_of_more_than_four_gigabytes():
    """Pages whose bytes lie past 2^32."""
    H, D = 32, 128
    cache = _cache(1, H, D, pages=16000, requests=2, max_length=400)
    assert cache.blocks.numel() > 2 ** 32
    q, k, v = (torch.randn(301, H, D).to(BF) for _ in range(3))
    plan = cache.plan([1], [301], 301)
    # the stack gives page 0 first; the last pages are what this is about
    cache.reset()
    cache.free.copy_(torch.arange(16000))
    plan = cache.plan([1], [301], 301)
    assert int(plan.slots.max()) > 15990 * PAGE
    cache.append(0, plan, None, k.to(DEV), v.to(DEV))
    y = cache.attend(0, plan, q.to(DEV))
    _near(y, q, held_as(k, 64), held_as(v, 64), [0], [301], BF, D ** -0.5)
    cache.truncate([1], [300])
    plan = cache.plan([1], [1], 1)
    one = cache.attend(0, plan, q[300:].to(DEV))
    _near(one, q[300:], held_as(k, 64), held_as(v, 64), [300], [1], BF, D ** -0.5)


@torch.no_grad()
def test_refusals():
    cache = _cache(2, 4, 64, n_kv_head=2, pages=4, requests=2, max_length=100)
    other = _cache(2, 4, 64, n_kv_head=2, pages=4, requests=2, max_length=100)
    old = cache.plan([0], [3], 3)
    cache.truncate([0], [0])
    plan = cache.plan([0], [3], 3)
    q, k = torch.zeros((3, 4, 64), dtype=BF, device=DEV), torch.zeros((3, 2, 64), dtype=BF, device=DEV)
    for call in (lambda: cache.attend(0, old, q), lambda: other.attend(0, plan, q), lambda: cache.attend(2, plan, q), lambda: cache.attend(-1, plan, q),
                 lambda: cache.attend(0, plan, q.half()), lambda: cache.attend(0, plan, q[:2]), lambda: cache.attend(0, plan, q.cpu()),
                 lambda: cache.attend(0, plan, q[:, :2]), lambda: cache.attend(0, plan, q, scale=0.0), lambda: cache.attend(0, plan, q, scale=math.nan),
                 lambda: cache.attend(0, plan, q, scale=-1.0), lambda: cache.attend(0, plan, q, out=q[:2]), lambda: cache.append(0, plan, q, q, k),
                 lambda: cache.append(0, plan, q, k, k.float()), lambda: cache.append(0, plan, None, k, k, rope=torch.zeros((100, 32, 2), device=DEV)),
                 lambda: cache.append(0, plan, q, k, k, rope=torch.zeros((99, 32, 2), device=DEV)),
                 lambda: cache.append(0, plan, q, k, k, rope=torch.zeros((100, 64, 2), device=DEV)),
                 lambda: cache.append(0, plan, q, k, k, rope=torch.zeros((100, 32, 2), dtype=HF, device=DEV)),
                 lambda: cache.plan([0], [1, 2], 3), lambda: cache.plan([], [], 0), lambda: cache.plan([0], [1], -1), lambda: cache.plan([0], [1], 1, max_count=-1),
                 lambda: cache.plan(torch.zeros(1, dtype=torch.int64, device=DEV), [1], 1), lambda: cache.truncate(torch.zeros(1, dtype=torch.int32), [1]),
                 lambda: cache.read(0, torch.zeros(1, device=DEV)), lambda: cache.read(5, plan.slots)):
        with pytest.raises(RuntimeError):
            call()
    with torch.enable_grad():
        with pytest.raises(RuntimeError, match="gradient"):
            cache.attend(0, plan, q.float().requires_grad_().to(BF))


@torch.no_grad()
def test_rows_of_any_stride():
    """Rows at odd distances, heads apart, off 16-byte boundaries: the same result as dense ones."""
    cache, plan, q, k, v = _filled([70, 3], [2, 5], 4, 2, 64, 64, BF)
    want = cache.attend(0, plan, q.to(DEV))
    for make in (lambda x: x.transpose(0, 1).contiguous().transpose(0, 1), lambda x: torch.cat([x, x], -1)[..., :64],
                 lambda x: torch.cat([x.flatten(1), x.flatten(1)[:, :3]], 1)[:, :256].unflatten(1, (4, 64)),
                 lambda x: torch.cat([x.flatten()[:1], x.flatten()])[1:].view(x.shape), lambda x: torch.cat([x.flatten(1)] * 3, 1)[:, :256].unflatten(1, (4, 64))):
        assert torch.equal(cache.attend(0, plan, make(q.to(DEV))), want)


@pytest.mark.parametrize("new", [1, 3, 80])
@torch.no_grad()
def test_a_captured_step_serves_other_lengths(new):
    """Plan, append and attention as one graph, replayed while requests grow and one of them pauses, on another stream than it was captured on."""
    H, G, D, B = 4, 2, 64, 3
    cache = _cache(1, H, D, n_kv_head=G, group=32, pages=60, requests=B, max_length=900)
    rope = _rope(900, D).to(DEV)
    rows, counts = torch.arange(B, dtype=torch.int32, device=DEV), torch.full((B,), new, dtype=torch.int32, device=DEV)
    T = B * new
    q, k, v = torch.zeros((T, H, D), dtype=BF, device=DEV), torch.zeros((T, G, D), dtype=BF, device=DEV), torch.zeros((T, G, D), dtype=BF, device=DEV)

    def step():
        plan = cache.plan(rows, counts, T, max_count=new)
        return plan, cache.attend(0, plan, cache.append(0, plan, q, k, v, rope=rope))

    step()
    cache.truncate([0, 1, 2], [0, 0, 0])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        plan, y = step()
    keys, values, held = [torch.zeros(0, G, D)] * B, [torch.zeros(0, G, D)] * B, [0] * B
    side = torch.cuda.Stream()
    for i in range(7):
        c = [new, new, 0 if i % 3 == 1 else new]
        total = sum(c)
        new_q, new_k, new_v = torch.randn(T, H, D).to(BF), torch.randn(T, G, D).to(BF), torch.randn(T, G, D).to(BF)
        for to, what in ((q, new_q), (k, new_k), (v, new_v), (counts, torch.tensor(c, dtype=torch.int32))):
            to.copy_(what)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            g.replay()
        torch.cuda.current_stream().wait_stream(side)
        assert plan.status.tolist() == [0, 0, 0]
        pos = plan.positions.cpu()[:total]
        tq, tk = turned(new_q[:total], pos, rope.cpu()), turned(new_k[:total], pos, rope.cpu())
        s = plan.starts.tolist()
        for b in range(B):
            keys[b] = torch.cat([keys[b].to(BF), tk[s[b]:s[b + 1]]])
            values[b] = torch.cat([values[b].to(BF), new_v[s[b]:s[b + 1]]])
            _near(y[s[b]:s[b + 1]], tq[s[b]:s[b + 1]], held_as(keys[b], 32), held_as(values[b], 32), [held[b]], [c[b]], BF, D ** -0.5)
            held[b] += c[b]
    assert cache.lengths.tolist() == held


@torch.no_grad()
def test_two_caches_at_once():
    """Steps of two caches on two streams, and two graphs replayed side by side: what each gives alone."""
    held, counts = [900, 2, 300], [1, 1, 1]
    sets = [_filled(held, counts, 4, 2, 128, 64, BF, seed=s) for s in (1, 2)]
    qs = [q.to(DEV) for _, _, q, _, _ in sets]
    want = [c.attend(0, p, q) for (c, p, *_), q in zip(sets, qs)]
    streams, graphs, outs = [torch.cuda.Stream() for _ in sets], [], []
    for (c, p, *_), q in zip(sets, qs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append([c.attend(0, p, q) for _ in range(4)])
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(20):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for got, w in zip(outs, want):
        assert all(torch.equal(x, w) for x in got)
    for _ in range(10):
        eager = []
        for s, (c, p, *_), q in zip(streams, sets, qs):
            with torch.cuda.stream(s):
                eager.append([c.attend(0, p, q) for _ in range(3)])
    torch.cuda.synchronize()
    for got, w in zip(eager, want):
        assert all(torch.equal(x, w) for x in got)


@torch.no_grad()
def test_the_same_bits_every_time():
    for held, counts in (([3000, 5, 900], [1, 1, 1]), ([300, 5], [9, 3]), ([300, 0], [130, 200])):
        cache, plan, q, _, _ = _filled(held, counts, 8, 2, 128, 64, BF)
        first = cache.attend(0, plan, q.to(DEV))
        assert all(torch.equal(cache.attend(0, plan, q.to(DEV)), first) for _ in range(20))


@pytest.mark.parametrize("counts", [[1], [8], [150]])
@torch.no_grad()
def test_slices_of_unequal_size(counts):
    """Values that are zeros for the keys of some slices and pages, 2^40 apart for others; keys 2^30 apart, under scores that stay small."""
    held, H, D, dtype = [330], 2, 64, BF
    torch.manual_seed(4)
    L = held[0] + counts[0]
    k, v = torch.randn(L, H, D), torch.randn(L, H, D) + 1.0
    v[:, 0, :] *= torch.tensor([0.0, 1.0, 2.0 ** 20, 2.0 ** -20])[(torch.arange(L) // 16) % 4][:, None]
    v[64:128] = 0.0
    v[128:200] *= 2.0 ** 25
    k[:, 1, :] *= torch.tensor([1.0, 2.0 ** -30, 0.0, 0.25])[(torch.arange(L) // 16) % 4][:, None]
    k, v, q = k.to(dtype), v.to(dtype), torch.randn(counts[0], H, D).to(dtype)
    cache = _cache(1, H, D, group=32, dtype=dtype, pages=9, requests=1, max_length=600)
    plan = cache.plan([0], [L], L)
    cache.append(0, plan, None, k.to(DEV), v.to(DEV))
    cache.truncate([0], held)
    plan = cache.plan([0], counts, counts[0], max_count=counts[0])
    _near(cache.attend(0, plan, q.to(DEV)), q, held_as(k, 32), held_as(v, 32), held, counts, dtype, D ** -0.5)


@pytest.mark.parametrize("held, counts, H, G", [
    ([1500], [1], 32, 1),                       # one token of as many columns as the few may have
    ([700, 5], [1, 1], 40, 1),                  # more of them: tcgen05 for single tokens
    ([200, 0, 64], [1, 7, 100], 9, 3),          # heads of a key head that are no power of two
    ([30, 600], [11, 1], 9, 3),
    ([4000], [40], 4, 4),                       # few queries over a long past: walks in many parts
    ([2000, 1], [300, 1], 8, 8),
])
@torch.no_grad()
def test_columns_of_any_number(held, counts, H, G):
    cache, plan, q, k, v = _filled(held, counts, H, G, 64, 32, BF, seed=6)
    _near(cache.attend(0, plan, q.to(DEV)), q, k, v, held, counts, BF, 0.125)


@pytest.mark.parametrize("n, new", [(1500, 1), (300, 2), (300, 40)])
@torch.no_grad()
def test_many_sequences(n, new):
    """More sequences than the planning block holds, or than look through the names before theirs."""
    rng = random.Random(n)
    held, counts = [rng.randrange(0, 90) for _ in range(n)], [rng.choice([0, 1, new]) for _ in range(n)]
    cache, plan, q, k, v = _filled(held, counts, 2, 1, 32, 32, BF, seed=7)
    _near(cache.attend(0, plan, q.to(DEV)), q, k, v, held, counts, BF, 32 ** -0.5)


@torch.no_grad()
def test_sequences_that_bring_more_than_was_said():
    """Tokens of a sequence that is refused for its count come out as no numbers, however many they are."""
    cache, plan, q, k, v = _filled([10, 20, 400], [1, 90, 1], 32, 1, 64, 32, BF)
    rows = plan.request.tolist()
    for most in (1, 2):
        cache.truncate(rows, [10, 20, 400])
        plan = cache.plan(rows, [1, 90, 1], 92, max_count=most)
        assert plan.status.tolist() == [0, 2, 0]
        y = cache.attend(0, plan, q.to(DEV))
        assert y[1:91].isnan().all()
        _near(y[:1], q[:1], k[:11], v[:11], [10], [1], BF, 0.125)


@pytest.mark.parametrize("count", [1, 6, 90])
@torch.no_grad()
def test_queries_that_are_no_numbers(count):
    """Such a query's output is none, the others' are as ever; large and small queries keep their 8 bits."""
    cache, plan, q, k, v = _filled([150], [count], 4, 2, 64, 32, BF, loud=False)
    q[count - 1, 3, 5] = math.inf
    q[0, 1] *= 2.0 ** 40
    q[0, 2] *= 2.0 ** -40
    q[0, 0, 7] = math.nan
    y = cache.attend(0, plan, q.to(DEV)).cpu()
    assert y[count - 1, 3].isnan().all() and y[0, 0].isnan().all()
    want = attention(q[:1, 2:3], k[:151, 1:], v[:151, 1:], 150, 0.125)[0]
    assert float((y[0, 2].double() - want[0, 0]).abs().max()) <= 2.0 ** -6
    # scores 2^40 apart: the largest key's value alone
    s = (q[0, 1].double() * k[:151, 0]).sum(-1)
    assert float((y[0, 1].double() - v[int(s.argmax()), 0]).abs().max()) <= 2.0 ** -7 * float(v.abs().max())
    if count > 1:
        rest = y.clone()
        rest[count - 1, 3] = 0
        rest[0, 0] = 0
        assert not rest.isnan().any()


@pytest.mark.parametrize("scale", [0.125, 1e-30])
@pytest.mark.parametrize("count", [1, 5, 100])
@torch.no_grad()
def test_queries_of_zeros_and_scales_of_nearly_nothing(count, scale):
    """All keys in sight weigh the same: the mean of their values."""
    cache, plan, q, k, v = _filled([70], [count], 2, 2, 64, 64, BF, loud=False)
    q[0] = 0
    y = cache.attend(0, plan, q.to(DEV), scale=scale).double().cpu()
    rows = range(1) if scale > 1e-20 else range(count)
    for r in rows:
        want = v[:71 + r].mean(0)
        assert float((y[r] - want).abs().max()) <= 2.0 ** -8 * float(want.abs().max()) + 2.0 ** -11 * float(v.abs().max())
