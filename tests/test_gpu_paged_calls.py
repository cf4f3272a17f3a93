"""Calls of the paged 4-bit cache at the ends of what it allows: steps that are divided whole, single tokens of any stride, counts of nothing, results
in place, the wait check of a batch."""
import sys
from pathlib import Path

import pytest
import torch

from tests.test_gpu_paged_cache import BF, DEV, HF, _cache, _filled, _near

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B, new", [(1, 1), (40, 3), (300, 1), (90, 12), (1200, 1)])
@torch.no_grad()
def test_every_walk_is_in_the_division(B, new):
    """Steps whose walks are not cut (no request is longer than 512 tokens): every tile of every sequence is in the list, and every row is written, each of many times."""
    cache = _cache(1, 2, 32, n_kv_head=1, group=32, pages=8 * B, requests=B, max_length=500)
    rows = torch.arange(B, dtype=torch.int32, device=DEV)
    held = torch.randint(0, 400, (B,), dtype=torch.int32, device=DEV)
    cache.plan(rows, held, int(held.sum())).check()
    counts = torch.full((B,), new, dtype=torch.int32, device=DEV)
    q = torch.zeros((B * new, 2, 32), dtype=BF, device=DEV)
    cache.blocks.zero_()
    out = torch.empty_like(q)
    cols = 4 if 2 * new <= 4 else 8 if 2 * new <= 8 else 16
    for _ in range(150):
        plan = cache.plan(rows, counts, B * new, max_count=new)
        out.fill_(7.0)
        cache.attend(0, plan, q, out=out)
        assert int(plan._data[0]) == B * -(-2 * new // cols)
        assert bool((out == 0.0).all())
        cache.truncate(rows, held)


@pytest.mark.parametrize("held, counts, H, G", [([70, 3], [1, 1], 4, 2), ([900], [1], 8, 8), ([5], [1], 40, 1)])
@torch.no_grad()
def test_single_tokens_of_any_stride(held, counts, H, G):
    """Rows of one or two tokens at any distance: the same result as dense ones, from ``append`` and from ``attend``."""
    cache, plan, q, k, v = _filled(held, counts, H, G, 64, 64, BF)
    want = cache.attend(0, plan, q.to(DEV))
    _near(want, q, k, v, held, counts, BF, 0.125)
    rope = torch.rand(cache.max_length, 32, 2, device=DEV)
    new = [torch.randn(len(counts), g, 64, device=DEV).to(BF) for g in (H, G, G)]
    turned = cache.append(0, plan, *new, rope=rope)
    kept = cache.read(0, plan.slots)
    makes = [lambda x, pad=pad: torch.cat([x.flatten(1), x.flatten(1)[:, :pad]], 1)[:, :x.shape[1] * 64].unflatten(1, (-1, 64)) for pad in (1, 3, 8, 60)]
    makes.append(lambda x: x.as_strided(x.shape, (1, 64, 1)) if x.shape[0] == 1 else x)
    for make in makes:
        cache.append(0, plan, None, torch.zeros_like(new[1]), torch.zeros_like(new[2]))
        assert torch.equal(cache.append(0, plan, *(make(x) for x in new), rope=rope), turned)
        assert all(torch.equal(a, b) for a, b in zip(cache.read(0, plan.slots), kept))
    at = [sum(held[:i + 1]) + sum(counts[:i]) for i in range(len(held))]
    cache.append(0, plan, None, *(x[at].to(DEV) for x in cache.brought))
    for make in makes:
        assert torch.equal(cache.attend(0, plan, make(q.to(DEV))), want)


@pytest.mark.parametrize("max_length", [400, 2000])
@torch.no_grad()
def test_a_step_whose_sequences_may_bring_nothing(max_length):
    """``max_count`` 0: every sequence that brings tokens is refused, its tokens come out as no numbers, and rows behind the last one are left alone."""
    for H, G in ((2, 2), (40, 1)):
        cache = _cache(1, H, 64, n_kv_head=G, pages=12, requests=3, max_length=max_length)
        plan = cache.plan([0, 1, 2], [2, 0, 1], 5, max_count=0)
        assert plan.status.tolist() == [2, 0, 2] and cache.lengths.tolist() == [0, 0, 0]
        q, out = torch.randn(5, H, 64, device=DEV).to(BF), torch.full((5, H, 64), 7.0, dtype=BF, device=DEV)
        y = cache.attend(0, plan, q, out=out)
        assert bool(y[:3].isnan().all()) and bool((y[3:] == 7.0).all())


@pytest.mark.parametrize("held, counts, H, G", [([70, 3], [1, 1], 4, 2), ([1900], [1], 8, 8), ([300, 5], [9, 3], 8, 2), ([300, 0], [130, 200], 8, 2), ([2000, 1], [300, 1], 8, 8)])
@pytest.mark.parametrize("large", [False, True])
@torch.no_grad()
def test_results_over_their_queries(held, counts, H, G, large):
    """``out`` may be the queries themselves."""
    cache, plan, q, k, v = _filled(held, counts, H, G, 64, 32, BF)
    if large:                                                 # values that a product of fp16 operands does not hold
        k, v = (x.clone() for x in cache.brought)
        v[0, :, 3] = 1e6
        rows, total = plan.request.tolist(), [a + b for a, b in zip(held, counts)]
        cache.truncate(rows, [0] * len(rows))
        cache.append(0, cache.plan(rows, total, sum(total)), None, k.to(DEV), v.to(DEV))
        cache.truncate(rows, held)
        plan = cache.plan(rows, counts, sum(counts), max_count=max(counts))
    want = cache.attend(0, plan, q.to(DEV))
    mine = q.to(DEV)
    assert cache.attend(0, plan, mine, out=mine) is mine and torch.equal(mine, want)


@torch.no_grad()
def test_a_batch_is_checked_when_it_is_done(monkeypatch):
    """generate_batch looks whether a bounded wait ran out after the last step has come to its end, not while it is under way."""
    sys.path.insert(0, str(Path(__file__).parent.parent / "lit-llama-ja_b200"))
    import generate
    from tests.test_gpu_paged_model import _model

    m, done, draw = _model(64), [], generate._draw

    def slow(*a):
        torch.cuda._sleep(20_000_000)                          # some ten milliseconds
        return draw(*a)

    monkeypatch.setattr(generate, "_draw", slow)
    monkeypatch.setattr(generate, "check_waits", lambda: done.append(torch.cuda.current_stream().query()))
    prompts = [torch.randint(0, 100, (n,), device=DEV) for n in (12, 3)]
    generate.generate_batch(m, prompts, 6, top_k=1)
    assert done == [True]


@pytest.mark.parametrize("held, counts, H, G, dtype", [([300, 0], [130, 200], 8, 2, BF), ([2000, 1, 40], [300, 1, 0], 8, 8, HF), ([1500], [40], 16, 2, BF)])
@torch.no_grad()
def test_prompts_over_large_values_are_the_same_every_time(held, counts, H, G, dtype):
    """Tiles that are left to the walk of few columns, in a captured step and beside another one: the same bits as alone."""
    sets = []
    for seed in (0, 1):
        cache, plan, q, _, _ = _filled(held, counts, H, G, 128, 64, dtype, seed=seed)
        k, v = (x.clone() for x in cache.brought)
        v[::50, :, 3], k[7, :, 9] = 3e4, 2e4
        rows, total = range(len(held)), [a + b for a, b in zip(held, counts)]
        cache.reset()
        cache.append(0, cache.plan(rows, total, sum(total)), None, k.to(DEV), v.to(DEV))
        cache.truncate(rows, held)
        plan = cache.plan(rows, counts, sum(counts), max_count=max(counts))
        plan.check()
        q = q.to(DEV)
        want = cache.attend(0, plan, q)
        assert bool(torch.isfinite(want).all()) and all(torch.equal(cache.attend(0, plan, q), want) for _ in range(5))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = [cache.attend(0, plan, q) for _ in range(3)]
        sets.append((cache, plan, q, want, g, out, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(10):
        for _, _, _, _, g, _, s in sets:
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for *_, want, _, out, _ in sets:
        assert all(torch.equal(x, want) for x in out)


@torch.no_grad()
def test_the_command_line_serves_its_samples_as_one_batch(monkeypatch, capsys, tmp_path):
    sys.path.insert(0, str(Path(__file__).parent.parent / "lit-llama-ja_b200"))
    import generate
    from tests.test_gpu_paged_model import _model

    (tmp_path / "x.pth").write_bytes(b"")
    monkeypatch.setattr(generate, "load_model", lambda *a: _model(64))
    generate.main(checkpoint_path=tmp_path / "x.pth", prompt_ids="5,17,3", num_samples=3, max_new_tokens=7, kv_cache="int4")
    out = capsys.readouterr()
    lines = [[int(t) for t in line.split(",")] for line in out.out.split()]
    assert len(lines) == 3 and all(x[:3] == [5, 17, 3] and len(x) == 10 for x in lines) and "tokens/sec" in out.err
