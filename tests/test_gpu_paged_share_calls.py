"""Calls of a cache whose requests share pages: results in the place of the queries, queries of a wider matrix, another stream, forks and cuts in a captured step."""
import pytest
import torch

from tests.test_gpu_paged_share import _cache, _filled, _near

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("H, G, D, dtype", [(4, 4, 64, BF), (8, 2, 128, HF)], ids=str)
def test_results_in_the_place_of_queries(H, G, D, dtype):
    """Groups large and small, sequences of no group with one part of a walk and with several, drafts."""
    held, copies = [700, 1, 300, 900], [20, 3, 2, 1]
    more = [(3 + i % 5, 1 + i % 3) for i in range(26)]
    cache, rows, counts, q, keys = _filled(H, G, D, 32, dtype, held, copies, more, seed=11)
    plan = cache.plan(rows, counts, sum(counts), max_count=3)
    y = cache.attend(1, plan, q.to(DEV))
    _near(y, q, keys, counts, dtype, D ** -0.5)
    place = q.to(DEV).clone()
    assert cache.attend(1, plan, place, out=place) is place and torch.equal(place, y)
    wide = torch.full((q.shape[0], 3, H, D), 5.0, dtype=dtype, device=DEV)
    wide[:, 1] = q.to(DEV)
    assert torch.equal(cache.attend(1, plan, wide[:, 1]), y) and bool((wide[:, ::2] == 5).all())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = cache.attend(1, plan, q.to(DEV))
    torch.cuda.synchronize()
    assert torch.equal(other, y)


def test_captured_forks():
    """A captured search step, which ends the copies of the step before, forks, cuts and goes on, next to the same calls one by one; its lists change between the replays."""
    H, D, n, c = 4, 64, 3, 5
    graphed, eager = (_cache(2, H, D, pages=90, requests=n + n * c, max_length=700) for _ in range(2))
    into = torch.arange(n, n + n * c, dtype=torch.int32, device=DEV)
    rows, cut, none, one = torch.zeros_like(into), torch.zeros_like(into), torch.zeros_like(into), torch.ones_like(into)
    gen = torch.Generator().manual_seed(2)
    new = lambda k: (torch.randn(k, H, D, generator=gen) * 2).to(BF).to(DEV)  # noqa: E731
    q, k, v = (new(n * c) for _ in range(3))
    pk, pv = new(1030), new(1030)
    for cache in (graphed, eager):
        plan = cache.plan([0, 1, 2], [600, 130, 300], 1030)
        for layer in range(2):
            cache.append(layer, plan, None, pk, pv)

    def step(cache):
        cache.truncate(into, none)
        status = cache.fork(rows, into)
        cuts = cache.truncate(into, cut)
        plan = cache.plan(into, one, n * c, max_count=1)
        for layer in range(2):
            cache.append(layer, plan, None, k, v)
        return status, cuts, plan.status, cache.attend(0, plan, q), cache.attend(1, plan, q)

    step(graphed)
    step(eager)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(graphed)
    for i in range(6):
        rows.copy_(torch.randint(0, n, (n * c,), generator=gen))
        if i % 2:
            rows.copy_(rows.sort().values)
        cut.copy_(torch.randint(1, 650, (n * c,), generator=gen))
        for t in (q, k, v):
            t.copy_(new(n * c))
        g.replay()
        want = step(eager)
        for a, b in zip(out, want):
            assert torch.equal(a, b)
        assert int(want[0].sum()) == 0 and not bool(want[3].isnan().any())
        assert torch.equal(graphed.table, eager.table) and torch.equal(graphed.lengths, eager.lengths) and torch.equal(graphed.n_free, eager.n_free)
        assert torch.equal(graphed.blocks[:, graphed.table[into[0], 0]], eager.blocks[:, eager.table[into[0], 0]])


@torch.no_grad()
def test_scores_of_plain_draws():
    """generate_batch with scores where tokens are drawn by torch, one answer and several: each new token's log-probability, under the model's own step."""
    import sys
    from pathlib import Path

    sys.path.insert(0, str(Path(__file__).parent.parent / "lit-llama-ja_b200"))
    import generate
    from lit_llama import LLaMA, LLaMAConfig

    torch.manual_seed(5)
    m = LLaMA(LLaMAConfig(block_size=320, vocab_size=100, n_layer=2, n_head=4, n_embd=256)).to(DEV, BF)
    m.apply(m._init_weights)
    m.eval()
    prompts = [torch.randint(0, 100, (size,), device=DEV) for size in (20, 64)]
    real, seen = generate.token_logprobs, []

    def noted(logits, tokens):
        seen.append(torch.log_softmax(logits.double(), -1).gather(1, tokens[:, None])[:, 0].cpu())
        return real(logits, tokens)

    generate.token_logprobs = noted
    try:
        for samples in (1, 3):
            seen.clear()
            out, scores = generate.generate_batch(m, prompts, 6, top_k=10, samples=samples, logprobs=True)
            assert len(out) == len(scores) == 2 * samples and all(len(s) == 6 for s in scores)
            # (fp32 sums over 100 tokens: half a step of a score of up to 16, and 2^-20 for the sum)
            assert all(abs(float(scores[b][i]) - float(seen[i][b])) <= 2.0**-19 for b in range(2 * samples) for i in range(6))
    finally:
        generate.token_logprobs = real
