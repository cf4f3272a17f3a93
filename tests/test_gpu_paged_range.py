"""Attention over the paged 4-bit cache where numbers are of very unequal size: keys and values behind a query, or in sight and without weight, leave no
trace in what the other keys give."""
import pytest
import torch

from tests.test_gpu_paged_cache import BF, DEV, HF, PAGE, _cache
from tests.util_paged import held_as

pytestmark = pytest.mark.gpu


def _attended(q, k, v, held, group, scale=None, n_kv_head=None, **plan):
    """One request's last tokens over all of its keys: what the kernels give, and what the cache holds."""
    L, G, D = k.shape
    cache = _cache(1, q.shape[1], D, n_kv_head=G, group=group, dtype=k.dtype, pages=-(-L // PAGE) + 2, requests=1, max_length=max(L, 1000))
    cache.free.copy_(torch.randperm(cache.pages))
    cache.blocks.fill_(255)
    whole = cache.plan([0], [L], L)
    whole.check()
    cache.append(0, whole, None, k.to(DEV), v.to(DEV))
    cache.truncate([0], [held])
    step = cache.plan([0], [L - held], L - held, max_count=L - held)
    step.check()
    return cache.attend(0, step, q.to(DEV), scale=scale).double().cpu(), held_as(k, group), held_as(v, group)


@pytest.mark.parametrize("counts, R", [([1], 1), ([4], 1), ([1], 8), ([5], 1), ([8], 1), ([16], 1), ([16], 2), ([1, 60], 1), ([1, 60], 6)])
@pytest.mark.parametrize("D, group", [(32, 32), (64, 64), (128, 128), (128, 32)])
@torch.no_grad()
def test_fp16_results_keep_their_bits(counts, R, D, group):
    """All keys of a request have the same value: whatever the weights, the result is that value, rounded once.  Before that, of the group's range: weights in
    two terms of 11 bits and their sum 2^-21; sums in fp32 8 * 2^-24; the products' sums, by far the most of it, as the tensor pipe adds 16 products to a sum C
    with each cut off two bits below the last one of C's fp32, and the sum at that: (17 / 4 + 1) 2^-23 C a product, of which a warp's 32 keys take four.
    Sums of codes c + 16 c' (255 of c' = 15, from which those of c are taken) give 5.25 * 2^-23 * 4 * (255 + 15) / (16 * 15) = 2^-18.4.  All of them: 2^-17.9."""
    torch.manual_seed(18)
    held, G = 37, 2
    L = [held + c for c in counts]
    k, q = torch.randn(sum(L), G, D).to(HF), torch.randn(sum(counts), G * R, D).to(HF)
    one = torch.randn(len(counts), G, D).to(HF)
    v = one.repeat_interleave(torch.tensor(L), 0)
    n = len(counts)
    cache = _cache(1, G * R, D, n_kv_head=G, group=group, dtype=HF, pages=8, requests=n, max_length=1000)
    plan = cache.plan(range(n), L, sum(L))
    cache.append(0, plan, None, k.to(DEV), v.to(DEV))
    cache.truncate(range(n), [held] * n)
    plan = cache.plan(range(n), counts, sum(counts), max_count=max(counts))
    plan.check()
    got = cache.attend(0, plan, q.to(DEV)).double().cpu()[:counts[0]]
    want = held_as(one, group)[0].repeat_interleave(R, 0)
    span = want.unflatten(-1, (-1, group)).amax(-1) - want.unflatten(-1, (-1, group)).amin(-1)
    tol = want.abs() * 2.0 ** -11 + span.repeat_interleave(group, -1) * 2.0 ** -17 + 2.0 ** -25
    assert bool(((got - want).abs() <= tol).all()), float(((got - want).abs() / tol).max())


@pytest.mark.parametrize("dtype", [BF, HF])
@torch.no_grad()
def test_a_query_of_zeros_beside_others_under_a_tiny_scale(dtype):
    """Its keys weigh the same, also those that a warp walks for it alone: the 65th, on a page that the other token does not see."""
    torch.manual_seed(19)
    D = 64
    k, v, q = torch.randn(65, 1, D), torch.zeros(65, 1, D), torch.randn(2, 1, D)
    v[64] = 65.0
    q[1] = 0
    got, K, V = _attended(q.to(dtype), k.to(dtype), v.to(dtype), 63, 64, scale=1e-7)
    assert float(got[0].abs().max()) <= 0.0 and float((got[1] - 1.0).abs().max()) <= 2.0 ** -8
