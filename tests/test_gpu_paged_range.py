"""Attention over the paged 4-bit cache where numbers are of very unequal size: keys and values behind a query, or in sight and without weight, leave no
trace in what the other keys give."""
import math

import pytest
import torch

from tests.test_gpu_paged_cache import BF, DEV, HF, PAGE, _cache
from tests.util_paged import attention, held_as

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


def _check(got, q, K, V, held, group, dtype, scale):
    """A weight and its sum are off by half a place of fp16 each (2^-11), a value too (2^-11, and up to twice that of its group's largest where it is a subnormal
    number), a score by 2^-11 of sum |q| |k| (keys in 11 bits) and 2^-18 for sums in fp32 and the exponential, which moves a weight by twice that; a weight may come to
    nothing below 2^-23 of the largest product of a weight and a group's range, once a key.  Errors of a weight meet codes, so that a group's largest value
    counts for all of its dimensions.  The result is rounded once."""
    top = V.abs().unflatten(-1, (-1, group)).amax(-1, keepdim=True).expand(*V.shape[:2], -1, group).flatten(-2)
    y, _, mag = attention(q, K, V, held, scale)
    size = attention(q, K, top, held, scale)[0]
    half = torch.finfo(dtype).eps / 2
    tol = y.abs() * half + size * (4 * 2.0 ** -11 + 2 * mag * (2.0 ** -11 + 2.0 ** -18) + K.shape[0] * 2.0 ** -22) + 1e-30
    off = (got - y).abs()
    assert bool((off <= tol).all()), float((off / tol).nan_to_num(math.inf).max())


def _columns(count, D=128, G=2, R=1, L=300, dtype=BF, spread=0.1):
    """Keys, values and queries of a request of ``L`` tokens, the last ``count`` of them the step's."""
    k, v, q = torch.randn(L, G, D), torch.randn(L, G, D) + 0.5, torch.randn(count, G * R, D) * spread
    return k.to(dtype), v.to(dtype), q.to(dtype)


FORMS = [(2, 1, BF, 64), (2, 1, HF, 64), (7, 1, BF, 32), (7, 1, HF, 128), (15, 2, BF, 64), (64, 1, BF, 64), (130, 2, HF, 32), (250, 1, BF, 128), (290, 2, BF, 64)]


@pytest.mark.parametrize("count, R, dtype, group", FORMS)
@pytest.mark.parametrize("size", [1500.0, 30000.0, 1e9, 1e30])
@torch.no_grad()
def test_a_later_value_leaves_earlier_rows_alone(count, R, dtype, group, size):
    """One number of the last token's value is large: the rows before it do not see it."""
    if size > torch.finfo(dtype).max:
        return
    torch.manual_seed(11)
    k, v, q = _columns(count, R=R, dtype=dtype)
    held = k.shape[0] - count
    v[-1, :, 3] = size
    got, K, V = _attended(q, k, v, held, group)
    _check(got[:-1], q[:-1], K[:-1], V[:-1], held, group, dtype, 128 ** -0.5)


@pytest.mark.parametrize("count, R, dtype, group", FORMS)
@pytest.mark.parametrize("size", [30000.0, 1e9, 1e30])
@torch.no_grad()
def test_a_later_key_leaves_earlier_rows_alone(count, R, dtype, group, size):
    if size > torch.finfo(dtype).max:
        return
    torch.manual_seed(12)
    k, v, q = _columns(count, R=R, dtype=dtype)
    held = k.shape[0] - count
    k[-1, :, 3] = -size
    got, K, V = _attended(q, k, v, held, group)
    _check(got[:-1], q[:-1], K[:-1], V[:-1], held, group, dtype, 128 ** -0.5)


@pytest.mark.parametrize("count, R, dtype, group", [(1, 1, BF, 64), (1, 1, HF, 32)] + FORMS)
@pytest.mark.parametrize("size", [1500.0, 30000.0, 1e9])
@pytest.mark.parametrize("at", [0, 40, 200])
@torch.no_grad()
def test_a_value_in_sight_without_weight(count, R, dtype, group, size, at):
    """A key that no query weighs (2^-80 and less) has a large value; the others share the weight."""
    if size > torch.finfo(dtype).max:
        return
    torch.manual_seed(13)
    k, v, q = _columns(count, R=R, dtype=dtype)
    held = k.shape[0] - count
    q[..., 0], k[..., 0] = 8.0, 0.0
    k[at, :, 0] = -80.0                                       # scores of -640 / sqrt(128)
    v[at, :, 3] = size
    got, K, V = _attended(q, k, v, held, group)
    first = max(0, at - held)
    _check(got, q, K, V, held, group, dtype, 128 ** -0.5)
    assert first == 0 or torch.isfinite(got).all()


@pytest.mark.parametrize("count, R, group", [(2, 1, 64), (3, 1, 32), (9, 1, 64), (15, 2, 64), (40, 1, 64), (150, 1, 32), (180, 2, 64)])
@pytest.mark.parametrize("large", [1100.0, 1e9])
@pytest.mark.parametrize("hidden", [False, True])
@torch.no_grad()
def test_many_small_weights_beside_a_first_token(count, R, group, large, hidden):
    """The first token has nearly all of the weight and a small value, so that the result is that of the others, at 2^-11 each; one value, in sight without
    weight or behind the query, is large."""
    torch.manual_seed(14)
    L = 190
    k, v, q = _columns(count, R=R, L=L)
    held = L - count
    q[..., 0], k[..., 0] = 8.0, 0.0
    k[0, :, 0] = 11 * math.log(2.0) * math.sqrt(128) / 8.0
    v[0] *= 2.0 ** -10
    v[-1 if hidden else 5, :, 5] = large
    if not hidden:
        k[5, :, 0] = -80.0
    got, K, V = _attended(q, k, v, held, group)
    n = count - 1 if hidden else count
    _check(got[:n], q[:n], K[:held + n], V[:held + n], held, group, BF, 128 ** -0.5)


@pytest.mark.parametrize("count, R, group", [(1, 1, 32), (4, 1, 32), (9, 1, 64), (16, 2, 32), (70, 1, 32), (300, 2, 64)])
@torch.no_grad()
def test_groups_of_very_unequal_size(count, R, group):
    """Groups of one token's values 2^40 apart, keys' alike: each group's result to its own size."""
    torch.manual_seed(15)
    k, v, q = _columns(count, R=R, L=330)
    v[..., :group] *= 2.0 ** 20
    v[..., group:] *= 2.0 ** -20
    k[..., :group] *= 2.0 ** -20
    got, K, V = _attended(q, k, v, 330 - count, group)
    _check(got, q, K, V, 330 - count, group, BF, 128 ** -0.5)


@pytest.mark.parametrize("count, R, group", [(1, 1, 64), (6, 1, 32), (16, 2, 64), (90, 1, 32), (300, 2, 64)])
@pytest.mark.parametrize("power", [-60, -20, -9, 0, 9, 20, 60])
@torch.no_grad()
def test_values_of_any_size(count, R, group, power):
    """All values under a power of two, and the queries' scores with them where the keys are: the same result under it."""
    torch.manual_seed(16)
    k, v, q = _columns(count, R=R, L=330)
    v, k, q = v * 2.0 ** power, k * 2.0 ** -(power // 3), q * 2.0 ** (power // 3)
    got, K, V = _attended(q, k, v, 330 - count, group)
    _check(got, q, K, V, 330 - count, group, BF, 128 ** -0.5)


@pytest.mark.parametrize("grow", [1, 40])
@pytest.mark.parametrize("count, R, dtype", [(1, 1, BF), (1, 1, HF), (6, 1, BF), (16, 2, HF), (80, 1, BF)])
@torch.no_grad()
def test_scores_that_rise_over_values_that_fall(count, R, dtype, grow):
    """Scores that rise along the keys, so that references move again and again, over values that get smaller (grow 1: larger): what counts is the
    product of weight and value."""
    torch.manual_seed(17)
    L = 700
    k, v, q = _columns(count, R=R, L=L, dtype=dtype)
    ramp = torch.arange(L) / L
    q[..., 0] = 8.0
    k[..., 0] = (30.0 * ramp)[:, None]
    v = (v.float() * 2.0 ** ((10 if grow == 1 else -10) * ramp)[:, None, None]).to(dtype)
    got, K, V = _attended(q, k, v, L - count, 64)
    _check(got, q, K, V, L - count, 64, dtype, 128 ** -0.5)


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


@pytest.mark.parametrize("D, group", [(32, 32), (64, 32), (64, 64), (128, 32), (128, 64), (128, 128)])
@pytest.mark.parametrize("held, count, R", [(0, 300, 1), (500, 140, 2), (40, 30, 3)])
@torch.no_grad()
def test_fp16_prompts_are_as_exact_as_their_values(D, group, held, count, R):
    """Scores that some large dimensions of the keys make: only a value's rounding to 11 bits and the result's are left to see.  Each is off by up to half a place,
    2^-11, evenly spread: 2^-11 / sqrt(3) of it in the mean square at most; values of both signs add up as their errors do, so that the norm of both together
    is sqrt(2 / 3) 2^-11 of the result's.  Weights and keys have 20 bits and more, sums in fp32 lose 2^-15 at most."""
    torch.manual_seed(20)
    G, L = 2, held + count
    loud = torch.where(torch.arange(D) % 20 == 3, 6.0, 1.0)
    k, v, q = (torch.randn(L, G, D) * loud).to(HF), torch.randn(L, G, D).to(HF), torch.randn(count, G * R, D).to(HF)
    got, K, V = _attended(q, k, v, held, group)
    want = attention(q, K, V, held, D ** -0.5)[0]
    assert float((got - want).norm() / want.norm()) <= math.sqrt(2 / 3) * 2.0 ** -11 + 2.0 ** -15


@pytest.mark.parametrize("D, group", [(32, 32), (64, 64), (128, 32), (128, 128)])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("held, count, R", [(700, 1, 1), (300, 4, 1), (90, 1, 8), (200, 9, 1), (100, 16, 2)])
@torch.no_grad()
def test_few_columns_take_keys_as_they_are(D, group, dtype, held, count, R):
    """Scores that large dimensions make, with nothing lost of keys and scales: 2^-18 of sum |q| |k| for sums in fp32 and the exponential, which moves a weight by
    twice that; half a place of fp16 for a weight, which meets codes (its group's largest), and 2^-22 of that once a key; the result is rounded once."""
    torch.manual_seed(21)
    G, L = 2, held + count
    loud = torch.where(torch.arange(D) % 20 == 3, 6.0, 1.0)
    k, v, q = (torch.randn(L, G, D) * loud).to(dtype), torch.randn(L, G, D).to(dtype), torch.randn(count, G * R, D).to(dtype)
    got, K, V = _attended(q, k, v, held, group)
    top = V.abs().unflatten(-1, (-1, group)).amax(-1, keepdim=True).expand(L, G, -1, group).flatten(-2)
    y, _, mag = attention(q, K, V, held, D ** -0.5)
    size = attention(q, K, top, held, D ** -0.5)[0]
    tol = y.abs() * torch.finfo(dtype).eps / 2 + size * (2 * 2.0 ** -11 + 2 * mag * 2.0 ** -18 + L * 2.0 ** -22)
    assert bool(((got - y).abs() <= tol).all()), float(((got - y).abs() / tol).max())


@pytest.mark.parametrize("R, D, group", [(1, 128, 32), (4, 64, 32), (8, 128, 128), (8, 64, 32), (16, 64, 64)])
@torch.no_grad()
def test_fp16_results_over_many_keys(R, D, group):
    """120 000 keys of weights some 2^9 apart, whose values leave little of one another: nothing is left to see but the result's rounding, half a place, 2^-11, at most and
    2^-11 / sqrt(3) of it in the mean square at most.  Sums in fp32 of parts that are added up in a tree lose 2^-24 of some 60 codes' worth of a value a part."""
    torch.manual_seed(22)
    L = 120000
    k, v, q = torch.randn(L, 1, D).to(HF), torch.randn(L, 1, D).to(HF), (torch.randn(1, R, D) * 1.5).to(HF)
    got, K, V = _attended(q, k, v, L - 1, group)
    want = attention(q, K, V, L - 1, D ** -0.5)[0]
    assert float((got - want).norm() / want.norm()) <= math.sqrt(1 / 3) * 2.0 ** -11 + 2.0 ** -15
