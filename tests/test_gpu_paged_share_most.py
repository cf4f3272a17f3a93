"""Steps of as many sequences as are divided by groups that share pages, and of more: the lists of groups and walks full, and steps that are divided without them."""
import pytest
import torch

from tests.test_gpu_paged_share import _filled, _near

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16


def _divided(cache, B, T, max_count):
    """Whether a step of that size is divided by groups: its sizes are others then."""
    from lit_llama import _native as N

    return cache._sizes(B, T, max_count)[0] != N.call_ret("ll_kv4_work_ints", cache._c, B, T, max_count)


MOST = [
    ([200] * 256, [2] * 256, 1),                       # 256 pairs: every place of the groups' lists
    ([130] * 171, [3] * 170 + [2], 1),                 # 512 in threes
    ([700], [512], 1),                                 # one group of all
    ([200] * 256, [2] * 255 + [3], 1),                 # 513: divided without groups
    ([700], [600], 1),
    ([300] * 128, [4] * 128, 2),                       # drafts
]


@pytest.mark.parametrize("H, G, D, group, dtype", [(2, 1, 64, 64, BF), (8, 1, 32, 32, HF)], ids=str)
@pytest.mark.parametrize("held, copies, new", MOST, ids=range(len(MOST)))
def test_as_many_sequences_as_there_may_be(held, copies, new, H, G, D, group, dtype):
    more = [(new + i % 5, new) for i in range(sum(copies))]
    held = held[:-1] + [max(held[-1], 600)]            # (caches of more than 512 tokens are divided)
    cache, rows, counts, q, keys = _filled(H, G, D, group, dtype, held, copies, more, seed=len(more))
    assert _divided(cache, len(rows), sum(counts), new) == (len(rows) <= 512)
    plan = cache.plan(rows, counts, sum(counts), max_count=new)
    y = cache.attend(1, plan, q.to(DEV))
    _near(y, q, keys, counts, dtype, D ** -0.5)
    again = cache.attend(1, plan, q.to(DEV))
    assert torch.equal(y, again)                       # the same bits


@pytest.mark.parametrize("T, divided", [(2390, True), (2400, False)])
def test_as_much_scratch_as_there_may_be(T, divided):
    """Rows behind the last token count for what a step's parts may need: the same sequences on both sides of the limit."""
    H, D, copies, new = 32, 128, 12, 8
    more = [(new + i % 3, new) for i in range(copies)]
    cache, rows, counts, q, keys = _filled(H, H, D, 128, BF, [600, 130], [10, 2], more, seed=4)
    B = 512
    rows, counts = rows + [0] * (B - copies), counts + [0] * (B - copies)
    assert _divided(cache, B, T, new) == divided
    work, scratch = cache._sizes(B, T, new)
    assert 0.98 * (512 << 20) < scratch <= 512 << 20 if divided else scratch < 512 << 20
    plan = cache.plan(rows, counts, T, max_count=new)
    wide = torch.zeros(T, H, D, dtype=BF)
    wide[:copies * new] = q
    out = torch.full((T, H, D), 7.0, dtype=BF, device=DEV)
    cache.attend(1, plan, wide.to(DEV), out=out)
    assert bool((out[copies * new:] == 7).all())
    _near(out[:copies * new], q, keys, counts[:copies], BF, D ** -0.5)
