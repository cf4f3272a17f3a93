"""Calls of the paged 4-bit cache at the ends of what it allows."""
import pytest
import torch

from tests.test_gpu_paged_cache import BF, DEV, _cache

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
