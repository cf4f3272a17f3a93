"""What the paged 4-bit cache refuses before anything reaches a GPU, and the host's restatement that the GPU tests compare with."""
import ctypes
import random

import pytest
import torch

from lit_llama import _native as N
from lit_llama.paged_cache import PagedCache4
from tests.util_paged import PAGE, Pool, held_as

ONE = dict(pages=4, requests=2, max_length=100)


@pytest.mark.parametrize("args, kind, error", [
    ((1, 4, 64), dict(ONE, device="cpu"), RuntimeError),
    ((1, 4, 64), dict(ONE, dtype=torch.float32), ValueError),
    ((1, 4, 48), ONE, ValueError),
    ((1, 4, 256), ONE, ValueError),
    ((1, 4, 64), dict(ONE, group=128), ValueError),
    ((1, 4, 64), dict(ONE, group=16), ValueError),
    ((1, 4, 64), dict(ONE, n_kv_head=3), ValueError),
    ((0, 4, 64), ONE, ValueError),
    ((1, 4, 64), dict(ONE, pages=0), ValueError),
    ((1, 4, 64), dict(ONE, requests=0), ValueError),
    ((1, 4, 64), dict(ONE, max_length=0), ValueError),
    ((1, 4, 64), dict(ONE, pages=1 << 25), ValueError),
    ((1, 4, 64), dict(ONE, max_length=(1 << 30) + 1), ValueError),
])
def test_refused_shapes(args, kind, error):
    with pytest.raises(error):
        PagedCache4(*args, **kind)


A = 1 << 12      # an address that no launch reads


def _struct(**other):
    kind = dict(table=A, lengths=A, free_pages=A, n_free=A, stamp=A, requests=1, width=1, pages=1, max_length=64, heads=2, kv_heads=2, head_size=64, group=64, dtype=1)
    kind.update(other)
    return N.Kv4Cache(*(kind[n] for n, _ in N.Kv4Cache._fields_))


PLAN, APPEND, READ, ATTN = (A, A, 1, 1, 1, A, A, 0), (A, 0, 0, A, 64, A, 64, 0, A, A, 0, 1, 0), (A, A, A, A, 1, 0), (A, A, 64, A, A, 1, 1, 1, 1.0, A, 0)


def _with(args, **at):
    return tuple(at.get(f"a{i}", a) for i, a in enumerate(args))


@pytest.mark.parametrize("name, cache, args", [
    ("ll_kv4_plan", {}, _with(PLAN, a0=0)),
    ("ll_kv4_plan", {}, _with(PLAN, a2=0)),
    ("ll_kv4_plan", {}, _with(PLAN, a3=-1)),
    ("ll_kv4_plan", {}, _with(PLAN, a6=A + 4)),
    ("ll_kv4_plan", {}, _with(PLAN, a3=1 << 30)),
    ("ll_kv4_plan", dict(max_length=65), PLAN),                   # a table too narrow for the longest request
    ("ll_kv4_plan", dict(pages=1 << 25), PLAN),
    ("ll_kv4_plan", dict(max_length=(1 << 30) + 64, width=1 << 25), PLAN),
    ("ll_kv4_plan", dict(table=0), PLAN),
    ("ll_kv4_truncate", {}, (A, 0, 1, 0)),
    ("ll_kv4_truncate", dict(requests=0), (A, A, 1, 0)),
    ("ll_kv4_append", dict(dtype=0), APPEND),
    ("ll_kv4_append", dict(group=48), APPEND),
    ("ll_kv4_append", dict(group=128), APPEND),
    ("ll_kv4_append", {}, _with(APPEND, a3=A + 2)),               # keys off a 16-byte boundary
    ("ll_kv4_append", {}, _with(APPEND, a4=65)),
    ("ll_kv4_append", {}, _with(APPEND, a7=A, a10=A)),            # a table and no queries
    ("ll_kv4_append", {}, _with(APPEND, a11=0)),
    ("ll_kv4_read", {}, _with(READ, a4=0)),
    ("ll_kv4_attn", dict(heads=3), ATTN),                         # three heads over two
    ("ll_kv4_attn", dict(dtype=0), ATTN),
    ("ll_kv4_attn", dict(head_size=96), ATTN),
    ("ll_kv4_attn", {}, _with(ATTN, a2=60)),
    ("ll_kv4_attn", {}, _with(ATTN, a8=0.0)),
    ("ll_kv4_attn", {}, _with(ATTN, a8=float("nan"))),
    ("ll_kv4_attn", {}, _with(ATTN, a9=0)),
])
def test_refused_calls(name, cache, args):
    c = _struct(**cache)
    with pytest.raises(RuntimeError, match="kv4"):
        N.call(name, ctypes.addressof(c), *args)


def test_sizes_of_steps_that_are_none():
    """No division by the heads that are not there, no sizes of nothing."""
    for name in ("ll_kv4_work_ints", "ll_kv4_attn_scratch_bytes"):
        assert N.call_ret(name, ctypes.addressof(_struct()), 2, 5, 5) > 0
        assert N.call_ret(name, None, 1, 1, 1) == 0
        for other in (dict(kv_heads=0), dict(heads=0), dict(heads=3), dict(kv_heads=-1), dict(max_length=0)):
            assert N.call_ret(name, ctypes.addressof(_struct(**other)), 1, 1, 1) == 0
        for step in ((0, 1, 1), (1, -1, 1), (1, 1, -1), (1, 1 << 30, 1)):
            assert N.call_ret(name, ctypes.addressof(_struct()), *step) == 0


def test_no_cache():
    for name, args in (("ll_kv4_plan", PLAN), ("ll_kv4_truncate", (A, A, 1, 0)), ("ll_kv4_append", APPEND), ("ll_kv4_read", READ), ("ll_kv4_attn", ATTN)):
        with pytest.raises(RuntimeError, match="no cache"):
            N.call(name, None, *args)


def test_page_bytes():
    """A slot of a head: D / 2 bytes of key codes and as many of value codes, and four bytes a group of either."""
    for D in (32, 64, 128):
        for group in (32, 64, 128):
            want = PAGE * (D + 8 * (D // group)) if group <= D else 0
            assert N.call_ret("ll_kv4_page_bytes", D, group) == want
    assert N.call_ret("ll_kv4_page_bytes", 96, 32) == 0


def test_truncation_undoes_a_plan():
    rng = random.Random(1)
    pool = Pool(20, 60, 500)
    for _ in range(50):
        rows = rng.sample(range(20), 12)
        before = ([list(t) for t in pool.table], list(pool.lengths), list(pool.free))
        counts = [rng.choice([0, 1, 1, rng.randrange(200)]) for _ in rows]
        first = pool.plan(rows, counts, sum(counts), 500)
        pool.truncate(rows, [before[1][r] for r in rows])
        assert before == (pool.table, pool.lengths, pool.free)
        assert pool.plan(rows, counts, sum(counts), 500) == first
        ended = rng.sample(range(20), 9)
        pool.truncate(ended, [0] * 9)


def test_rounding_is_half_a_step_at_most():
    """Half a step, and at the upper end what 15 steps fall short of the range by (the scale is rounded, by half a place at most)."""
    torch.manual_seed(0)
    for dtype in (torch.bfloat16, torch.float16):
        x = torch.randn(50, 3, 128).to(dtype)
        for group in (32, 64, 128):
            g = x.double().unflatten(-1, (-1, group))
            span = g.amax(-1, keepdim=True) - g.amin(-1, keepdim=True)
            off = (held_as(x, group) - x.double()).unflatten(-1, (-1, group)).abs()
            half = torch.finfo(dtype).eps / 2
            assert bool((off <= span / 15 * (1 + half) / 2 * (1 + 1e-6) + span * half).all())
            low = held_as(x, group).unflatten(-1, (-1, group)).amin(-1)
            assert torch.equal(low, g.amin(-1))


def test_generate_batch_refuses(monkeypatch):
    import sys
    from pathlib import Path
    from types import SimpleNamespace

    sys.path.insert(0, str(Path(__file__).parent.parent / "lit-llama-ja_b200"))
    import generate

    model = SimpleNamespace(config=SimpleNamespace(block_size=64))
    one = torch.zeros(5, dtype=torch.int64)
    for prompts, new in (([], 3), ([one], 0), ([one, one[:0]], 3), ([one[None]], 3), ([one], 61), ([one, torch.zeros(60, dtype=torch.int64)], 6)):
        with pytest.raises(ValueError):
            generate.generate_batch(model, prompts, new)
    with pytest.raises(ValueError, match="kv_cache"):
        generate.main(kv_cache="int8")
