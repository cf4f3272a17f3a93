"""What draws, scores and forks refuse before anything reaches a GPU, and the host's restatements that the GPU tests compare with."""
import math

import numpy as np
import pytest
import torch

from lit_llama import _native as N
from lit_llama.sampling import sample, token_logprobs
from tests.util_share import ONE, SharedPool, drawn

A = 1 << 12      # an address that no launch reads
SAMPLE = (A, 1, 1, 100, 100, A, 0, 1.0, 0, 0, 0, 1.0, 0, 0.0, A, 0)
SCORE = (A, 1, 1, 100, 100, A, 0, 1.0, A, 0)
FORK = (A, A, 1, A, A, A, 1, A, A, 0)


def _struct(**other):
    kind = dict(table=A, lengths=A, free_pages=A, n_free=A, stamp=A, requests=1, width=1, pages=1, max_length=64, heads=2, kv_heads=2, head_size=64, group=64, dtype=1)
    kind.update(other)
    return N.Kv4Cache(*(kind[n] for n, _ in N.Kv4Cache._fields_))


@pytest.mark.parametrize("name, args, at, value", [
    ("ll_sample_rows", SAMPLE, 0, 0), ("ll_sample_rows", SAMPLE, 1, 3), ("ll_sample_rows", SAMPLE, 1, -1), ("ll_sample_rows", SAMPLE, 2, 0), ("ll_sample_rows", SAMPLE, 3, 0),
    ("ll_sample_rows", SAMPLE, 3, (1 << 18) + 1), ("ll_sample_rows", SAMPLE, 5, 0), ("ll_sample_rows", SAMPLE, 14, 0),
    ("ll_token_logprobs", SCORE, 0, 0), ("ll_token_logprobs", SCORE, 1, 7), ("ll_token_logprobs", SCORE, 2, -1), ("ll_token_logprobs", SCORE, 3, (1 << 18) + 1),
    ("ll_token_logprobs", SCORE, 5, 0), ("ll_token_logprobs", SCORE, 8, 0),
])
def test_refused_calls(name, args, at, value):
    with pytest.raises(RuntimeError):
        N.call(name, *args[:at], value, *args[at + 1:])


@pytest.mark.parametrize("name", ["ll_kv4_fork", "ll_kv4_release"])
@pytest.mark.parametrize("at, value, cache", [(1, 0, {}), (1, A + 4, {}), (2, 0, {}), (2, 65536, {}), (3, 0, {}), (4, 0, {}), (5, 0, {}), (6, 0, {}), (7, 0, {}), (8, 0, {}),
                                              (6, 1, dict(max_length=65)), (6, 1, dict(table=0)), (6, 1, dict(head_size=48)), (6, 1, dict(dtype=0))])
def test_refused_forks(name, at, value, cache):
    import ctypes

    s = _struct(**cache)
    args = [ctypes.addressof(s), *FORK[1:]]
    args[at] = value
    with pytest.raises(RuntimeError):
        N.call(name, *args)


X, U = torch.zeros(2, 5), torch.zeros(2)


@pytest.mark.parametrize("call", [
    lambda: sample(X, U),                                                        # on the host
    lambda: sample(X[0], U),
    lambda: sample(X.long(), U),
    lambda: sample(X.double(), U),
    lambda: token_logprobs(X, U.long()),
    lambda: token_logprobs(X[None], U.long()),
])
def test_refused_arguments(call):
    with pytest.raises(RuntimeError):
        call()


def test_draws_of_a_few_tokens():
    x = [0.0, math.log(2.0), -math.inf, math.log(5.0)]                            # 1, 2, 0 and 5 eighths
    assert [drawn(x, u) for u in (0.0, 0.124, 0.126, 0.374, 0.376, 0.999, 1.0)] == [0, 0, 1, 1, 3, 3, 3]
    assert {drawn(x, u, top_k=1) for u in (0.0, 0.5, 1.0)} == {3}
    assert [drawn(x, u, top_k=2) for u in (0.0, 0.28, 0.29)] == [1, 1, 3]
    assert {drawn(x, u, top_p=0.6) for u in (0.0, 1.0)} == {3} and drawn(x, 0.0, top_p=0.63) == 1 and drawn(x, 0.0, top_p=0.88) == 0
    assert drawn(x, 0.0, min_p=0.3) == 1 and drawn(x, 0.0, min_p=0.41) == 3 and drawn(x, 0.0, min_p=7.0) == 3
    assert drawn(x, 0.0, top_k=2, top_p=0.72) == 1 and drawn(x, 0.0, top_k=2, top_p=0.7) == 3
    assert drawn([2.0, 1.0, 2.0, 2.0], 0.5, top_k=1) == 2 and drawn([2.0, 1.0, 2.0], 0.9, temperature=0.0) == 0
    assert drawn([-math.inf] * 3, 0.5) == -1 and drawn([0.0, math.nan], 0.5) == -1 and drawn([0.0], 1.5) == -1 and drawn([0.0], 0.5, temperature=-1.0) == -1
    assert drawn([math.inf, 0.0, math.inf], 0.7) == 2
    assert drawn(np.zeros(7), 0.5) == 3 and ONE == 2**44


def test_pools_that_share():
    pool = SharedPool(5, 6, 400)
    pool.plan([0], [150], 150, 150)                                              # pages 0, 1 and 22 tokens in 2
    assert pool.fork([0, 0, 0, 3], [1, 2, 1, 4]) == [0, 0, 3, 0]
    assert pool.table[1] == [0, 1, 3] and pool.table[2] == [0, 1, 4] and pool.holders[:5] == [3, 3, 1, 1, 1] and pool.bytes[3] == 2 and pool.lengths[4] == 0
    assert pool.truncate([2], [70]) == [0]                                       # into page 1, which others hold: a copy in 5, and 4 is free
    assert pool.table[2] == [0, 5] and pool.free == [4] and pool.bytes[5] == 1 and pool.holders == [3, 2, 1, 1, 0, 1]
    assert pool.truncate([0, 1], [100, 100]) == [0, 1] and pool.table[0] == [0, 4] and pool.lengths[1] == 150 and pool.free == [2]
    assert pool.truncate([0, 1, 2], [0, 0, 0]) == [0, 0, 0] and sorted(pool.free) == list(range(6)) and pool.holders == [0] * 6
