"""Scores of tokens in rows of nearly equal logits, whose terms are all of one size and whose batches may have a new largest one each."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def _bound(x, dtype, want):
    """Half a step of the result.  Of the sum of exponentials, in its own size: a term's arguments on its way from its batch's largest logit to the row's are d together, each in three
    roundings; it is an exponential of its own (2^-22) and takes a warp's and a block's factor (2^-22 each); and 5 additions (vectors of four numbers, four to a batch) or 10 (of eight,
    eight).  Where sums are of 64 bits (32-bit numbers in a block or more a row) its warp's largest logits bring it 2^-22 for each factor of 2, or half of one and more.  Else each of its thread's batches may bring a
    factor (2^-22) and three roundings, and so many additions and products follow: 5 over a warp, 7 for a block's warps, 7 for a row's blocks."""
    V = x.shape[-1]
    d = x.double().amax(-1, keepdim=True) - x.double()
    mean = ((-d).softmax(-1) * d).sum(-1)
    roundings = 5 if dtype is FP else 10
    if dtype is not FP or V <= 32 * 20 * 4:
        a_warp, a_block = (32 * 16, 256 * 16) if dtype is FP else (32 * 64, 256 * 64)      # numbers of a batch
        batches = max(-(-(V + 7) // a_warp) if V <= 32 * 20 * 8 else 0, -(-(V + 7) // a_block))
        roundings += batches * (4 + 3) + 19
    return want.abs() * 2.0**-24 + mean * 3 * 2.0**-24 + (3 + mean / math.log(2.0)) * 2.0**-22 + roundings * 2.0**-24


def _alike(kind, V, dtype):
    """24 rows: rising, falling, of one number but one, of any."""
    gen = torch.Generator().manual_seed(6)
    up = torch.logspace(-6, 1.5, 24, dtype=torch.float64)[:, None]
    if kind == "rising":
        return (torch.arange(V)[None] / V * up).to(dtype)
    if kind == "falling":
        return _alike("rising", V, dtype).flip(1)
    if kind == "but one":
        x = -torch.rand(24, 1, generator=gen).expand(24, V).clone()
        x[:, V // 3] = 0.0
        return x.to(dtype)
    return (torch.rand(24, V, generator=gen) * up).to(dtype)


@pytest.mark.parametrize("dtype", [FP, BF, HF], ids=str)
@pytest.mark.parametrize("V", [600, 5003, 32000, 100003, 1 << 18])
@pytest.mark.parametrize("kind", ["rising", "falling", "but one", "any"])
def test_rows_of_one_size(kind, V, dtype):
    """A row by itself, whose sums several blocks share, and many times, a block or a warp each."""
    from lit_llama.sampling import token_logprobs

    x = _alike(kind, V, dtype).to(DEV)
    tokens = torch.tensor([0, V - 1, V // 3, V // 2, 1, 5] * 4, device=DEV)
    want = torch.cat([torch.log_softmax(r.double(), -1)[t][None] for r, t in zip(x, tokens)])
    bound = torch.cat([_bound(r[None], dtype, w[None]) for r, w in zip(x, want)])
    off = [float(((token_logprobs(x, tokens).double() - want).abs() / bound).max())]
    for r in range(24):
        for n in (500, 3000):
            got = token_logprobs(x[r:r + 1].expand(n, V), tokens[r:r + 1].expand(n)).double()
            off.append(float(((got - want[r]).abs() / bound[r]).max()))
    assert max(off) <= 1, max(off)
