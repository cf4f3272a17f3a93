"""Scores of tokens whose logits lie further apart than a number of 32 bits, under temperatures of their size."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, FP = torch.bfloat16, torch.float32


def _bound(x, want):
    """Half a step of the result (its first part, (l - m) / T, is of 64 bits).  Of the sum of exponentials: arguments in three roundings, once more where a warp's or a block's sums are brought to
    the row's largest logit; and in these sizes no more than ten batches a thread, which bring 16 roundings and a factor each (2^-22 and 2^-23): less than 2^-17 together, and 2^-18 for
    warps and blocks."""
    d = x.amax(-1, keepdim=True) - x
    p = (-d).softmax(-1)
    mean = torch.where(p > 0, p * d.clamp(max=1e30), 0.0).sum(-1)
    return want.abs() * 2.0**-24 + mean * 6 * 2.0**-24 + 2.0**-16


@pytest.mark.parametrize("dtype", [FP, BF], ids=str)
@pytest.mark.parametrize("V", [2, 700, 40000])
def test_logits_far_apart(V, dtype):
    """Differences that no number of 32 bits holds, under temperatures of their size; and at the other end, where they are all steps of the smallest numbers."""
    from lit_llama.sampling import token_logprobs

    gen = torch.Generator().manual_seed(2)
    rows, temperatures = [], []
    for size, t in ((3e38, 3e38), (3.3e38, 1e38), (3e38, 2e37), (1e37, 3e36), (3e38, 5e35), (1e36, 1.1e36), (1e36, 0.9e36), (1.6e38, 1.0), (1e-30, 1e-30)):
        x = (torch.rand(V, generator=gen, dtype=torch.float64) * 2 - 1) * size
        x[0], x[-1] = size, -size
        rows.append(x.to(dtype))
        temperatures.append(t)
    x = torch.stack(rows)
    t = torch.tensor(temperatures)
    for token in (0, V - 1, V // 2):
        tokens = torch.full((len(rows),), token)
        scaled = x.double() / t.double()[:, None]
        want = torch.log_softmax(scaled, -1)[:, token]
        bound = _bound(scaled, want)
        got = token_logprobs(x.to(DEV), tokens.to(DEV), temperature=t.to(DEV)).cpu().double()
        assert bool(((got - want).abs() <= bound).all()), ((got - want).abs() / bound).tolist()
        for r in range(len(rows)):
            one = token_logprobs(x[r:r + 1].to(DEV), tokens[r:r + 1].to(DEV), temperature=temperatures[r]).cpu().double()
            assert float((one - want[r]).abs()) <= float(bound[r])
    x = torch.tensor([[3e38, -3e38]], device=DEV, dtype=dtype)
    score = float(token_logprobs(x, torch.tensor([0], device=DEV), temperature=3e38))
    assert abs(score + math.log1p(math.exp(-2 * float(x[0, 0]) / float(torch.tensor(3e38))))) <= 2.0**-20
