"""Draws and scores of rows of logits (csrc/sample_rows.cu, csrc/token_logprobs.cu) against the definition on the host."""
import math

import numpy as np
import pytest
import torch

from tests.util_share import drawn

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def _logits(R, V, dtype, seed, spread=2.2):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(R, V, generator=gen) * spread
    x.scatter_add_(1, torch.randint(0, V, (R, 6), generator=gen), 8 * torch.rand(R, 6, generator=gen))
    return x.to(dtype)


def _same(x, u, **settings):
    """Tokens of the kernel and of the host; ``x`` a CPU tensor, settings numbers or CPU tensors."""
    from lit_llama.sampling import sample

    there = {n: s.to(DEV) if isinstance(s, torch.Tensor) else s for n, s in settings.items()}
    got = sample(x.to(DEV), u.to(DEV), **there).tolist()
    off = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
    want = []
    for r in range(x.shape[0]):
        mine = {n: (off[n] if s is None else float(s[r]) if isinstance(s, torch.Tensor) else s if n == "top_k" else float(np.float32(s))) for n, s in settings.items()}
        mine["top_k"] = int(mine.get("top_k", 0))
        want.append(drawn(x[r].float().numpy(), float(u[r]), **mine))
    assert got == want
    return got


SETTINGS = [dict(), dict(top_k=1), dict(top_k=40, temperature=0.7), dict(top_p=0.9), dict(min_p=0.05, temperature=1.5), dict(top_k=50, top_p=0.8, min_p=0.01), dict(top_p=0.0),
            dict(top_p=0.999, temperature=0.3), dict(min_p=1.0), dict(top_k=1000, top_p=0.95)]


@pytest.mark.parametrize("dtype", [BF, HF, FP], ids=str)
@pytest.mark.parametrize("R, V", [(5, 1), (7, 2), (6, 31), (3, 33), (9, 257), (4, 1000), (3, 4097), (8, 32000), (5, 35000), (3, 100003), (2, 200001), (1, 1 << 18)])
def test_rows_and_settings(R, V, dtype):
    for i, s in enumerate(SETTINGS if V < 50000 else SETTINGS[1::2]):
        x = _logits(R, V, dtype, 100 * R + i)
        u = torch.rand(R, generator=torch.Generator().manual_seed(i))
        u[0] = 0.0 if i % 2 else 1.0
        _same(x, u, **s)


@pytest.mark.parametrize("dtype", [BF, FP], ids=str)
def test_settings_of_each_row(dtype):
    """A batch whose requests differ in all of them, with values that change nothing among them, more rows than the card has SMs."""
    R, V = 333, 5003
    x = _logits(R, V, dtype, 1)
    gen = torch.Generator().manual_seed(2)
    pick = lambda *v: torch.tensor(v)[torch.randint(0, len(v), (R,), generator=gen)]  # noqa: E731
    got = _same(x, torch.rand(R, generator=gen), temperature=pick(0.0, 0.5, 1.0, 1.0, 2.0), top_k=pick(0, -3, 1, 7, 50, V, V + 1, 2**31 - 1).int(),
                top_p=pick(0.0, 0.3, 0.9, 1.0, 1.5), min_p=pick(-1.0, 0.0, 0.0, 0.02, 0.5, 2.0))
    assert min(got) >= 0


def test_rows_that_allow_no_draw():
    inf, nan = math.inf, math.nan
    x = torch.tensor([[0.0, 1.0, nan, 2.0], [-inf, -inf, -inf, -inf], [0.0, inf, 1.0, inf], [-inf, -inf, 3.0, -inf], [0.0, 1.0, 2.0, 3.0]])
    u = torch.tensor([0.5, 0.5, 0.9, 0.999, 0.2])
    for dtype in (BF, HF, FP):
        assert _same(x.to(dtype), u)[:4] == [-1, -1, 3, 2]
    one = x[4:].expand(6, 4)
    half = torch.full((6,), 0.5)
    assert _same(one, torch.tensor([-0.1, 1.1, nan, inf, -inf, -0.0]))[:5] == [-1] * 5
    assert _same(one, half, temperature=torch.tensor([-1.0, nan, inf, 0.0, 1e-30, 3e38]))[:4] == [-1, -1, -1, 3]
    assert _same(one, half, top_p=torch.tensor([nan, -1.0, 0.0, inf, 1.0, 0.5]))[0] == -1
    assert _same(one, half, min_p=torch.tensor([nan, -1.0, 0.0, inf, 1.0, -inf]))[0] == -1


@pytest.mark.parametrize("dtype", [BF, HF, FP], ids=str)
def test_masks_and_equal_logits(dtype):
    """Most of a row masked, at -inf or at the type's lowest value; rows of one value, of two, of values next to each other, of zeros of both signs."""
    V = 4099
    gen = torch.Generator().manual_seed(4)
    low = torch.finfo(dtype).min
    rows = [torch.where(torch.rand(V, generator=gen) < 0.95, -math.inf, torch.randn(V, generator=gen)),
            torch.where(torch.rand(V, generator=gen) < 0.95, low, torch.randn(V, generator=gen)),
            torch.full((V,), low), torch.full((V,), torch.finfo(dtype).max), torch.full((V,), 3.0), torch.where(torch.arange(V) % 2 == 0, 1.0, 1.5), torch.where(torch.rand(V, generator=gen) < 0.5, 0.0, -0.0),
            3.0 + torch.arange(V) % 7 * torch.finfo(dtype).eps, -1000.0 - torch.rand(V, generator=gen), torch.where(torch.arange(V) == 77, 1000.0, 0.0)]
    x = torch.stack(rows).to(dtype)
    for s in SETTINGS:
        for seed in range(2):
            _same(x, torch.rand(len(rows), generator=gen), **s)


def test_draws_go_through_all_of_a_row():
    """One row under many numbers, which come in the order of the vocabulary: every kept token as often as its probability says."""
    from lit_llama.sampling import sample

    V, n = 300, 60000
    x = _logits(1, V, FP, 7, spread=1.0).to(DEV)
    u = torch.arange(n, device=DEV, dtype=torch.float64).add(0.5).div(n).float()
    got = sample(x.expand(n, V), u, top_p=0.9)
    assert bool((got[1:] >= got[:-1]).all())
    count = torch.bincount(got, minlength=V).double()
    p = x[0].double().softmax(-1)
    order = p.argsort(descending=True)
    kept = order[: int((p[order].cumsum(0) < 0.9).sum()) + 1]
    want = torch.zeros_like(p).index_copy(0, kept, p[kept] / p[kept].sum()) * n
    assert float((count - want).abs().max()) <= 1.01                              # both ends of a token's numbers fall between two of u (and 2^-24 of n)


def test_rows_anywhere():
    """Rows of a wider matrix, at odd places, backwards in memory by columns, one row for all; settings that are views."""
    from lit_llama.sampling import sample, token_logprobs

    for dtype in (BF, FP):
        wide = _logits(6, 2100, dtype, 9).to(DEV)
        u = torch.rand(12, device=DEV)[::2]
        for view in (wide[:, 3:1500], wide[::2, 1:], wide[:, ::2], wide.T[:6, :6], wide[:1].expand(6, 2100), wide[1:].T[:6].contiguous().T[:5, :6]):
            R = view.shape[0]
            dense = view.contiguous().clone()
            k = torch.tensor([5, 0, 9, 1, 70, 3], dtype=torch.int32, device=DEV)[:R]
            assert torch.equal(sample(view, u[:R], top_k=k, top_p=0.9), sample(dense, u[:R].contiguous(), top_k=k, top_p=0.9))
            tokens = torch.randint(0, view.shape[1], (2 * R,), device=DEV)[::2]
            # sums of 32 bits are by vectors that begin at 16-byte boundaries: where a row begins otherwise, its terms meet in another order, and either
            # result is within the bound of a score's error of the exact one, so that two are within twice the bound of each other
            got, other = token_logprobs(view, tokens).double().cpu(), token_logprobs(dense, tokens.contiguous()).double().cpu()
            exact = torch.log_softmax(dense.double().cpu(), -1).gather(1, tokens.cpu()[:, None])[:, 0]
            assert bool(((got - other).abs() <= 2 * _score_bound(dense.cpu(), 1.0, exact)).all())
    empty = sample(wide[:0], u[:0])
    assert empty.shape == (0,) and empty.dtype is torch.int64 and token_logprobs(wide[:0], empty).shape == (0,)


def test_rows_past_32_bits():
    """The last rows of a matrix of more than 2^32 bytes and 2^31 numbers."""
    from lit_llama.sampling import sample, token_logprobs

    R, V = 70000, 32003
    x = torch.zeros(R, V, dtype=BF, device=DEV)
    tail = _logits(5, V, BF, 11)
    x[-5:] = tail.to(DEV)
    u = torch.full((R,), 0.3, device=DEV)
    got = sample(x, u, top_p=0.9)
    assert got[-5:].tolist() == [drawn(r.float().numpy(), float(np.float32(0.3)), top_p=float(np.float32(0.9))) for r in tail]
    assert got[:3].tolist() == [math.floor(float(np.float32(0.3)) * V)] * 3      # (equal logits are all kept)
    tokens = torch.full((R,), 7, device=DEV)
    want = torch.log_softmax(tail.double(), -1)[:, 7]
    assert bool(((token_logprobs(x, tokens)[-5:].cpu().double() - want).abs() <= _score_bound(tail, 1.0, want)).all())


@pytest.mark.parametrize("dtype", [BF, HF, FP], ids=str)
def test_borders_among_many_alike(dtype):
    """Borders of top-k and top-p among more equal, or nearly equal, logits than a block compares with one another; over and under what one block finishes alone."""
    V = 60000
    gen = torch.Generator().manual_seed(8)
    eps = torch.finfo(dtype).eps
    some = torch.randint(0, 3, (V,), generator=gen).float()
    rows = [4.0 + some * 4 * eps, 4.0 + torch.rand(V, generator=gen) * 0.01, torch.where(torch.rand(V, generator=gen) < 0.02, 6.0 + some * 4 * eps, 1.0), torch.rand(V, generator=gen) * 1e-3]
    x = torch.stack(rows).to(dtype)
    for s in (dict(top_k=700), dict(top_k=30000), dict(top_p=0.3), dict(top_p=0.97, temperature=0.5), dict(top_k=900, top_p=0.5), dict(top_k=300, top_p=0.5, min_p=0.9)):
        _same(x, torch.rand(len(rows), generator=gen), **s)


@pytest.mark.parametrize("dtype", [BF, HF, FP], ids=str)
@pytest.mark.parametrize("R, V", [(6, 60000), (3, 150001), (40, 9000)])
def test_top_p_beside_min_p(R, V, dtype):
    """Borders of min-p below, among and above the numbers that top-p's falls into; one draw from each part of a row."""
    for i, (p, m, t, k) in enumerate([(0.9, 1e-4, 1.0, 0), (0.9, 0.004, 1.0, 0), (0.9, 0.02, 1.0, 0), (0.95, 0.3, 1.0, 0), (0.99, 1e-3, 1.5, 0), (0.7, 0.01, 0.8, 5000), (0.999, 1e-6, 2.0, 0)]):
        x = _logits(R, V, dtype, 50 + i)
        u = torch.arange(R).float().add(0.5).div(R)
        _same(x, u, top_p=p, min_p=m, temperature=t, top_k=k if k else None)


def test_refusals():
    from lit_llama.sampling import sample, token_logprobs

    x, u = torch.zeros(3, 9, device=DEV), torch.zeros(3, device=DEV)
    for kind in (dict(temperature=-1.0), dict(temperature=math.nan), dict(temperature=math.inf), dict(top_k=0), dict(top_k=-1), dict(top_k=2.5), dict(top_p=-0.1), dict(top_p=1.1), dict(top_p=math.nan),
                 dict(min_p=-0.1), dict(min_p=1.1)):
        with pytest.raises(ValueError):
            sample(x, u, **kind)
    for kind in (dict(temperature=u[:2]), dict(temperature=u.double()), dict(top_k=u), dict(top_k=u.long()), dict(top_p=u.cpu()), dict(min_p=u[None])):
        with pytest.raises(RuntimeError):
            sample(x, u, **kind)
    for a, b in ((x, u[:2]), (x, u.double()), (x, u.cpu()), (x.requires_grad_(), u), (torch.zeros(1, (1 << 18) + 1, device=DEV), u[:1]), (torch.zeros(3, 0, device=DEV), u)):
        with pytest.raises(RuntimeError):
            sample(a, b)
    x = torch.zeros(3, 9, device=DEV)
    for tokens in (u, u.int(), u.long()[:2], u.long().cpu()):
        with pytest.raises(RuntimeError):
            token_logprobs(x, tokens)
    for t in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(ValueError):
            token_logprobs(x, u.long(), temperature=t)


def test_captured_draws():
    """Two graphs of one pool's streams, replayed over other logits, numbers and settings; draws on a stream of their own."""
    from lit_llama.sampling import sample, token_logprobs

    R, V = 17, 32000
    x, u, k, p = torch.empty(R, V, dtype=BF, device=DEV), torch.empty(R, device=DEV), torch.empty(R, dtype=torch.int32, device=DEV), torch.empty(R, device=DEV)
    sample(x.zero_(), u.zero_(), top_k=k.zero_(), top_p=p.fill_(1))
    graphs, outs = [], []
    for _ in range(2):
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            t = sample(x, u, top_k=k, top_p=p)
            outs.append((t, token_logprobs(x, t)))
        graphs.append(g)
    gen = torch.Generator().manual_seed(3)
    side = torch.cuda.Stream()
    for i in range(4):
        x.copy_(_logits(R, V, BF, 30 + i))
        u.copy_(torch.rand(R, generator=gen))
        k.copy_(torch.randint(0, 300, (R,), generator=gen))
        p.copy_(torch.rand(R, generator=gen))
        graphs[i % 2].replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            t = sample(x, u, top_k=k, top_p=p)
            lp = token_logprobs(x, t)
        torch.cuda.synchronize()
        assert torch.equal(t, outs[i % 2][0]) and torch.equal(lp, outs[i % 2][1])
        assert t.tolist() == _same(x.cpu(), u.cpu(), top_k=k.cpu(), top_p=p.cpu())


# ---------------------------------------------------------------------------------------------------------------- scores
def _score_bound(x, temperature, want):
    """Half a step of the result; of the sum's exponentials each is off by the rounding of its argument (of size |d|: 2^-24 |d|, twice with the
    difference's) and by 2^-22 of itself, so that the sum's logarithm is by the weighted mean of these."""
    d = (x.double() - x.double().amax(-1, keepdim=True)) / temperature
    p = d.softmax(-1)
    mean = torch.where(p > 0, p * d.abs().clamp(max=1e30), 0.0).sum(-1)
    return want.abs() * 2.0**-23 + mean * 2.0**-22 + 2.0**-21


@pytest.mark.parametrize("dtype", [BF, HF, FP], ids=str)
@pytest.mark.parametrize("R, V", [(3, 1), (4, 2), (5, 33), (130, 1001), (64, 32000), (300, 35000), (9, 100003), (2, 1 << 18)])
def test_scores(R, V, dtype):
    from lit_llama.sampling import token_logprobs

    for seed, temperature in ((0, 1.0), (1, 0.3), (2, 2.5)):
        x = _logits(R, V, dtype, seed)
        if seed == 1 and V > 2:
            x[:, V // 3::2] = -math.inf
            x[R // 2, 1] = torch.finfo(dtype).max                                # sure of its token
        tokens = torch.randint(0, V, (R,), generator=torch.Generator().manual_seed(seed))
        tokens[::2] = x.float().argmax(-1)[::2]
        temperatures = torch.full((R,), temperature)
        want = torch.log_softmax(x.double() / temperatures.double()[:, None], -1).gather(1, tokens[:, None])[:, 0]
        for t in (temperature, temperatures.to(DEV)):
            got = token_logprobs(x.to(DEV), tokens.to(DEV), temperature=t).cpu().double()
            off = want == -math.inf
            assert bool((got[off] == -math.inf).all())
            assert bool(((got - want).abs()[~off] <= _score_bound(x, temperatures.double()[:, None], want)[~off]).all())


def test_scores_of_sure_rows():
    """A token that has all but little: minus the others' sum, not what is left of 1 in 32 bits."""
    from lit_llama.sampling import token_logprobs

    x = torch.tensor([[0.0, 20.0, 0.0, 1.0], [5.0, -30.0, -30.0, -31.0]], device=DEV)
    got = token_logprobs(x, torch.tensor([1, 0], device=DEV)).cpu().double()
    want = torch.log_softmax(x.cpu().double(), -1)
    want = torch.stack((want[0, 1], want[1, 0]))
    # the others' exponentials: arguments rounded (36 at most), 2^-22 of themselves
    assert bool(((got - want).abs() <= want.abs() * (36 * 2.0**-23 + 2.0**-21)).all())


def test_scores_that_are_none():
    from lit_llama.sampling import token_logprobs

    inf, nan = math.inf, math.nan
    x = torch.tensor([[0.0, nan, 1.0], [-inf, -inf, -inf], [0.0, 1.0, 2.0], [0.0, 1.0, 2.0], [0.0, 1.0, 2.0]], device=DEV)
    got = token_logprobs(x, torch.tensor([0, 0, 3, -1, 2**40], device=DEV))
    assert bool(got.isnan().all())
    t = torch.tensor([0.0, -1.0, nan, inf, 1.0], device=DEV)
    got = token_logprobs(x[2:3].expand(5, 3), torch.zeros(5, dtype=torch.int64, device=DEV), temperature=t)
    assert got.isnan().tolist() == [True] * 4 + [False]
    x = torch.tensor([[inf, 0.0, inf], [inf, 0.0, 1.0]], device=DEV)              # the limit
    got = token_logprobs(x.expand(2, 3), torch.tensor([2, 1], device=DEV))
    assert abs(float(got[0]) + math.log(2.0)) <= 2.0**-23 and float(got[1]) == -inf
