"""The weights of a draw, rint(2^44 exp((l - m) / T)), one by one: min-p compares them with a number of 24 bits, which is every whole number up to 2^24.

Exact ones by decimal numbers of 50 digits."""
import math
import random
from decimal import Decimal, getcontext
from fractions import Fraction

import numpy as np
import pytest
import torch

ONE = 1 << 44
DEV = "cuda"
getcontext().prec = 50
LOG2E = 1.4426950408889634


def weight(d, temperature):
    """2^44 exp(d / T) as a Fraction, right to some 48 digits."""
    return Fraction((Decimal(d) / Decimal(temperature)).exp()) * ONE


def whole(x):
    """The nearest whole number, the even one of two (as rint)."""
    return round(x)


def restated(d, temperature):
    """The kernel's arithmetic, rounding by rounding: 256 d / (T ln 2) in 256ths of a power of two, of which the table knows the whole ones, and a polynomial of degree
    four for the rest, before the last rounding to a whole number."""
    fma = lambda a, b, c: float(Fraction(a) * Fraction(b) + Fraction(c))  # noqa: E731
    c, shift, ln = 256 * LOG2E / temperature, 6755399441055744.0, 0.0027076061740622863
    shifted = fma(d, c, shift)
    k = int(shifted - shift)
    r = fma(d, c, shift - shifted)
    p = r * fma(r, fma(r, fma(r, ln * ln * ln * ln / 24, ln * ln * ln / 6), ln * ln / 2), ln)
    at = 2.0 ** ((k & 255) / 256)
    return fma(at, p, at) * 2.0 ** (44 + (k >> 8))


def test_the_arithmetic_of_a_weight():
    """A weight is off by less than 2^-6 of a whole one before it is rounded: by 2^-52 |d / T| of itself with the scale and its division (|x| exp(x) is 0.37 at most, so 2^-9.4), 2^-52 with the
    table (2^-8), 2^-53 with the last product (2^-9) and 2^-54 with the polynomial's next term (2^-10): 2^-6.9 together."""
    rng = random.Random(3)
    other = 0
    for i in range(3000):
        temperature = float(np.float32(rng.choice([1.0, 0.7, 1.3, 0.01, 50.0])))
        d = -float(np.float32(temperature * rng.choice([rng.random() * 31, math.exp(rng.uniform(-14, 3.4))])))
        exact, got = weight(d, temperature), restated(d, temperature)
        assert abs(Fraction(got) - exact) < Fraction(1, 64)
        assert abs(whole(got) - whole(exact)) <= 1
        other += whole(got) != whole(exact)
    assert other <= 3000 // 64 * 2                                            # (those whose fraction is within 2^-6 of a half, on either side)


def _f32(n, up):
    """The number of 24 bits next to n / 2^44, from above or below."""
    x = np.float32(n)
    if up and int(x) < n:
        x = np.nextafter(x, np.float32(np.inf))
    if not up and int(x) > n:
        x = np.nextafter(x, np.float32(0))
    return float(x) / ONE


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("temperature", [1.0, 0.7, 1.3, 0.01, 50.0, 2.0**-60, 1e30])
@pytest.mark.parametrize("V, top_k", [(2, None), (3, 2), (1500, None), (1500, 2), (20000, 2), (40000, None)])
def test_weights(V, top_k, temperature, dtype):
    """Rows of two tokens, the rest masked, u = 1 (the last token that is kept): min-p at a whole one less than the second one's weight, which keeps it, and at two more, which does not."""
    from lit_llama.sampling import sample

    rng = random.Random(5)
    n = 1500 if V < 1000 else 200
    t = float(np.float32(temperature))
    x, p, want = torch.full((2 * n, V), -math.inf), [], []
    while len(want) < 2 * n:
        d = torch.tensor(-t * rng.choice([rng.uniform(8, 30), rng.uniform(11, 31), math.exp(rng.uniform(-14, 3.4))])).to(dtype)
        w = whole(weight(float(d), t))
        if not 3 <= w <= ONE - 3:
            continue
        at = rng.randrange(1, V)
        for keep in (True, False):
            x[len(want), 0], x[len(want), at] = 0.0, d
            p.append(_f32(w - 1, False) if keep else _f32(w + 2, True))
            want.append(at if keep else 0)
    got = sample(x.to(dtype).to(DEV), torch.ones(2 * n, device=DEV), temperature=temperature, top_k=top_k, min_p=torch.tensor(p, dtype=torch.float32, device=DEV)).cpu()
    wrong = int((got != torch.tensor(want)).sum())
    assert wrong == 0, f"{wrong} of {2 * n} weights are off"


@pytest.mark.gpu
def test_a_weight_that_min_p_keeps():
    """exp(-14) 2^44 is 14628408: as many 2^-44 are kept, and one more is not."""
    from lit_llama.sampling import sample
    from tests.util_share import drawn

    x, w = torch.tensor([[0.0, -14.0]]), 14628408
    assert whole(weight(-14.0, 1.0)) == w
    for n in (w - 1, w, w + 1):
        m = _f32(n, True)
        assert float(np.float32(m)) * ONE == n
        want = drawn(x[0].numpy(), 1.0, min_p=m)
        assert want == (1 if n <= w else 0) and sample(x.to(DEV), torch.ones(1, device=DEV), min_p=m).tolist() == [want]
