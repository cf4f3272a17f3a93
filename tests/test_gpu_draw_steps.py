"""Draws whose borders lie where two of the steps meet by which a draw looks for them: logits half way between the middles of two steps, and a few roundings beside that."""
import math
import random

import numpy as np
import pytest
import torch

from tests.util_share import drawn

pytestmark = pytest.mark.gpu
DEV = "cuda"
STEP = 31.25 / 1024                   # of a temperature


def _rows(dtype, m, n, seed):
    """(logit, temperature) pairs that are (k + 1/2) steps below m but for a few roundings of the temperature."""
    rng = random.Random(seed)
    out = []
    while len(out) < n:
        x = float(torch.tensor(m - math.exp(rng.uniform(-4, 3))).to(dtype))
        k = rng.randrange(0, 400)
        if not x < m:
            continue
        t = np.float32((m - x) / ((k + 0.5) * STEP))
        for _ in range(abs(j := rng.randrange(-4, 5))):
            t = np.nextafter(t, np.float32(np.inf if j > 0 else 0))
        out.append((x, float(t)))
    return out


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("V, n", [(4, 4000), (300, 2000), (1500, 1000), (20000, 150), (40000, 150), (140000, 40)])
@pytest.mark.parametrize("kind", ["top_k", "top_p", "both"])
def test_borders_between_steps(kind, V, n, dtype):
    """Three tokens of a row that is else masked: the border is at the second one, which is drawn by u = 1 where it comes last, and by a smaller number too."""
    m = float(torch.tensor(-999.1875 if dtype is torch.float32 else 3.0).to(dtype))
    pairs = _rows(dtype, m, n, V)
    rng = random.Random(V)
    x = torch.full((n, V), -math.inf)
    places = [sorted(rng.sample(range(V), 3)) for _ in range(n)]
    top_p, u = [], []
    for r, ((v, t), (a, b, c)) in enumerate(zip(pairs, places)):
        third = float(torch.tensor(v - 2 * t).to(dtype))
        x[r, a], x[r, b], x[r, c] = third, m, v
        w = [math.exp((z - m) / t) for z in (m, v, third)]
        top_p.append((w[0] + 0.5 * w[1]) / (w[0] + w[1] + (0.0 if kind == "both" else w[2])))
        u.append(1.0 if r % 2 else (w[0] + 0.5 * w[1]) / (w[0] + w[1]))
    x = x.to(dtype)
    settings = dict(temperature=torch.tensor([t for _, t in pairs], dtype=torch.float32))
    if kind != "top_p":
        settings["top_k"] = torch.full((n,), 2, dtype=torch.int32)
    if kind != "top_k":
        settings["top_p"] = torch.tensor(top_p, dtype=torch.float32)
    u = torch.tensor(u, dtype=torch.float32)
    from lit_llama.sampling import sample

    got = sample(x.to(DEV), u.to(DEV), **{k: s.to(DEV) for k, s in settings.items()}).tolist()
    wrong = []
    for r, (place, (v, t)) in enumerate(zip(places, pairs)):
        few = x[r, place].float().numpy()      # (the others weigh nothing)
        want = place[drawn(few, float(u[r]), **{k: (int if k == "top_k" else float)(s[r]) for k, s in settings.items()})]
        if got[r] != want:
            wrong.append((r, v, t))
    assert not wrong, f"{len(wrong)} of {n}: {wrong[:3]}"
