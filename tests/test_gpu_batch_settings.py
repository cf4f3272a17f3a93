"""Settings of generate_batch that are tensors: numbers without a dimension and columns are the settings of torch's draw, vectors are one number a sequence."""
import sys
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu
sys.path.insert(0, str(Path(__file__).parent.parent / "lit-llama-ja_b200"))
DEV, BF = "cuda", torch.bfloat16


@torch.no_grad()
def test_settings_without_a_dimension():
    from generate import generate_batch
    from lit_llama import LLaMA, LLaMAConfig

    torch.manual_seed(5)
    m = LLaMA(LLaMAConfig(block_size=320, vocab_size=100, n_layer=2, n_head=4, n_embd=256)).to(DEV, BF)
    m.apply(m._init_weights)
    m.eval()
    prompts = [torch.randint(0, 100, (n,), device=DEV) for n in (20, 70)]
    out = []
    for t, k in ((0.5, 20), (torch.tensor(0.5), 20), (torch.tensor(0.5, device=DEV), torch.tensor(20)), (torch.full((2, 1), 0.5, device=DEV, dtype=BF), 20)):
        torch.manual_seed(3)
        out.append(generate_batch(m, prompts, 8, temperature=t, top_k=k))
    for other in out[1:]:
        assert all(torch.equal(a, b) for a, b in zip(out[0], other))
    rows = generate_batch(m, prompts, 8, temperature=torch.full((2,), 0.5, device=DEV), top_k=torch.tensor([1, 20], dtype=torch.int32, device=DEV))
    assert [len(r) for r in rows] == [28, 78]
