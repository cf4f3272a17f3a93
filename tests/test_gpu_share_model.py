"""Several answers to a prompt: generate and generate_batch with top-p and min-p, forked requests through the model, scores."""
import sys
from pathlib import Path

import pytest
import torch

from tests.util_share import drawn

pytestmark = pytest.mark.gpu
sys.path.insert(0, str(Path(__file__).parent.parent / "lit-llama-ja_b200"))
DEV, BF = "cuda", torch.bfloat16


def _model(block_size=320, n_layer=2):
    from lit_llama import LLaMA, LLaMAConfig

    torch.manual_seed(5)
    m = LLaMA(LLaMAConfig(block_size=block_size, vocab_size=100, n_layer=n_layer, n_head=4, n_embd=256)).to(DEV, BF)
    m.apply(m._init_weights)
    return m.eval()


def _same_tokens_again(m, sequences, prompts, group=32):
    """Logits of the sequences' own steps, all at once, and the slack of sums of other sizes: 2^-8 a sum, two layers, products and attention."""
    cache = m.paged_cache(pages=sum(-(-len(o) // 64) for o in sequences), requests=len(sequences), group=group)
    n = [len(o) - 1 for o in sequences]
    logits = m.forward_paged(torch.cat([o[:-1] for o in sequences]), cache, cache.plan(range(len(n)), n, sum(n)), all_rows=True).float()
    return [part[len(p) - 1:] for part, p in zip(logits.split(n), prompts)], 4 * 2.0 ** -8 * float(logits.abs().max())


@pytest.mark.parametrize("block_size", [320, 1024])
@torch.no_grad()
def test_answers_that_share_their_prompt(block_size):
    """The best token at every step: the answers to a prompt are alike, and those that the model gives to its sequence; lengths at, before and behind pages' ends.
    (Caches for more than 512 tokens walk shared pages once.)"""
    from generate import generate_batch

    m = _model(block_size)
    sizes = (40, 1, 64, 130) if block_size == 320 else (700, 128, 1, 639)
    prompts = [torch.randint(0, 100, (n,), device=DEV) for n in sizes]
    new = 70 if block_size == 320 else 9
    out = generate_batch(m, prompts, new, top_k=1, group=32, samples=3)
    assert len(out) == 12 and all(torch.equal(o[:len(p)], p) and len(o) == len(p) + new for o, p in zip(out, [p for p in prompts for _ in range(3)]))
    parts, slack = _same_tokens_again(m, out, [p for p in prompts for _ in range(3)])
    for part, o in zip(parts, out):
        t = o[-new:, None]
        assert bool((part.gather(1, t)[:, 0] >= part.max(1).values - slack).all())


@torch.no_grad()
def test_drawn_answers_and_their_scores():
    """Tokens from the same numbers, one by one on the host from the same logits; their log-probabilities; sequences that end."""
    import generate
    from generate import generate_batch

    m = _model()
    prompts = [torch.randint(0, 100, (n,), device=DEV) for n in (20, 70)]
    seen, real = [], generate.sample

    def noted(logits, u, **s):
        seen.append((logits.float().cpu(), u.cpu(), real(logits, u, **s).cpu()))
        return real(logits, u, **s)

    generate.sample = noted
    try:
        k = torch.tensor([5, 0, 50, 1, 0, 100, 2, 3], dtype=torch.int32, device=DEV)
        torch.manual_seed(3)
        out, scores = generate_batch(m, prompts, 8, temperature=0.7, top_k=k, top_p=0.9, min_p=0.01, samples=4, logprobs=True)
    finally:
        generate.sample = real
    assert len(out) == len(scores) == 8 and len(seen) == 8
    for i, (logits, u, tokens) in enumerate(seen):
        for b in range(8):
            want = drawn(logits[b].numpy(), float(u[b]), float(torch.tensor(0.7)), int(k[b]), float(torch.tensor(0.9)), float(torch.tensor(0.01)))
            assert int(tokens[b]) == want and int(out[b][len(prompts[b // 4]) + i]) == want
            # (scores of fp32: half a step, and 2^-22 for each of the sum's terms and their arguments of up to 16)
            p = torch.log_softmax(logits[b].double(), -1)[want]
            assert abs(float(scores[b][i]) - float(p)) <= 2.0**-17
    eos = int(out[0][20])
    torch.manual_seed(3)
    cut, parts = generate_batch(m, prompts, 8, temperature=0.7, top_k=k, top_p=0.9, min_p=0.01, samples=4, logprobs=True, eos_id=eos)
    assert torch.equal(cut[0], prompts[0]) and parts[0].numel() == 0 and all(eos not in c[len(prompts[b // 4]):].tolist() for b, c in enumerate(cut))


@torch.no_grad()
def test_one_sequence_by_top_p():
    from generate import generate

    m = _model()
    prompt = torch.randint(0, 100, (17,), device=DEV)
    torch.manual_seed(1)
    a = generate(m, prompt, 12, temperature=0.9, top_p=0.8)
    m.reset_cache()
    torch.manual_seed(1)
    b = generate(m, prompt, 12, temperature=0.9, top_p=0.8)
    m.reset_cache()
    assert torch.equal(a, b) and len(a) == 29
    # the best tokens: logits of bf16 are often alike, equal ones are kept together and drawn by the same numbers; at temperature 0 the first of them, by any
    best = []
    for seed, kind in ((2, dict(top_k=1, min_p=0.5)), (2, dict(temperature=0.5, top_p=0.0)), (3, dict(temperature=0.0, min_p=0.1)), (4, dict(temperature=0.0, top_p=1.0))):
        torch.manual_seed(seed)
        best.append(generate(m, prompt, 12, **kind))
        m.reset_cache()
    assert torch.equal(best[0], best[1]) and torch.equal(best[2], best[3])


@torch.no_grad()
def test_logits_that_allow_no_draw():
    """A model whose logits are no numbers: an error at the end, and no token outside of the table on the way."""
    from generate import generate, generate_batch

    m = _model()
    m.lm_head.weight.fill_(float("nan"))
    prompt = torch.randint(0, 100, (9,), device=DEV)
    with pytest.raises(RuntimeError, match="no draw"):
        generate_batch(m, [prompt, prompt[:4]], 5, top_p=0.9)
    with pytest.raises(RuntimeError, match="no draw"):
        generate(m, prompt, 3, min_p=0.1)


@torch.no_grad()
def test_refusals():
    from generate import generate_batch, main

    m = _model()
    prompt = torch.randint(0, 100, (9,), device=DEV)
    for kind in (dict(samples=0), dict(top_p=2.0), dict(min_p=-1.0), dict(top_p=0.9, temperature=-1.0)):
        with pytest.raises(ValueError):
            generate_batch(m, [prompt], 4, **kind)
    with pytest.raises(RuntimeError):
        generate_batch(m, [prompt], 4, samples=2, temperature=torch.ones(1, device=DEV))
    with pytest.raises(ValueError):
        main(share_prompt=True)


@torch.no_grad()
def test_the_command_line(monkeypatch, capsys, tmp_path):
    import generate

    (tmp_path / "x.pth").write_bytes(b"")
    monkeypatch.setattr(generate, "load_model", lambda *a: _model())
    for kind in (dict(kv_cache="int4", share_prompt=True), dict(kv_cache="int4"), dict()):
        generate.main(checkpoint_path=tmp_path / "x.pth", prompt_ids="5,17,3", num_samples=3, max_new_tokens=7, top_p=0.9, min_p=0.02, **kind)
        lines = [[int(t) for t in line.split(",")] for line in capsys.readouterr().out.split()]
        assert len(lines) == 3 and all(x[:3] == [5, 17, 3] and len(x) == 10 and max(x) < 128 for x in lines)
