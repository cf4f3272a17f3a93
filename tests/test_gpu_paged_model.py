"""LLaMA over the paged 4-bit cache: a step of requests of unequal lengths against the same blocks with attention in 64 bits, and generate_batch."""
import math
import sys
from pathlib import Path

import pytest
import torch

from tests.util_paged import held_as, turned

pytestmark = pytest.mark.gpu
DEV, BF = "cuda", torch.bfloat16


def _model(hs=32, quantize=None, n_layer=2):
    from lit_llama import LLaMA, LLaMAConfig
    from lit_llama.utils import EmptyInitOnDevice

    torch.manual_seed(5)
    cfg = LLaMAConfig(block_size=320, vocab_size=100, n_layer=n_layer, n_head=4, n_embd=4 * hs)
    if quantize is None:
        m = LLaMA(cfg).to(DEV, BF)
        m.apply(m._init_weights)
        return m.eval()
    src = _model(hs, n_layer=n_layer)
    with EmptyInitOnDevice(device=DEV, dtype=BF, quantization_mode=quantize):
        m = LLaMA(cfg)
    m.load_state_dict(src.state_dict())
    return m.eval()


def _attend64(q, k, v):
    """``q, k, v [n, H, hs]`` of one request in 64 bits, causal."""
    s = torch.einsum("nhd,lhd->hnl", q.double(), k) / math.sqrt(q.shape[-1])
    s = s.masked_fill(torch.ones(s.shape[1:], dtype=torch.bool).triu(1), -math.inf)
    return torch.einsum("hnl,lhd->nhd", s.softmax(-1), v)


@torch.no_grad()
def _plain(m, prompts, group):
    """Logits of every token: the model's own layers, keys and values as the cache holds them, attention in 64 bits rounded once."""
    n, hs = [len(p) for p in prompts], m.config.head_size
    m._ensure_caches(prompts[0])
    pos = torch.cat([torch.arange(a) for a in n])
    x = m.transformer.wte(torch.cat(prompts))[None]
    for b in m.transformer.h:
        q, k, v = (t.cpu() for t in b.attn.c_attn(b.rms_1(x)).view(sum(n), 3, 4, hs).unbind(1))
        rope = m._rope_f32.cpu()
        q, k, v = turned(q, pos, rope), held_as(turned(k, pos, rope), group), held_as(v, group)
        y = torch.cat([_attend64(*(t.split(n)[i] for t in (q, k, v))) for i in range(len(n))]).to(BF).to(DEV)
        x = x + b.attn.c_proj(y.reshape(1, sum(n), -1))
        x = x + b.mlp(b.rms_2(x))
    return m.lm_head(m.transformer.ln_f(x))[0]


@pytest.mark.parametrize("hs, quantize", [(32, None), (64, None), (128, None), (64, "llm.int8")])
@torch.no_grad()
def test_steps_of_unequal_requests(hs, quantize):
    """Prompts at once, then drafts and single tokens beside one another: the logits of the whole sequences.  An output of the attention may be off by
    one rounding of bf16, 2^-8 of its size, and by no more than about as much again for its weights; two layers add that to a stream of which they are
    a part: 2^-8 * 2 * 2 of the logits' norm, and as much for llm.int8, whose steps at a border of two codes a place of its inputs moves."""
    m = _model(hs, quantize)
    whole = [torch.randint(0, 100, (n,), device=DEV) for n in (70, 3, 129, 64, 1)]
    want = _plain(m, whole, 32)
    cache = m.paged_cache(pages=12, requests=6, group=32)
    cache.free.copy_(torch.randperm(12))
    rows, fed, got = [4, 0, 5, 2, 3], [0] * 5, [[] for _ in whole]
    for counts in ([60, 0, 100, 33, 0], [1, 1, 1, 0, 1], [5, 2, 28, 31, 0], [4, 0, 0, 0, 0]):
        plan = cache.plan(rows, counts, sum(counts), max_count=max(counts))
        plan.check()
        tokens = torch.cat([w[f:f + c] for w, f, c in zip(whole, fed, counts)])
        logits = m.forward_paged(tokens, cache, plan, all_rows=True)
        for i, part in enumerate(logits.split(counts)):
            got[i].append(part)
            fed[i] += counts[i]
    assert fed == [len(w) for w in whole]
    got = torch.cat([torch.cat(g) for g in got])
    assert float((got.double() - want.double()).norm() / want.double().norm()) <= (2 if quantize else 1) * 4 * 2.0 ** -8


@torch.no_grad()
def test_the_last_tokens_logits():
    m = _model()
    cache = m.paged_cache(pages=9, requests=3)
    tokens = torch.randint(0, 100, (31,), device=DEV)
    a = m.forward_paged(tokens, cache, cache.plan([2, 1, 0], [20, 1, 10], 31))
    cache.truncate([0, 1, 2], [0, 0, 0])
    b = m.forward_paged(tokens, cache, cache.plan([2, 1, 0], [20, 1, 10], 31), all_rows=True)
    assert a.shape == (3, 128) and float((a - b[[19, 20, 30]]).abs().max()) <= 2.0 ** -7 * float(b.abs().max())      # (other sizes of product: one place)


@pytest.mark.parametrize("quantize", [None, "llm.int8"])
@torch.no_grad()
def test_generate_batch(quantize):
    """Every token drawn with top_k 1 is, up to the places that kernels of other sizes round otherwise, the best of its sequence's own logits."""
    sys.path.insert(0, str(Path(__file__).parent.parent / "lit-llama-ja_b200"))
    from generate import generate_batch

    m = _model(64, quantize)
    prompts = [torch.randint(0, 100, (n,), device=DEV) for n in (40, 1, 65, 130)]
    out = generate_batch(m, prompts, 9, top_k=1, group=32)
    assert [len(o) for o in out] == [len(p) + 9 for p in prompts] and all(torch.equal(o[:len(p)], p) for o, p in zip(out, prompts))
    cache = m.paged_cache(pages=40, requests=4, group=32)
    n = [len(o) - 1 for o in out]
    logits = m.forward_paged(torch.cat([o[:-1] for o in out]), cache, cache.plan(range(4), n, sum(n)), all_rows=True).float()
    slack = (2 if quantize else 1) * 4 * 2.0 ** -8 * float(logits.abs().max())
    for part, o, p in zip(logits.split(n), out, prompts):
        part = part[len(p) - 1:]
        assert bool((part.gather(1, o[len(p):, None])[:, 0] >= part.max(1).values - slack).all())


@torch.no_grad()
def test_generate_batch_of_int4_weights(golden):
    """Weights in 4 bits too: rows of a step through the modules that single tokens, batches and prompts take."""
    from generate import generate_batch
    from tests.test_gpu_model import build_q_model

    m = build_q_model(golden["model_tiny"], "rtn32bf16.", BF)
    prompts = [torch.randint(0, 100, (n,), device=DEV) for n in (20, 1, 33)]
    out = generate_batch(m, prompts, 8, top_k=1)
    assert [len(o) for o in out] == [len(p) + 8 for p in prompts]
    cache = m.paged_cache(pages=6, requests=3)
    n = [len(o) - 1 for o in out]
    logits = m.forward_paged(torch.cat([o[:-1] for o in out]), cache, cache.plan(range(3), n, sum(n)), all_rows=True).float()
    slack = 4 * 2.0 ** -8 * float(logits.abs().max())
    for part, o, p in zip(logits.split(n), out, prompts):
        part = part[len(p) - 1:]
        assert bool((part.gather(1, o[len(p):, None])[:, 0] >= part.max(1).values - slack).all())


@torch.no_grad()
def test_generate_batch_ends_at_eos():
    """Sequences that meet the end token stop before it and no longer change; the others go on."""
    from generate import generate_batch

    m = _model(64)
    prompts = [torch.randint(0, 100, (n,), device=DEV) for n in (12, 30, 7)]
    full = generate_batch(m, prompts, 12, top_k=1)
    eos = int(full[1][len(prompts[1])])                       # the second one's first token
    cut = generate_batch(m, prompts, 12, top_k=1, eos_id=eos)
    assert torch.equal(cut[1], prompts[1])
    for f, c, p in zip(full, cut, prompts):
        # (tokens after the first may differ where two logits are alike: sums of other sizes)
        assert eos not in c[len(p):].tolist() and len(p) <= len(c) <= len(p) + 12 and torch.equal(c[:len(p)], p)
        assert len(c) == len(p) or int(c[len(p)]) == int(f[len(p)])


@torch.no_grad()
def test_refusals():
    from lit_llama.adapter import LLaMA as Adapter, LLaMAConfig as AdapterConfig

    m = _model()
    cache = m.paged_cache(pages=4, requests=2)
    plan = cache.plan([0], [3], 3)
    tokens = torch.zeros(3, dtype=torch.int64, device=DEV)
    other = _model(n_layer=3)
    adapter = Adapter(AdapterConfig(block_size=320, vocab_size=100, n_layer=2, n_head=4, n_embd=128, adapter_prompt_length=3, adapter_start_layer=1)).to(DEV, BF)
    with pytest.raises(ValueError, match="block size"):
        m.paged_cache(pages=4, requests=2, max_length=321)
    for call in (lambda: m.forward_paged(tokens[:2], cache, plan), lambda: m.forward_paged(tokens.float(), cache, plan), lambda: other.forward_paged(tokens, cache, plan),
                 lambda: adapter.forward_paged(tokens, cache, plan)):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(ValueError):
        _model().float().paged_cache(pages=4, requests=2)
