"""What the operators of several answers to one prompt are measured on: their plain forms, and the framework's kernels on the same inputs.

The operators, in the order of a serving step:

``fork``      requests of the paged key/value cache become copies of others: whole pages are shared, the last one, which is still written, is copied; ``truncate``
              into a page that others hold copies it, and pages that nobody holds any more are free again
``attend``    softmax attention of a step whose requests share pages: what they share, and what each has of its own
``sample``    a token a row of logits from given random numbers, with temperature, top-k, top-p and min-p
``logprobs``  log-probabilities of given tokens

A draw from a row l with temperature T, in whole numbers so that no sum depends on an order: with the largest logit m,

    w_i = rint(2^44 exp((l_i - m) / T))                     weights, in 64 bits
    top-k   keeps what is at least as large as the k-th largest logit (equal ones together)
    top-p   keeps the largest ones up to the first logit with which their weights reach top_p of what top-k left (equal ones together)
    min-p   keeps w_i >= min_p 2^44
    token   the first one whose running sum of kept weights is more than floor(u times their sum)
"""
import math
import random
import sys

import numpy as np
import torch

own = False

PAGE = 64
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ONE = 1 << 44


def listed():
    return [
        # sixteen answers to one prompt of the 7B configuration's heads (two layers of them)
        dict(name="fork_samples", op="fork", sources=1, copies=16, longest=500, layers=2, kv_heads=32, head_size=128, group=64, pool=1.0, rewind=0, mix=1),
        # a search over many requests of odd lengths, for a pool that does not hold all copies; eight key heads
        dict(name="fork_many", op="fork", sources=29, copies=7, longest=2001, layers=5, kv_heads=8, head_size=64, group=32, pool=0.9, rewind=0, mix=2),
        # copies that are cut back into the pages that they share, and go on from there
        dict(name="fork_rewind", op="fork", sources=5, copies=9, longest=1472, layers=3, kv_heads=32, head_size=128, group=128, pool=1.0, rewind=700, mix=3),
        # four answers of the smallest configuration: latency
        dict(name="attend_small", op="attend", sources=1, copies=4, longest=300, more=40, heads=8, kv_heads=8, head_size=64, group=64, dtype="bf16", mix=4),
        # 64 answers to a prompt of the 7B configuration's block size
        dict(name="attend_7b", op="attend", sources=1, copies=64, longest=2048, more=200, heads=32, kv_heads=32, head_size=128, group=64, dtype="bf16", mix=5),
        # some answers each to a few prompts of odd lengths, eight key heads
        dict(name="attend_groups", op="attend", sources=5, copies=13, longest=3333, more=333, heads=32, kv_heads=8, head_size=128, group=32, dtype="fp16", mix=6),
        # one user: the command line's settings, latency
        dict(name="sample_one", op="sample", rows=1, vocab=32000, dtype="bf16", k="all", p="none", floor="none", masked=0.0, mix=7),
        # a served batch whose requests differ in all their settings
        dict(name="sample_batch", op="sample", rows=64, vocab=32000, dtype="bf16", k="some", p="some", floor="some", masked=0.1, mix=8),
        # many rows of an odd, larger vocabulary in 32 bits, by their mass alone
        dict(name="sample_wide", op="sample", rows=301, vocab=100003, dtype="fp32", k="none", p="all", floor="some", masked=0.0, mix=9),
        # the tokens of a step of 64 requests
        dict(name="logprobs_step", op="logprobs", rows=64, vocab=32000, dtype="bf16", masked=0.0, mix=10),
        # a text of the 7B configuration's block size
        dict(name="logprobs_text", op="logprobs", rows=2048, vocab=32000, dtype="bf16", masked=0.0, mix=11),
        # rows that begin at odd places, in 32 bits
        dict(name="logprobs_wide", op="logprobs", rows=777, vocab=100003, dtype="fp32", masked=0.1, mix=12),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["fork", "attend", "attend", "sample", "sample", "sample", "logprobs"])
    case = dict(op=op, mix=rng.randrange(1 << 30))
    if op in ("sample", "logprobs"):
        vocab = rng.choice([32000, _spread(rng, 2, 200000), _spread(rng, 1000, 200000)])
        most = (30_000_000 if op == "sample" else 75_000_000) // vocab
        case.update(rows=_spread(rng, 1, min(4000, most)), vocab=vocab, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), masked=rng.choice([0.0, 0.0, 0.1, 0.9]))
        if op == "sample":
            case.update(k=rng.choice(["none", "all", "some"]), p=rng.choice(["none", "all", "some"]), floor=rng.choice(["none", "none", "all", "some"]))
        return case
    kv = rng.choice([1, 2, 4, 8, 10, 32])
    size = rng.choice([32, 64, 128, 128])
    group = rng.choice([g for g in (32, 64, 128) if g <= size])
    case.update(kv_heads=kv, head_size=size, group=group, sources=_spread(rng, 1, 30), copies=_spread(rng, 2, 64), longest=_spread(rng, 20, 4000))
    case["copies"] = max(1, min(case["copies"], 100 // case["sources"]))
    if op == "fork":
        case.update(layers=rng.randrange(1, 7), pool=rng.choice([0.8, 1.0, 1.0]), rewind=rng.choice([0, 0, rng.randrange(1, case["longest"] + 1)]))
        if case["rewind"]:
            case.update(pool=1.0, longest=-(-case["longest"] // PAGE) * PAGE)
        while case["layers"] * _pool(case) * kv * page_bytes(case) > 100_000_000 and (case["sources"] > 1 or case["layers"] > 1):
            case["sources" if case["sources"] > 1 else "layers"] //= 2
        return case
    case.update(heads=kv * rng.choice([1, 1, 1, 4] if kv > 4 else [1, 2, 4, 8]), more=_spread(rng, 1, 400), dtype=rng.choice(["bf16", "bf16", "fp16"]))
    # keys and values of the plain form in 32 bits, padded to the longest request, no more than those of the largest listed case
    while case["copies"] > 1 and case["sources"] * case["copies"] * (case["longest"] + case["more"]) * kv * size > 600_000_000:
        case["copies"] //= 2
    return case


def _pages(n):
    return -(-n // PAGE)


def page_bytes(case):
    """Bytes of one head's page: 64 keys and values of 4 bits, a scale and a lowest value of 16 for each group."""
    D = case["head_size"]
    return PAGE * (D + 8 * (D // case["group"]))


def lengths_of(case):
    """Tokens of the sources and of every copy's own part, the first ones the longest."""
    rng = random.Random(case["mix"])
    n, longest = case["sources"], case["longest"]
    held = [longest] + [rng.randrange(1, longest + 1) for _ in range(n - 1)]
    if case.get("rewind"):
        held = [_pages(h) * PAGE for h in held]
    more = case.get("more", 0)
    return held, [[rng.randrange(0, more) + 1 if more else 0 for _ in range(case["copies"])] for _ in held]


def _pool(case):
    """Pages that the requests of a fork hold, and those of its copies."""
    held, _ = lengths_of(case)
    have = sum(_pages(h) for h in held)
    wanted = case["copies"] * (sum(1 for h in held if h % PAGE) if not case["rewind"] else case["sources"])
    return have + math.ceil(wanted * case["pool"])


# ---------------------------------------------------------------------------------------------------------------- the plain forms
def _scatter_some(to, at, what, where):
    """``to`` with what[i] at at[i] for the places that ``where`` names; the others go to a place behind the end."""
    more = torch.cat([to, to.new_zeros(1)])
    return more.scatter(0, torch.where(where, at, to.numel()).reshape(-1), torch.where(where, what, 0).reshape(-1).to(to.dtype))[:-1]


def _copy_pages(blocks, src, dst, which):
    src, dst = src[which].long(), dst[which].long()
    blocks[:, dst] = blocks[:, src]


def plain_truncate(s, rows, keep):
    """Cuts requests to ``keep`` tokens.  One that ends inside a page which others hold gets a copy of it, or stays as it was where there is no page for
    that (status 1); a page is free again when its last holder has given it back, in the order of the requests."""
    P = s["table"].shape[1]
    rows = rows.long()
    old = s["lengths"][rows].long()
    keep = torch.minimum(keep.long(), old)
    table = s["table"][rows]
    part = keep // PAGE
    last = table.gather(1, part.clamp(max=P - 1)[:, None])[:, 0].long().clamp(min=0)
    copies = (keep < old) & (keep % PAGE > 0) & (s["shared"][last] > 0)
    used = copies.long().cumsum(0)
    refused = copies & (used > s["n_free"])
    copies &= ~refused
    keep = torch.where(refused, old, keep)
    new = s["free"][(s["n_free"].long() - used).clamp(min=0)]
    n_free = s["n_free"].long() - copies.sum()
    page = torch.arange(P, device=rows.device)
    first = torch.where(copies, part, (keep + PAGE - 1) // PAGE)
    given = (page >= first[:, None]) & (page < ((old + PAGE - 1) // PAGE)[:, None])
    held = torch.where(given, table, 0).long()
    shared = s["shared"].long() - torch.zeros_like(s["shared"]).long().index_add(0, held.reshape(-1), given.reshape(-1).long())
    seq = torch.arange(rows.numel(), device=rows.device)[:, None].expand_as(held)
    latest = torch.full_like(shared, -1).scatter_reduce(0, held.reshape(-1), torch.where(given, seq, -1).reshape(-1), "amax")
    freed = given & (shared[held] < 0) & (latest[held] == seq)
    order = freed.reshape(-1).long().cumsum(0).reshape(freed.shape)
    s["free"] = _scatter_some(s["free"], n_free + freed.sum() - order, table, freed)
    s["n_free"] = (n_free + freed.sum()).int()
    s["shared"] = shared.clamp(min=0).int()
    _copy_pages(s["blocks"], last, new, copies)
    table = torch.where(given, -1, table)
    table = torch.where(copies[:, None] & (page == part[:, None]), new[:, None], table)
    s["table"] = s["table"].index_copy(0, rows, table)
    s["lengths"] = s["lengths"].index_copy(0, rows, keep.int())
    return refused.int()


def plain_fork(s, rows, into):
    """Empty requests ``into`` become copies of ``rows``: whole pages are shared, a last one that is not full is copied to a page from the stack (status 1
    where there is none)."""
    P = s["table"].shape[1]
    rows, into = rows.long(), into.long()
    old = s["lengths"][rows].long()
    table = s["table"][rows]
    whole, partial = old // PAGE, old % PAGE > 0
    used = partial.long().cumsum(0)
    refused = partial & (used > s["n_free"])
    copies = partial & ~refused
    new = s["free"][(s["n_free"].long() - used).clamp(min=0)]
    page = torch.arange(P, device=rows.device)
    share = (page < whole[:, None]) & ~refused[:, None]
    s["shared"] = s["shared"].index_add(0, torch.where(share, table, 0).long().reshape(-1), share.reshape(-1).int())
    _copy_pages(s["blocks"], table.gather(1, whole.clamp(max=P - 1)[:, None])[:, 0], new, copies)
    mine = torch.where(share, table, -1)
    mine = torch.where(copies[:, None] & (page == whole[:, None]), new[:, None], mine)
    s["table"] = s["table"].index_copy(0, into, mine)
    s["lengths"] = s["lengths"].index_copy(0, into, torch.where(refused, 0, old).int())
    s["n_free"] = (s["n_free"] - copies.sum()).int()
    return refused.int()


def plain_values(c, s, lo):
    g = c.float().unflatten(-1, (s.shape[-1], -1))
    return (g * s.float()[..., None] + lo.float()[..., None]).flatten(-2)


def plain_attend(s):
    """All requests at once, padded to the longest: keys and values of 32 bits, scores, their softmax and the weighted sum."""
    q, table, lengths = s["q"], s["table"], s["lengths"]
    B, H, D = q.shape
    j = torch.arange(s["longest"], device=q.device)
    page, at = table[:, j // PAGE].long().clamp(min=0), j % PAGE
    k, v = (plain_values(*(a[page, at] for a in s[x])) for x in "kv")        # [B, L, Hkv, D]
    there = j < lengths[:, None]
    v = torch.where(there[:, :, None, None], v, 0)
    mine = (q.float() * D ** -0.5).unflatten(1, (k.shape[2], -1))            # [B, Hkv, G, D]
    scores = torch.matmul(mine, k.permute(0, 2, 3, 1)).masked_fill(~there[:, None, None], -math.inf)
    w = torch.exp(scores - scores.amax(-1, keepdim=True))
    return (torch.matmul(w, v.permute(0, 2, 1, 3)) / w.sum(-1, keepdim=True)).flatten(1, 2).to(q.dtype)


def plain_sample(logits, u, temperature, top_k, top_p, min_p):
    x = logits.double()
    m = x.amax(-1, keepdim=True)
    w = torch.exp((x - m) * (1.0 / temperature.double())[:, None])
    w = torch.round(torch.where(x == m, 1.0, w) * ONE).long()
    kept = w > 0
    if top_k is not None or top_p is not None:
        ordered, at = logits.sort(-1, descending=True)
        if top_k is not None:
            kept &= logits >= ordered.gather(1, (top_k.long().clamp(max=x.shape[1]) - 1)[:, None])
        if top_p is not None:
            mass = torch.where(kept, w, 0).gather(1, at).cumsum(-1)
            reached = mass.double() >= top_p.double()[:, None] * mass[:, -1:].double()
            kept &= logits >= ordered.gather(1, reached.long().argmax(-1, keepdim=True))
    if min_p is not None:
        kept &= w.double() >= min_p.double()[:, None] * ONE
    mass = torch.where(kept, w, 0).cumsum(-1)
    total = mass[:, -1]
    target = torch.minimum((u.double() * total.double()).floor().long(), total - 1)
    token = (mass <= target[:, None]).sum(-1)
    return torch.where(m[:, 0] == -math.inf, -1, token)


def plain_logprobs(logits, tokens, temperature):
    x = logits.float() / temperature
    m = x.amax(-1)
    return x.gather(1, tokens[:, None])[:, 0] - m - torch.log(torch.exp(x - m[:, None]).sum(-1))


# ---------------------------------------------------------------------------------------------------------------- inputs
def _package():
    if "lit-llama-ja_b200" not in sys.path:
        sys.path.insert(0, "lit-llama-ja_b200")
    from lit_llama.paged_cache import PagedCache4
    from lit_llama.sampling import sample, token_logprobs

    return PagedCache4, sample, token_logprobs


def _int(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _logits(case, gen):
    """A head's logits: most tokens unlikely, a few far above them, some rows sure of theirs; masked ones at -inf or at the type's lowest value."""
    R, V, dtype = case["rows"], case["vocab"], DTYPES[case["dtype"]]
    x = torch.randn(R, V, generator=gen, device="cuda") * 2.2 - 1.0
    few = torch.randint(0, V, (R, 12), generator=gen, device="cuda")
    x.scatter_add_(1, few, 9.0 * torch.rand(R, 12, generator=gen, device="cuda") * torch.rand(R, 1, generator=gen, device="cuda"))
    x = x.to(dtype)
    if case["masked"]:
        low = torch.where(torch.rand(R, 1, generator=gen, device="cuda") < 0.5, -math.inf, torch.finfo(dtype).min).to(dtype)
        off = torch.rand(R, V, generator=gen, device="cuda") < case["masked"]
        off[:, 0] = False
        x = torch.where(off, low, x)
    return x


def _setting(kind, R, gen, values, off):
    """A setting of the rows: none, one of all, or another one each, some without."""
    if kind == "none":
        return None
    x = torch.tensor(values, device="cuda")[torch.randint(0, len(values), (R,), generator=gen, device="cuda")]
    if kind == "all":
        return x[:1].expand(R).contiguous()
    return torch.where(torch.rand(R, generator=gen, device="cuda") < 0.25, torch.tensor(off, device="cuda", dtype=x.dtype), x)


def inputs(case, seed):
    """Everything that both sides and the 64-bit form start from."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] in ("sample", "logprobs"):
        R, V = case["rows"], case["vocab"]
        x = dict(logits=_logits(case, gen))
        if case["op"] == "logprobs":
            # half of the tokens are likely ones
            likely, some = x["logits"].argmax(-1), torch.randint(0, V, (R,), generator=gen, device="cuda")
            some = torch.where(x["logits"].gather(1, some[:, None])[:, 0] > -1e4, some, 0)
            return dict(x, tokens=torch.where(torch.rand(R, generator=gen, device="cuda") < 0.5, likely, some), temperature=1.0)
        return dict(x, u=torch.rand(R, generator=gen, device="cuda"),
                    temperature=_setting("some" if case["k"] == "some" else "all", R, gen, [0.6, 0.8, 1.0, 1.3], 1.0).float(),
                    top_k=_setting(case["k"], R, gen, np.array([1, 5, 40, 50, 200, 200, 1000], dtype=np.int32), V), top_p=_setting(case["p"], R, gen, [0.5, 0.8, 0.9, 0.95, 0.99], 1.0),
                    min_p=_setting(case["floor"], R, gen, [0.01, 0.02, 0.05, 0.1], 0.0))
    held, more = lengths_of(case)
    n, c = case["sources"], case["copies"]
    x = dict(held=_int(held), rows=torch.arange(n, dtype=torch.int32, device="cuda").repeat_interleave(c),
             into=torch.arange(n, n + n * c, dtype=torch.int32, device="cuda"), max_length=max(held) + case.get("more", 0))
    if case["op"] == "fork":
        pages = _pool(case)
        x.update(pages=pages, order=torch.randperm(pages, generator=gen, device="cuda").int(),
                 blocks=torch.randint(0, 256, (case["layers"], pages, case["kv_heads"], page_bytes(case)), generator=gen, device="cuda", dtype=torch.uint8))
        if case["rewind"]:
            x["cut"] = (torch.rand(n * c, generator=gen, device="cuda") * x["held"].repeat_interleave(c).clamp(max=case["rewind"])).int() + 1
        return x
    dtype, H, K, D = DTYPES[case["dtype"]], case["heads"], case["kv_heads"], case["head_size"]
    # some dimensions of a head's keys are much larger than the others
    loud = torch.where(torch.rand(K, D, generator=gen, device="cuda") < 0.03, 6.0, 1.0)
    own_part = [m for of_one in more for m in of_one]
    total = sum(held) + sum(own_part)
    k, v = (torch.randn(total, K, D, generator=gen, device="cuda").mul_(a).to(dtype) for a in (loud, 1.0))
    return dict(x, k=k, v=v, q=torch.randn(n * c, H, D, generator=gen, device="cuda").to(dtype), more=_int(own_part),
                pages=sum(_pages(h) for h in held) + sum(_pages(h % PAGE + m) for h, of_one in zip(held, more) for m in of_one))


def prepare(case, seed):
    x = inputs(case, seed)
    if case["op"] in ("sample", "logprobs"):
        return dict(x, case=case)
    n, c = case["sources"], case["copies"]
    kind = dict(n_head=case.get("heads", case["kv_heads"]), n_kv_head=case["kv_heads"], head_size=case["head_size"], group=case["group"], pages=x["pages"], requests=n + n * c,
                max_length=x["max_length"])
    state = dict(case=case, rows=x["rows"], into=x["into"], none=torch.zeros_like(x["into"]), cut=x.get("cut"))
    if case["op"] == "fork":
        if own:
            cache = state["cache"] = _package()[0](case["layers"], **kind, device="cuda", share=True)
            cache.free.copy_(x["order"])
            cache.blocks.copy_(x["blocks"])
            cache.plan(torch.arange(n, dtype=torch.int32, device="cuda"), x["held"], int(x["held"].sum()))
        else:
            state["s"] = _with_sources(case, x, n + n * c)
        return state
    state["q"] = x["q"]
    if own:
        # the prompts' keys and values, their copies, and the copies' own tokens, of which the last ones are the step's
        cache = state["cache"] = _package()[0](1, dtype=DTYPES[case["dtype"]], **kind, device="cuda", share=True)
        first, more = int(x["held"].sum()), x["more"]
        filled = cache.plan(torch.arange(n, dtype=torch.int32, device="cuda"), x["held"], first)
        cache.append(0, filled, None, x["k"][:first], x["v"][:first])
        cache.fork(x["rows"], x["into"])
        filled = cache.plan(x["into"], more, int(more.sum()))
        cache.append(0, filled, None, x["k"][first:], x["v"][first:])
        cache.truncate(x["into"], x["held"].repeat_interleave(c) + more - 1)         # the step's tokens again: their slots hold what they held
        state["plan"] = cache.plan(x["into"], torch.ones_like(more), n * c, max_count=1)
        return state
    state["s"] = _paged(case, x)
    return state


def _with_sources(case, x, requests):
    """A pool whose first requests hold the sources, given out from the end of the stack."""
    P = _pages(x["max_length"])
    pages = (x["held"].long() + PAGE - 1) // PAGE
    cum = pages.cumsum(0)
    page = torch.arange(P, device="cuda")
    at = x["pages"] - 1 - ((cum - pages)[:, None] + page)
    table = torch.full((requests, P), -1, dtype=torch.int32, device="cuda")
    table[:pages.numel()] = torch.where(page < pages[:, None], x["order"][at.clamp(min=0)], -1)
    lengths = torch.zeros(requests, dtype=torch.int32, device="cuda")
    lengths[:pages.numel()] = x["held"]
    return dict(table=table, lengths=lengths, free=x["order"].clone(), n_free=(x["pages"] - cum[-1]).int(), shared=torch.zeros(x["pages"], dtype=torch.int32, device="cuda"),
                blocks=x["blocks"])


def _segments(counts):
    """For every token of the sequences its sequence and its place in it."""
    seq = torch.repeat_interleave(torch.arange(counts.numel(), device=counts.device), counts)
    return seq, torch.arange(seq.numel(), device=counts.device) - (counts.cumsum(0) - counts)[seq]


def _quantized(x, group):
    g = x.float().unflatten(-1, (-1, group))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s = ((hi - lo) * torch.tensor(1 / 15, device=x.device)).to(x.dtype).float()
    c = torch.where(s > 0, torch.round((g - lo) / torch.where(s > 0, s, 1)).clamp(0, 15), 0)
    return c.to(torch.uint8).flatten(-2), s.squeeze(-1).to(x.dtype), lo.squeeze(-1).to(x.dtype)


def _paged(case, x):
    """The copies' tables over shared and own pages, and the pages: codes, scales and lowest values."""
    c, P = case["copies"], _pages(x["max_length"])
    held, more = x["held"].long(), x["more"].long()
    mine = held.repeat_interleave(c)                                         # tokens that a copy has from its source
    whole, ends = mine // PAGE, mine + more
    from_source = (held + PAGE - 1) // PAGE
    at_source = (from_source.cumsum(0) - from_source).repeat_interleave(c)
    own_pages = (ends + PAGE - 1) // PAGE - whole
    at_own = from_source.sum() + own_pages.cumsum(0) - own_pages
    page = torch.arange(P, device="cuda")
    table = torch.where(page < whole[:, None], at_source[:, None] + page, torch.where(page < whole[:, None] + own_pages[:, None], at_own[:, None] + page - whole[:, None], -1))
    seq, at = _segments(held)                                                # the sources' tokens, then the copies' own ones
    pos = at
    slots = [(from_source.cumsum(0) - from_source)[seq] * PAGE + pos]
    seq, at = _segments(more)
    pos = mine[seq] + at
    slots.append((at_own[seq] + pos // PAGE - whole[seq]) * PAGE + pos % PAGE)
    # a last page that is not full is the copies' own, with what the source has in it
    seq, at = _segments(mine % PAGE)
    to = at_own[seq] * PAGE + at
    was = (at_source[seq] + whole[seq]) * PAGE + at
    s = dict(q=x["q"], table=table.int(), lengths=ends.int(), longest=x["max_length"])
    K, D, dtype = case["kv_heads"], case["head_size"], x["q"].dtype
    for name in "kv":
        s[name] = (torch.zeros((x["pages"], PAGE, K, D), dtype=torch.uint8, device="cuda"),
                   *(torch.zeros((x["pages"], PAGE, K, D // case["group"]), dtype=dtype, device="cuda") for _ in range(2)))
        for a, what in zip(s[name], _quantized(x[name], case["group"])):
            a.flatten(0, 1)[torch.cat(slots)] = what
            a.flatten(0, 1)[to] = a.flatten(0, 1)[was]
    return s


# ---------------------------------------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if case["op"] == "sample":
        settings = {n: state[n] for n in ("temperature", "top_k", "top_p", "min_p")}
        if own:
            return _package()[1](state["logits"], state["u"], **settings)
        return plain_sample(state["logits"], state["u"], **settings)
    if case["op"] == "logprobs":
        if own:
            return _package()[2](state["logits"], state["tokens"], temperature=state["temperature"])
        return plain_logprobs(state["logits"], state["tokens"], state["temperature"])
    if case["op"] == "attend":
        if own:
            return state["cache"].attend(0, state["plan"], state["q"])
        return plain_attend(state["s"])
    # the copies of the pass before end first
    out = {}
    if own:
        cache = state["cache"]
        cache.truncate(state["into"], state["none"])
        out["status"] = cache.fork(state["rows"], state["into"])
        if state["cut"] is not None:
            out["cut"] = cache.truncate(state["into"], state["cut"])
        return dict(out, table=cache.table, lengths=cache.lengths, n_free=cache.n_free, blocks=cache.blocks)
    s = state["s"]
    plain_truncate(s, state["into"], state["none"])
    out["status"] = plain_fork(s, state["rows"], state["into"])
    if state["cut"] is not None:
        out["cut"] = plain_truncate(s, state["into"], state["cut"])
    return dict(out, table=s["table"], lengths=s["lengths"], n_free=s["n_free"].reshape(1), blocks=s["blocks"])


def work(case):
    if case["op"] in ("sample", "logprobs"):
        R, V = case["rows"], case["vocab"]
        size = 4 if case["dtype"] == "fp32" else 2
        # every logit read once, with its difference, exponential and sum
        return {"bytes": R * V * size + R * (12 if case["op"] == "logprobs" else 28), "flops": 4 * R * V}
    held, more = lengths_of(case)
    n, c, K, D = case["sources"], case["copies"], case["kv_heads"], case["head_size"]
    if case["op"] == "fork":
        page = case["layers"] * K * page_bytes(case)
        copied = sum(1 for h in held if h % PAGE) if not case["rewind"] else n
        new = min(copied * c, _pool(case) - sum(_pages(h) for h in held))
        # pages that are copied, each read once; the table's entries
        return {"bytes": (copied + new) * page + 4 * c * sum(_pages(h) for h in held) * 2, "flops": 0}
    row = 2 * K * (D // 2 + D // case["group"] * 4)                          # a token's codes, scales and lowest values
    kept = sum(h // PAGE * PAGE for h in held) + sum(h % PAGE + m for h, of_one in zip(held, more) for m in of_one)
    seen = sum(h + m for h, of_one in zip(held, more) for m in of_one)
    return {"bytes": kept * row + 2 * n * c * case["heads"] * D * 2, "flops": 4 * seen * case["heads"] * D}


# ---------------------------------------------------------------------------------------------------------------- the same in 64 bits
def _held_as(x, group, dtype):
    """The values that the cache holds for ``x``: the definition, number by number in 64 bits, scales and lowest values rounded to the cache's type."""
    x = x.double()
    parts = []
    for a in range(0, x.shape[-1], group):
        g = x[..., a:a + group]
        lo = g.min(-1, keepdim=True).values
        s = ((g.max(-1, keepdim=True).values - lo) / 15).to(dtype).double()
        c = ((g - lo) / s).round().clamp(0, 15).nan_to_num(0.0)
        parts.append(c * s + lo)
    return torch.cat(parts, -1)


def exact(case, seed):
    if case["op"] in ("fork", "sample"):                                     # whole numbers
        return None
    x = inputs(case, seed)
    if case["op"] == "logprobs":
        out = [torch.log_softmax(row.double() / x["temperature"], -1)[t] for row, t in zip(x["logits"], x["tokens"])]
        return torch.stack(out)
    held, more = lengths_of(case)
    H, K, D = case["heads"], case["kv_heads"], case["head_size"]
    k, v = (_held_as(x[name], case["group"], x["q"].dtype) for name in "kv")
    y = torch.empty(x["q"].shape, dtype=torch.float64, device="cuda")
    source, part, at = 0, sum(held), 0
    for h, of_one in zip(held, more):
        for m in of_one:
            keys, values = (torch.cat([t[source:source + h], t[part:part + m]]).repeat_interleave(H // K, 1) for t in (k, v))
            weights = (torch.einsum("hd,jhd->hj", x["q"][at].double(), keys) / math.sqrt(D)).softmax(-1)
            y[at] = torch.einsum("hj,jhd->hd", weights, values)
            part, at = part + m, at + 1
        source += h
    return y
