"""What the operators of the paged 4-bit key/value cache are measured on: their plain forms, and the framework's kernels on the same inputs.

The operators, in the order of a serving step:

``plan``    pages and slots of a step, on the GPU, from the lengths that requests hold and the tokens that they bring: a request's tokens go to pages
            of 64 slots that a stack of free ones gives out in the order of the requests; ``truncate`` gives them back
``append``  queries and keys turned by their positions, keys and values rounded to 4 bits by groups of a head's dimensions and written to their slots
``attend``  softmax attention of a step's tokens over what the cache holds of their requests, from one token to whole prompts

A group of values x is held as codes: lo = min(x), s = round_T((max(x) - lo) * (1/15)), c = clamp(rint((x - lo) / s), 0, 15), and stands for c * s + lo.
"""
import math
import random
import sys

import numpy as np
import torch

own = False

PAGE = 64
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # 64 requests in the middle of their answers, one token each, some of them idle
        dict(name="plan_step", op="plan", requests=64, longest=4096, new=1, others="same", pool=1.0, mix=1),
        # a burst of prompts for a pool that does not hold them all
        dict(name="plan_prompts", op="plan", requests=200, longest=5000, new=1900, others="spread", pool=0.9, mix=2),
        # one layer's tokens of a step of 64 requests (heads of the 7B configuration)
        dict(name="append_step", op="append", requests=64, longest=4096, new=1, others="same", heads=32, kv_heads=32, head_size=128, group=64, dtype="bf16", mix=3),
        # prompts of one layer, odd lengths, fewer key heads
        dict(name="append_prompts", op="append", requests=9, longest=1501, new=1437, others="spread", heads=40, kv_heads=8, head_size=128, group=32, dtype="fp16", mix=4),
        # one user of the smallest configuration: latency
        dict(name="step_small", op="attend", requests=1, longest=300, new=1, others="same", heads=8, kv_heads=8, head_size=64, group=64, dtype="bf16", mix=5),
        # one user of the 7B configuration at its block size
        dict(name="step_7b", op="attend", requests=1, longest=2048, new=1, others="same", heads=32, kv_heads=32, head_size=128, group=128, dtype="bf16", mix=6),
        # a served batch of unequal requests
        dict(name="step_batch", op="attend", requests=64, longest=4096, new=1, others="same", heads=32, kv_heads=32, head_size=128, group=64, dtype="bf16", mix=7),
        # one long document, eight key heads
        dict(name="step_long", op="attend", requests=1, longest=130001, new=1, others="same", heads=32, kv_heads=8, head_size=128, group=32, dtype="fp16", mix=8),
        # drafts of four tokens to be checked
        dict(name="drafts", op="attend", requests=12, longest=3001, new=4, others="same", heads=40, kv_heads=40, head_size=128, group=128, dtype="bf16", mix=9),
        # a prompt of the 7B configuration's block size
        dict(name="prompt_7b", op="attend", requests=1, longest=2048, new=2048, others="same", heads=32, kv_heads=32, head_size=128, group=64, dtype="bf16", mix=10),
        # a part of a long prompt beside requests that bring one token
        dict(name="mixed", op="attend", requests=10, longest=5000, new=700, others="one", heads=32, kv_heads=8, head_size=128, group=64, dtype="bf16", mix=11),
        # prompts of odd lengths of the smallest head size among the configurations
        dict(name="prompts_64", op="attend", requests=5, longest=4000, new=3333, others="spread", heads=8, kv_heads=8, head_size=64, group=32, dtype="fp16", mix=12),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["plan", "append", "append", "attend", "attend", "attend", "attend"])
    case = dict(op=op, mix=rng.randrange(1 << 30))
    if op == "plan":
        new = rng.choice([1, 1, _spread(rng, 2, 4096)])
        case.update(requests=_spread(rng, 1, 700), longest=new + _spread(rng, 1, 16384), new=new, others=rng.choice(["same", "one", "spread"]), pool=rng.choice([0.8, 1.0, 1.0]))
        if case["others"] == "same" and new > 64:
            case["others"] = "spread"
        return case
    kv = rng.choice([1, 2, 4, 8, 10, 32])
    heads = kv * rng.choice([1, 1, 1, 4] if kv > 4 else [1, 2, 4, 8])
    size = rng.choice([32, 64, 128, 128])
    case.update(heads=heads, kv_heads=kv, head_size=size, group=rng.choice([g for g in (32, 64, 128) if g <= size]), dtype=rng.choice(["bf16", "bf16", "fp16"]))
    if op == "append":
        new = rng.choice([1, _spread(rng, 2, 2048)])
        case.update(requests=_spread(rng, 1, 100 if new < 64 else 8), longest=new + _spread(rng, 1, 4096), new=new, others=rng.choice(["same", "spread"]))
        return case
    kind = rng.choice(["step", "step", "drafts", "prompt", "mixed"])
    if kind == "step":
        requests = _spread(rng, 1, 100)
        case.update(requests=requests, longest=_spread(rng, 1, min(100000, 400000 // (requests * max(1, kv // 8)))), new=1, others="same")
    elif kind == "drafts":
        new = rng.randrange(2, 20)
        case.update(requests=_spread(rng, 1, 16), longest=new + _spread(rng, 1, 4000), new=new, others=rng.choice(["same", "spread"]))
    elif kind == "prompt":
        new = _spread(rng, 20, 2000)
        case.update(requests=_spread(rng, 1, 4), longest=new + rng.choice([0, 0, _spread(rng, 1, 2000)]), new=new, others="spread")
    else:
        new = _spread(rng, 20, 1000)
        case.update(requests=_spread(rng, 2, 16), longest=new + _spread(rng, 1, 3000), new=new, others="one")
    # scores and 32-bit keys of the plain form, padded to the longest request, no more than those of the largest listed cases
    while case["requests"] > 1 and case["requests"] * case["longest"] * max(heads * case["new"], kv * size) > 1_000_000_000:
        case["requests"] //= 2
    return case


def ragged(case):
    """What the requests hold before the step and how many tokens each brings; the first one is the longest."""
    rng = random.Random(case["mix"])
    n, longest, new = case["requests"], case["longest"], case["new"]
    held, counts = [longest - new], [new]
    for i in range(1, n):
        c = {"same": new, "one": 1, "spread": rng.randrange(1, new + 1)}[case["others"]]
        if n >= 8 and rng.random() < 1 / 16:
            c = 0                                   # a request that waits
        held.append(rng.randrange(0, longest - c + 1))
        counts.append(c)
    return held, counts


def _pages(n):
    return -(-n // PAGE)


# ---------------------------------------------------------------------------------------------------------------- the plain forms
def _segments(ends, total):
    """For each of ``total`` places the segment that holds it (empty ones are passed over); ``ends`` are the places behind the segments."""
    at = torch.arange(total, device=ends.device)
    return torch.searchsorted(ends.contiguous(), at, right=True), at


def plain_truncate(s, rows, keep):
    """Cuts requests to ``keep`` tokens: pages behind go back to the stack, so that the next plan takes them in the same order."""
    P = s["table"].shape[1]
    old = s["lengths"][rows.long()].long()
    keep = torch.minimum(keep.long(), old)
    first, last = (keep + PAGE - 1) // PAGE, (old + PAGE - 1) // PAGE
    n = last - first
    cum = n.cumsum(0)
    page = torch.arange(P, device=rows.device)
    table = s["table"][rows.long()]
    out = (page >= first[:, None]) & (page < last[:, None])
    order = (cum - n)[:, None] + page - first[:, None]                       # the how-manieth page given back
    at = s["n_free"].long() + cum[-1] - 1 - order
    s["free"] = _scatter_some(s["free"], at, table, out)
    s["table"] = s["table"].index_copy(0, rows.long(), torch.where(out, -1, table))
    s["lengths"] = s["lengths"].index_copy(0, rows.long(), keep.int())
    s["n_free"] = (s["n_free"] + cum[-1]).int()


def _scatter_some(to, at, what, where):
    """``to`` with what[i] at at[i] for the places that ``where`` names; the others go to a place behind the end."""
    more = torch.cat([to, to.new_zeros(1)])
    return more.scatter(0, torch.where(where, at, to.numel()).reshape(-1), torch.where(where, what, 0).reshape(-1).to(to.dtype))[:-1]


def plain_plan(s, rows, counts, tokens):
    n = counts.long().clamp(min=0)
    cum = n.cumsum(0)
    starts = torch.cat([cum.new_zeros(1), cum])
    old = s["lengths"][rows.long()].long()
    P = s["table"].shape[1]
    status = torch.zeros_like(rows)
    status = torch.where(old + n > s["max_length"], 2, status)
    status = torch.where(cum > tokens, 4, status)
    first, last = (old + PAGE - 1) // PAGE, (old + n + PAGE - 1) // PAGE
    need = torch.where(status == 0, last - first, 0)
    used = need.cumsum(0)
    status = torch.where((status == 0) & (need > 0) & (used > s["n_free"]), 1, status)
    ok = (status == 0) & (n > 0)
    page = torch.arange(P, device=rows.device)
    at = s["n_free"].long() - 1 - ((used - need)[:, None] + page - first[:, None])
    mine = ok[:, None] & (page >= first[:, None]) & (page < last[:, None])
    table = torch.where(mine, s["free"][at.clamp(0, s["free"].numel() - 1)], s["table"][rows.long()])
    s["table"] = s["table"].index_copy(0, rows.long(), table)
    s["lengths"] = s["lengths"].index_copy(0, rows.long(), torch.where(ok, old + n, old).int())
    s["n_free"] = (s["n_free"] - torch.where(ok, need, 0).sum()).int()
    seq, t = _segments(cum, tokens)
    there = t < cum[-1]
    seq = torch.where(there, seq, 0)
    there = there & ok[seq]
    pos = old[seq] + t - starts[seq]
    slot = table[seq, (pos // PAGE).clamp(0, P - 1)].long() * PAGE + pos % PAGE
    none = torch.full_like(pos, -1)
    return dict(starts=starts.clamp(max=tokens).int(), ends=torch.where(status == 0, s["lengths"][rows.long()], 0), status=status.int(),
                positions=torch.where(there, pos, none).int(), slots=torch.where(there, slot, none).int())


def plain_quantize(x, group):
    """Codes, scales and lowest values of ``x [..., D]`` by groups along its last dimension."""
    g = x.float().unflatten(-1, (-1, group))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s = ((hi - lo) * torch.tensor(1 / 15, device=x.device)).to(x.dtype).float()
    c = torch.where(s > 0, torch.round((g - lo) / torch.where(s > 0, s, 1)).clamp(0, 15), 0)
    return c.to(torch.uint8).flatten(-2), s.squeeze(-1).to(x.dtype), lo.squeeze(-1).to(x.dtype)


def plain_values(c, s, lo):
    g = c.float().unflatten(-1, (s.shape[-1], -1))
    return (g * s.float()[..., None] + lo.float()[..., None]).flatten(-2)


def plain_turn(x, positions, rope):
    cs = rope[positions.long().clamp(min=0)][:, None]                        # [T, 1, D/2, 2]
    p = x.float().unflatten(-1, (-1, 2))
    a, b = p[..., 0], p[..., 1]
    return torch.stack((a * cs[..., 0] - b * cs[..., 1], b * cs[..., 0] + a * cs[..., 1]), -1).flatten(-2).to(x.dtype)


def plain_append(s, q, k, v):
    q, k = plain_turn(q, s["positions"], s["rope"]), plain_turn(k, s["positions"], s["rope"])
    page, at = s["slots"].long() // PAGE, s["slots"].long() % PAGE
    for_k, for_v = plain_quantize(k, s["group"]), plain_quantize(v, s["group"])
    s["k"][0][page, at], s["k"][1][page, at], s["k"][2][page, at] = for_k
    s["v"][0][page, at], s["v"][1][page, at], s["v"][2][page, at] = for_v
    read = [plain_values(*(a[page, at] for a in s[x])).to(q.dtype) for x in "kv"]
    return {"q": q, "k": read[0], "v": read[1]}


def plain_attend(s):
    """All requests at once, padded to the longest: keys and values of 32 bits, scores, their softmax and the weighted sum."""
    q, starts, ends, counts, rows = s["q"], s["starts"], s["ends"], s["counts"], s["rows"]
    T, H, D = q.shape
    longest, new, G = s["longest"], s["new"], H // s["k"][0].shape[2]
    j = torch.arange(longest, device=q.device)
    page, at = s["table"][rows.long()][:, j // PAGE].long().clamp(min=0), j % PAGE
    k, v = (plain_values(*(a[page, at] for a in s[x])) for x in "kv")        # [B, L, Hkv, D]
    held = (j < ends[:, None])[:, :, None, None]
    v = torch.where(held, v, 0)
    r = torch.arange(new, device=q.device)
    t = (starts[:-1, None] + r).clamp(max=T - 1)
    mine = q.float()[t] * D ** -0.5                                          # [B, n, H, D]
    k, v = k.permute(0, 2, 3, 1), v.permute(0, 2, 1, 3)                      # [B, Hkv, D, L], [B, Hkv, L, D]
    mine = mine.unflatten(2, (-1, G)).permute(0, 2, 1, 3, 4).flatten(2, 3)   # [B, Hkv, n * G, D]
    scores = torch.matmul(mine, k)
    pos = (ends - counts)[:, None] + r                                       # [B, n]
    seen = (j[None, None, :] <= pos[:, :, None]) & (j < ends[:, None])[:, None, :]
    scores = scores.masked_fill(~seen.repeat_interleave(G, 1)[:, None], -math.inf)
    w = torch.exp(scores - scores.amax(-1, keepdim=True))
    y = torch.matmul(w, v) / w.sum(-1, keepdim=True)
    y = y.unflatten(2, (new, G)).permute(0, 2, 1, 3, 4).flatten(2, 3)        # [B, n, H, D]
    seq, t = _segments(starts[1:], T)
    return y[seq, t - starts[seq]].to(q.dtype)


# ---------------------------------------------------------------------------------------------------------------- inputs
def _package():
    if "lit-llama-ja_b200" not in sys.path:
        sys.path.insert(0, "lit-llama-ja_b200")
    from lit_llama.paged_cache import PagedCache4

    return PagedCache4


def _numbers(shape, dtype, gen, spread):
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    return x.mul_(spread).to(dtype)


def _rope(n, D):
    theta = 1.0 / 10000 ** (torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D)
    angle = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * theta
    return torch.stack((angle.cos(), angle.sin()), -1).float().contiguous()


def inputs(case, seed):
    """Everything that both sides and the 64-bit form start from."""
    held, counts = ragged(case)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n, T = len(held), sum(counts)
    need = sum(_pages(h + c) for h, c in zip(held, counts))
    have = sum(_pages(h) for h in held)
    pages = max(1, have + math.ceil((need - have) * case.get("pool", 1.0)))
    x = dict(held=torch.tensor(held, dtype=torch.int32, device="cuda"), counts=torch.tensor(counts, dtype=torch.int32, device="cuda"), tokens=T, pages=pages,
             rows=torch.randperm(n, generator=gen, device="cuda").int(), order=torch.randperm(pages, generator=gen, device="cuda").int(), max_length=case["longest"])
    if case["op"] == "plan":
        return x
    dtype, H, K, D = DTYPES[case["dtype"]], case["heads"], case["kv_heads"], case["head_size"]
    # some dimensions of a head's keys are much larger than the others
    loud = torch.where(torch.rand(K, D, generator=gen, device="cuda") < 0.03, 6.0, 1.0)
    x["q"] = _numbers((T, H, D), dtype, gen, 1.0)
    rows = T if case["op"] == "append" else T + sum(held)
    x["k"], x["v"] = _numbers((rows, K, D), dtype, gen, loud), _numbers((rows, K, D), dtype, gen, 1.0)
    return x


def prepare(case, seed):
    x = inputs(case, seed)
    n, longest, op = case["requests"], case["longest"], case["op"]
    state = dict(x, case=case)
    if own:
        Cache = _package()
        kind = dict(n_layer=1, n_head=1, head_size=32, group=32) if op == "plan" else dict(
            n_layer=1, n_head=case["heads"], n_kv_head=case["kv_heads"], head_size=case["head_size"], group=case["group"], dtype=DTYPES[case["dtype"]])
        cache = state["cache"] = Cache(**kind, pages=x["pages"], requests=n, max_length=longest, device="cuda")
        cache.free.copy_(x["order"])
    state["s"] = s = dict(table=torch.full((n, _pages(longest)), -1, dtype=torch.int32, device="cuda"), lengths=torch.zeros(n, dtype=torch.int32, device="cuda"),
                          free=x["order"].clone(), n_free=torch.tensor(x["pages"], dtype=torch.int32, device="cuda"), pages=x["pages"], max_length=longest)
    if op != "attend":                                                       # the requests as they are before the step
        before = int(x["held"].sum())
        if own:
            if before:
                cache.plan(x["rows"], x["held"], before)
        else:
            plain_plan(s, x["rows"], x["held"], before)
        if op == "plan":
            return state
    else:                                                                    # all that they hold, the step's tokens too, was brought at once
        x["counts"], step = x["held"] + x["counts"], x["counts"]
    if op == "append":
        state["rope"] = _rope(longest, case["head_size"])
        if own:
            state["plan"] = cache.plan(x["rows"], x["counts"], x["tokens"], max_count=case["new"])
        else:
            s.update(plain_plan(s, x["rows"], x["counts"], x["tokens"]), rope=state["rope"], group=case["group"])
            s.update(_plain_cache(case, x))
        return state
    total = int(x["k"].shape[0])
    if own:
        filled = cache.plan(x["rows"], x["counts"], total)
        cache.append(0, filled, None, x["k"], x["v"])
        cache.truncate(x["rows"], x["held"])                                 # the step's tokens again: their slots hold what they held
        state["plan"] = cache.plan(x["rows"], step, x["tokens"], max_count=case["new"])
    else:
        plan = plain_plan(s, x["rows"], x["counts"], total)
        s.update(_plain_cache(case, x))
        page, at = plan["slots"].long() // PAGE, plan["slots"].long() % PAGE
        for name in "kv":
            for to, what in zip(s[name], plain_quantize(x[name], case["group"])):
                to[page, at] = what
        starts = torch.cat([step.new_zeros(1), step.cumsum(0).int()])
        s.update(q=x["q"], rows=x["rows"], counts=step, starts=starts, ends=plan["ends"], longest=longest, new=case["new"])
    for name in ("k", "v"):
        state.pop(name)
    return state


def _plain_cache(case, x):
    K, D, dtype = case["kv_heads"], case["head_size"], DTYPES[case["dtype"]]
    make = lambda: (torch.zeros((x["pages"], PAGE, K, D), dtype=torch.uint8, device="cuda"),  # noqa: E731
                    *(torch.zeros((x["pages"], PAGE, K, D // case["group"]), dtype=dtype, device="cuda") for _ in range(2)))
    return dict(k=make(), v=make())


# ---------------------------------------------------------------------------------------------------------------- one pass
def run(state):
    case, s = state["case"], state["s"]
    if case["op"] == "plan":
        # what the pass before has given out goes back first: a step's rejected tokens
        if own:
            cache = state["cache"]
            cache.truncate(state["rows"], state["held"])
            p = cache.plan(state["rows"], state["counts"], state["tokens"], max_count=case["new"])
            return {"starts": p.starts, "ends": p.ends, "status": p.status, "positions": p.positions, "slots": p.slots, "table": cache.table, "lengths": cache.lengths,
                    "n_free": cache.n_free}
        plain_truncate(s, state["rows"], state["held"])
        p = plain_plan(s, state["rows"], state["counts"], state["tokens"])
        return {**p, "table": s["table"], "lengths": s["lengths"], "n_free": s["n_free"].reshape(1)}
    if case["op"] == "append":
        if own:
            cache, plan = state["cache"], state["plan"]
            q = cache.append(0, plan, state["q"], state["k"], state["v"], rope=state["rope"])
            k, v = cache.read(0, plan.slots)
            return {"q": q, "k": k, "v": v}
        return plain_append(s, state["q"], state["k"], state["v"])
    if own:
        return state["cache"].attend(0, state["plan"], state["q"])
    return plain_attend(s)


def work(case):
    held, counts = ragged(case)
    T = sum(counts)
    if case["op"] == "plan":
        # lengths, rows and counts, the plan by request and by token, and the table's entries of new pages
        new = sum(_pages(h + c) - _pages(h) for h, c in zip(held, counts))
        return {"bytes": 4 * (7 * len(held) + 2 * T + 4 * new), "flops": 0}
    H, K, D = case["heads"], case["kv_heads"], case["head_size"]
    row = 2 * K * (D // 2 + D // case["group"] * 4)                          # a token's codes, scales and lowest values
    if case["op"] == "append":
        # queries, keys and values read, queries, codes and the values that they stand for written
        return {"bytes": T * (2 * H * D * 2 + 2 * K * D * 2 * 2 + 2 * row), "flops": T * (H + K) * D * 3 + T * K * D * 2 * 4}
    seen = sum(c * h + c * (c + 1) // 2 for h, c in zip(held, counts))
    return {"bytes": sum(h + c for h, c in zip(held, counts) if c) * row + 2 * T * H * D * 2, "flops": 4 * seen * H * D}


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
    if case["op"] == "plan":
        return None
    x = inputs(case, seed)
    held, counts = ragged(case)
    dtype, H, K, D = DTYPES[case["dtype"]], case["heads"], case["kv_heads"], case["head_size"]
    if case["op"] == "append":
        pos = torch.tensor(np.concatenate([np.arange(h, h + c) for h, c in zip(held, counts)]), device="cuda", dtype=torch.float64)
        # the table's numbers are of 32 bits
        angle = pos[:, None] / 10000 ** (torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D)
        turn = torch.polar(torch.ones_like(angle), angle)
        turn = torch.complex(turn.real.float().double(), turn.imag.float().double())[:, None]
        q, k = (torch.view_as_real(torch.view_as_complex(x[n].double().reshape(*x[n].shape[:2], D // 2, 2)) * turn).flatten(-2) for n in ("q", "k"))
        return {"q": q, "k": _held_as(k.to(dtype), case["group"], dtype), "v": _held_as(x["v"], case["group"], dtype)}
    if 4 * sum(c * (h + c) for h, c in zip(held, counts)) * H * D > 4e12:
        return None
    out, at, first = [], 0, 0
    for h, c in zip(held, counts):
        k, v = (_held_as(x[n][at:at + h + c], case["group"], dtype) for n in "kv")
        mask = torch.arange(h + c, device="cuda")[None] > torch.arange(h, h + c, device="cuda")[:, None]
        y = torch.empty(c, H, D, dtype=torch.float64, device="cuda")
        for head in range(H if c else 0):
            score = x["q"][first:first + c, head].double() @ k[:, head * K // H].T / math.sqrt(D)
            y[:, head] = score.masked_fill(mask, -math.inf).softmax(-1) @ v[:, head * K // H]
        out.append(y)
        at, first = at + h + c, first + c
    return torch.cat(out)
