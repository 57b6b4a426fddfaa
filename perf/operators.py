"""Cases for the paged key/value cache a retrieval user keeps beside the index: append, attend and evict.

A retrieved passage's keys and values sit in pages of a cache; a page table per sequence (made from the search's ids)
says which pages a sequence reads. `append` writes new tokens behind a sequence, `attend` is the attention of its new
tokens (one, a few, or a chunk) over all its slots, with the attention weight that each slot gathers on request, and
`evict` cuts a sequence back to the slots that gathered most, into fresh pages.

run() computes either the plain form (elementary torch operations in 32 bits, padded to the longest sequence) or, with
`own`, the calls of veckern_b200.PagedCache.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    """Types, head counts, page sizes and both page layouts ("slot": [pages, slot, head, dim]; "head": [pages, head,
    slot, dim]) go round the cases; `length` is the longest sequence, the others of a ragged batch are spread below it."""
    return [
        # one decoding step's write for a few streams: latency
        dict(name="append step", op="append", type="bf16", batch=13, tokens=1, length=2000, kv_heads=8, dim=128, page=16,
             layout="slot", ragged=True),
        # prompts of several requests written behind the passages that were retrieved for them
        dict(name="append prompts", op="append", type="f16", batch=9, tokens=2011, length=6007, kv_heads=8, dim=128,
             page=64, layout="head", ragged=True),
        # one request's single token over a short cache: latency
        dict(name="attend step, one", op="attend", type="bf16", batch=1, tokens=1, length=1000, heads=32, kv_heads=8,
             dim=128, page=16, layout="slot", causal=True, scores=False, ragged=False, shared=0),
        # a serving batch's step over ragged caches
        dict(name="attend step, batch", op="attend", type="bf16", batch=32, tokens=1, length=8192, heads=32, kv_heads=8,
             dim=128, page=64, layout="slot", causal=True, scores=False, ragged=True, shared=0),
        # the same with the weights that eviction goes by, long caches
        dict(name="attend step, weights", op="attend", type="f16", batch=4, tokens=1, length=50021, heads=32, kv_heads=8,
             dim=128, page=32, layout="head", causal=True, scores=True, ragged=True, shared=0),
        # a few drafted tokens checked at once
        dict(name="attend drafted", op="attend", type="bf16", batch=8, tokens=5, length=4001, heads=24, kv_heads=8,
             dim=64, page=16, layout="slot", causal=True, scores=False, ragged=True, shared=0),
        # questions that read the retrieved passages' pages, which several of them share, without a causal mask
        dict(name="attend passages", op="attend", type="f16", batch=16, tokens=77, length=2560, heads=16, kv_heads=4,
             dim=128, page=128, layout="head", causal=False, scores=False, ragged=True, shared=8),
        # a chunk of a long prompt
        dict(name="attend prompt", op="attend", type="bf16", batch=1, tokens=4096, length=16384, heads=32, kv_heads=8,
             dim=128, page=64, layout="slot", causal=True, scores=False, ragged=False, shared=0),
        # ragged chunks with weights, odd sizes
        dict(name="attend chunks, weights", op="attend", type="bf16", batch=3, tokens=1023, length=5003, heads=16,
             kv_heads=8, dim=80, page=32, layout="slot", causal=True, scores=True, ragged=True, shared=0),
        # one sequence that went a little over its budget
        dict(name="evict one", op="evict", type="bf16", batch=1, length=1087, kv_heads=8, dim=128, page=16, layout="slot",
             keep=1024, recent=64, ragged=False),
        # a batch cut back to half
        dict(name="evict batch", op="evict", type="f16", batch=16, length=8192, kv_heads=8, dim=128, page=64,
             layout="head", keep=4096, recent=512, ragged=True),
        # a long context cut to an eighth
        dict(name="evict long", op="evict", type="bf16", batch=1, length=131072, kv_heads=8, dim=128, page=64,
             layout="slot", keep=16384, recent=1024, ragged=False),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "evict"])
    case = dict(op=op, type=rng.choice(["bf16", "f16"]), kv_heads=rng.choice([1, 2, 4, 5, 8]),
                dim=rng.choice([64, 72, 80, 96, 112, 128, 128]), page=rng.choice([8, 16, 32, 64, 128, 256]),
                layout=rng.choice(["slot", "head"]), ragged=rng.random() < 0.7)
    if op == "append":
        batch = _log(rng, 1, 64)
        tokens = _log(rng, 1, max(1, 16000 // batch))
        case.update(batch=batch, tokens=tokens, length=tokens + _log(rng, 1, max(2, 60000 // batch)))
    elif op == "evict":
        batch = _log(rng, 1, 32)
        length = _log(rng, 16, min(131072, 131072 // batch))
        keep = _log(rng, 2, length)
        case.update(batch=batch, length=length, keep=keep, recent=rng.randrange(0, keep))
    else:
        kind = rng.choice(["step", "few", "chunk"])
        tokens = 1 if kind == "step" else _log(rng, 2, 12) if kind == "few" else _log(rng, 13, 4096)
        heads = case["kv_heads"] * rng.choice([1, 2, 3, 4, 8])
        batch = _log(rng, 1, 64 if kind != "chunk" else max(1, min(16, 8192 // tokens)))
        # slots of all sequences together: the cache stays under 2 GB, the plain form's products under 1.8 G values
        most = min(260000, 1_800_000_000 // (heads * tokens)) // batch
        length = _log(rng, max(2, min(tokens, most)), max(2, most))
        case.update(tokens=min(tokens, length), batch=batch, heads=heads, length=length, causal=rng.random() < 0.75,
                    scores=rng.random() < 0.4, shared=0)
    return case


def _lengths(case):
    """(length, new tokens) of each sequence: the first has the longest; a ragged batch goes down to about a third."""
    out = []
    for b in range(case["batch"]):
        n, t = case["length"], case.get("tokens", 0)
        if case["ragged"] and b:
            n = max(1, n - (n * 2 * b) // (3 * case["batch"]) - (b * 37) % 29)
            t = max(1, t - (t * 2 * b) // (3 * case["batch"]) - b % 2) if t > 1 else t
        out.append((n, min(t, n)))
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, page, g, d = TYPES[case["type"]], case["page"], case["kv_heads"], case["dim"]
    pairs = _lengths(case)
    need = [-(-n // page) for n, _ in pairs]
    fresh = [-(-min(n, case["keep"]) // page) for n, _ in pairs] if case["op"] == "evict" else []
    shared = min(case.get("shared", 0), min(need))
    pages = shared + sum(w - shared for w in need) + sum(fresh) + 3
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)

    def random(*size, scale=1.0):
        return (torch.randn(size, generator=gen, device="cuda") * scale).to(kind)

    def cached():  # keys and values: a common direction for each channel and noise, as projections give them
        shape = (pages, page, g, d) if case["layout"] == "slot" else (pages, g, page, d)
        x = random(*shape)
        x += random(d, scale=0.5)
        return x if case["layout"] == "slot" else x.transpose(1, 2)

    def tables(counts, first, common):
        t = torch.full((len(counts), max(counts)), -1, dtype=torch.int32, device="cuda")
        at = first
        for b, w in enumerate(counts):
            t[b, :common] = order[:common]
            t[b, common:w] = order[at:at + w - common]
            at += w - common
        return t, at

    state = dict(case=case, k=cached(), v=cached())
    state["table"], at = tables(need, shared, shared)
    state["lens"] = torch.tensor([n for n, _ in pairs], dtype=torch.int32, device="cuda")
    offsets = [0]
    for _, t in pairs:
        offsets.append(offsets[-1] + t)
    state["offsets"] = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    state["most"] = max(t for _, t in pairs)
    width = max(n for n, _ in pairs)
    if case["op"] == "append":
        both = random(offsets[-1], 2, g, d)  # the two projections of one product, side by side
        state["new_k"], state["new_v"] = both[:, 0], both[:, 1]
    elif case["op"] == "attend":
        state["q"] = random(offsets[-1], case["heads"], d, scale=2.0)
        state["scores"] = torch.rand((len(pairs), g, width), generator=gen, device="cuda") if case["scores"] else None
    else:
        state["new_table"], _ = tables(fresh, at, 0)
        # gathered weights: most slots little, a few much; later slots had less time
        w = torch.randn((len(pairs), g, width), generator=gen, device="cuda").mul_(2.0).exp_()
        state["scores"] = w * torch.linspace(1.0, 0.1, width, device="cuda")
        state["scores"][..., 5::7] = 0.0  # slots that nothing looked at: ties
    if own:
        from veckern_b200 import PagedCache

        state["cache"] = PagedCache(state["k"], state["v"])
    return state


def run(state):
    case = state["case"]
    if own:
        cache = state["cache"]
        if case["op"] == "append":
            cache.append(state["new_k"], state["new_v"], state["offsets"], state["table"], state["lens"])
            return {"k": state["k"], "v": state["v"]}
        if case["op"] == "attend":
            out, lse = cache.attend(state["q"], state["offsets"], state["table"], state["lens"], causal=case["causal"],
                                    scores=state["scores"], max_q=state["most"])
            return {"out": out, "lse": lse, "scores": state["scores"]}
        kept, new_lens, new_scores = cache.evict(state["table"], state["lens"], state["new_table"], case["keep"],
                                                 case["recent"], state["scores"])
        return {"kept": kept, "lens": new_lens, "scores": new_scores, "k": state["k"], "v": state["v"]}
    return {"append": _plain_append, "attend": _plain_attend, "evict": _plain_evict}[case["op"]](state)


def _plain_append(state):
    offsets, lens, table = state["offsets"].long(), state["lens"].long(), state["table"].long()
    page = state["case"]["page"]
    row = torch.arange(state["new_k"].shape[0], device="cuda")
    b = torch.searchsorted(offsets, row, right=True) - 1
    slot = lens[b] - offsets[b + 1] + row
    at = table[b, slot // page]
    state["k"][at, slot % page] = state["new_k"]
    state["v"][at, slot % page] = state["new_v"]
    return {"k": state["k"], "v": state["v"]}


def _plain_attend(state):
    case, q, offsets, lens = state["case"], state["q"], state["offsets"].long(), state["lens"].long()
    batch, group = lens.shape[0], case["heads"] // case["kv_heads"]
    count = offsets[1:] - offsets[:-1]
    table = state["table"].long().clamp(min=0)
    width = case["length"]
    keys = state["k"][table].flatten(1, 2)[:, :width].float()  # [batch, width, kv heads, dim]
    values = state["v"][table].flatten(1, 2)[:, :width].float()
    t = torch.arange(state["most"], device="cuda")
    j = torch.arange(width, device="cuda")
    rows = (offsets[:-1, None] + t).clamp(max=q.shape[0] - 1)
    used = t < count[:, None]
    x = q[rows].float().unflatten(2, (case["kv_heads"], group))  # [batch, t, kv heads, group, dim]
    seen = (j < lens[:, None])[:, None, :] & used[:, :, None]
    if case["causal"]:
        seen = seen & (j <= (lens - count)[:, None, None] + t[None, :, None])
    seen = seen[:, None, None]
    x = x.permute(0, 2, 3, 1, 4).flatten(2, 3) / math.sqrt(case["dim"])
    s = (x @ keys.permute(0, 2, 3, 1)).unflatten(2, (group, -1))  # [batch, kv heads, group, t, width]
    s.masked_fill_(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    s.sub_(top).exp_()
    total = s.sum(-1, keepdim=True)
    s.div_(torch.where(total == 0, 1.0, total))
    out = (s.flatten(2, 3) @ values.transpose(1, 2)).unflatten(2, (group, -1))
    lse = (top + total.log()).squeeze(-1)
    out = out.permute(0, 3, 1, 2, 4).flatten(2, 3)[used].to(q.dtype)
    lse = lse.permute(0, 3, 1, 2).flatten(2, 3)[used]
    if state["scores"] is not None:
        state["scores"] += s.sum((2, 3))
    return {"out": out, "lse": lse, "scores": state["scores"]}


def _plain_evict(state):
    case, scores = state["case"], state["scores"]
    lens = state["lens"].long()
    page, width = case["page"], scores.shape[2]
    new_lens = lens.clamp(max=case["keep"])
    recent = new_lens.clamp(max=case["recent"])
    j = torch.arange(width, device="cuda")
    rank = scores.masked_fill((j >= (lens - recent)[:, None])[:, None], math.inf)
    rank = rank.masked_fill((j >= lens[:, None])[:, None], -math.inf)
    first = rank.sort(dim=2, descending=True, stable=True).indices[:, :, :case["keep"]]
    i = torch.arange(first.shape[2], device="cuda")
    held = (i < new_lens[:, None])[:, None].expand(first.shape)
    slots = first.masked_fill(~held, width).sort(dim=2).values
    kept = torch.where(held, slots, -1).to(torch.int32)
    slots = torch.where(held, slots, 0)
    new_scores = torch.zeros_like(scores)
    new_scores[:, :, :i.shape[0]] = torch.where(held, scores.gather(2, slots), 0.0)
    b, h, at = held.nonzero(as_tuple=True)
    old = slots[b, h, at]
    old_page, new_page = state["table"].long()[b, old // page], state["new_table"].long()[b, at // page]
    state["k"][new_page, at % page, h] = state["k"][old_page, old % page, h]
    state["v"][new_page, at % page, h] = state["v"][old_page, old % page, h]
    if kept.shape[2] < case["keep"]:
        kept = torch.nn.functional.pad(kept, (0, case["keep"] - kept.shape[2]), value=-1)
    return {"kept": kept, "lens": new_lens.to(torch.int32), "scores": new_scores, "k": state["k"], "v": state["v"]}


def work(case):
    """Slots of shared pages are read once. An attended slot costs a product with its key and one with its value for
    every row that sees it."""
    pairs = _lengths(case)
    g, d = case["kv_heads"], case["dim"]
    slot = 2 * g * d * 2  # bytes of a slot's keys and values
    tables = 4 * sum(2 + -(-n // case["page"]) for n, _ in pairs)
    if case["op"] == "append":
        return {"bytes": 2 * slot * sum(t for _, t in pairs) + tables, "flops": 0}
    if case["op"] == "evict":
        held = sum(min(n, case["keep"]) for n, _ in pairs)
        width = max(n for n, _ in pairs)
        return {"bytes": 2 * slot * held + 4 * g * sum(n for n, _ in pairs) + 4 * g * len(pairs) * (case["keep"] + width)
                + tables, "flops": 0}
    shared = min(case["shared"] * case["page"], min(n for n, _ in pairs))
    slots = shared + sum(n - shared for n, _ in pairs)
    seen = 0
    for n, t in pairs:
        seen += n * t - t * (t - 1) // 2 if case["causal"] else n * t
    rows = sum(t for _, t in pairs) * case["heads"]
    moved = slot * slots + rows * (4 * d + 4) + tables
    if case["scores"]:
        moved += 8 * g * sum(n for n, _ in pairs)
    return {"bytes": moved, "flops": 4 * d * seen * case["heads"]}


def exact(case, seed):
    """attend in 64 bits, sequence by sequence and head by head; append and evict only move values."""
    if case["op"] != "attend":
        return None
    state = prepare(case, seed)
    pairs = _lengths(case)
    group = case["heads"] // case["kv_heads"]
    rows = sum(t for _, t in pairs)
    out = torch.zeros((rows, case["heads"], case["dim"]), dtype=torch.float64, device="cuda")
    lse = torch.full((rows, case["heads"]), -math.inf, dtype=torch.float64, device="cuda")
    scores = None if state["scores"] is None else state["scores"].double()
    at = 0
    for b, (n, t) in enumerate(pairs):
        slots = torch.arange(n, device="cuda")
        pages = state["table"][b].long()[slots // case["page"]]
        hidden = None
        if case["causal"]:
            hidden = slots[None, :] > (torch.arange(t, device="cuda") + (n - t))[:, None]
        for h in range(case["heads"]):
            key = state["k"][pages, slots % case["page"], h // group].double()
            value = state["v"][pages, slots % case["page"], h // group].double()
            s = state["q"][at:at + t, h].double() @ key.T * case["dim"] ** -0.5
            if hidden is not None:
                s[hidden] = -math.inf
            lse[at:at + t, h] = torch.logsumexp(s, 1)
            weights = torch.exp(s - lse[at:at + t, h, None])
            out[at:at + t, h] = weights @ value
            if scores is not None:
                scores[b, h // group, :n] += weights.sum(0)
        at += t
    return {"out": out, "lse": lse, "scores": scores}
