"""Search, read, forget: passages found by the PQ index are read by attention over their cached keys and values, and the
memory is cut back to what was looked at.

    python -m veckern_b200.examples.retrieval_memory

Every passage has 64 tokens, and its keys and values fill one page of a PagedCache, written once (here with random
projections of random token vectors in place of a model's layer). The index holds one vector per passage. For a batch of
questions:

  1. the index finds each question's 8 passages; their ids ARE the numbers of their pages, so the ids are the page table
  2. the question's tokens are written behind them, into pages of their own, and attend over passages and themselves;
     the weight that every slot gathers is kept
  3. every sequence is cut back to the 192 slots per head that gathered most (its own tokens stay), in pages of its own
  4. new tokens follow one at a time: append, attend
"""
from __future__ import annotations

import torch

from .. import PagedCache, PQSearcher, Tuning, data, device_result_split

PAGE, HEADS, KV_HEADS, DIM, WIDTH = 64, 16, 4, 64, 128


def run(passages: int = 4096, questions: int = 12, found: int = 8, asked: int = 40, keep: int = 192, steps: int = 6,
        seed: int = 0) -> dict:
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = torch.bfloat16

    def normal(*size):
        return torch.randn(size, generator=gen, device="cuda")

    # A passage's tokens lie around its own direction; a question is made of tokens of one passage.
    topic = normal(passages, WIDTH)
    tokens = topic[:, None] + 0.7 * normal(passages, PAGE, WIDTH)
    to_q, to_k, to_v = normal(WIDTH, HEADS * DIM) / WIDTH, normal(WIDTH, KV_HEADS * DIM) / WIDTH ** 0.5, \
        normal(WIDTH, KV_HEADS * DIM) / WIDTH ** 0.5
    to_q = (to_k.view(WIDTH, KV_HEADS, 1, DIM) * 1.5).expand(-1, -1, HEADS // KV_HEADS, -1).reshape(WIDTH, -1) + to_q
    about = torch.randint(passages, (questions,), generator=gen, device="cuda")

    def project(x):
        """(q, k, v) of tokens [n, WIDTH], as slices of one product."""
        y = (x @ torch.cat([to_q, to_k, to_v], 1)).to(kind).view(x.shape[0], -1, DIM)
        return y[:, :HEADS], y[:, HEADS:HEADS + KV_HEADS], y[:, HEADS + KV_HEADS:]

    # the pages: one per passage, then each question's own (its tokens, then what is kept and the tokens that follow)
    tail, kept_pages = -(-asked // PAGE), -(-(keep + steps) // PAGE)
    pages = passages + questions * (tail + kept_pages)
    k_pages, v_pages = (torch.zeros((pages, PAGE, KV_HEADS, DIM), dtype=kind, device="cuda") for _ in range(2))
    cache = PagedCache(k_pages, v_pages)
    i32 = dict(dtype=torch.int32, device="cuda")
    _, k, v = project(tokens.view(-1, WIDTH))
    cache.append(k, v, torch.arange(0, passages * PAGE + 1, PAGE, **i32), torch.arange(passages, **i32)[:, None],
                 torch.full((passages,), PAGE, **i32))

    # 1. search: passages by their mean token
    vectors = tokens.mean(1)
    centroids = data.pq_train_gpu(vectors, 16, 5, seed + 1)
    codes = data.gpu_encoder()(centroids, vectors.cpu().numpy())
    question = tokens[about][:, torch.randperm(PAGE, generator=gen, device="cuda")[:asked]]
    hits = torch.empty((questions, found), dtype=torch.int64, device="cuda")
    with PQSearcher(centroids, codes) as index:
        index.set_tuning(Tuning(queries_per_block=8, vectors_per_step=2))
        index.search_device(question.mean(1).contiguous(), found, hits)
        index.sync()
    ids = device_result_split(hits)[1]

    # 2. read: the passages' pages and the question's own
    own = passages + torch.arange(questions * (tail + kept_pages), **i32).view(questions, -1)
    table = torch.cat([ids, own[:, :tail]], 1).contiguous()
    lens = torch.full((questions,), found * PAGE + asked, **i32)
    offsets = torch.arange(0, questions * asked + 1, asked, **i32)
    weights = torch.zeros((questions, KV_HEADS, found * PAGE + asked + steps), device="cuda")
    q, k, v = project(question.reshape(-1, WIDTH))
    cache.append(k, v, offsets, table, lens)
    cache.attend(q, offsets, table, lens, scores=weights, max_q=asked)
    read = weights[:, :, :found * PAGE].view(questions, KV_HEADS, found, PAGE).sum((1, 3))  # by passage

    # 3. forget: into the question's remaining pages
    table = own[:, tail:].contiguous()
    before = torch.cat([ids, own[:, :tail]], 1).contiguous()
    kept, lens, weights = cache.evict(before, lens, table, keep, asked, weights)

    # 4. go on: each new token sees what was kept and the tokens before it
    offsets = torch.arange(questions + 1, **i32)
    x = question[:, -1]
    for _ in range(steps):
        lens += 1
        q, k, v = project(x)
        cache.append(k, v, offsets, table, lens)
        out, lse = cache.attend(q, offsets, table, lens, scores=weights, max_q=1)
        x = x + 0.1 * out.float().view(questions, HEADS, DIM).mean(1).repeat(1, WIDTH // DIM)
    cache.sync()
    return {"about": about, "ids": ids, "read": read, "kept": kept, "lens": lens, "weights": weights, "out": out, "lse": lse,
            "q": q, "table": table, "k": k_pages, "v": v_pages, "cache": cache, "keep": keep, "asked": asked}


def main() -> None:
    r = run()
    first = (r["ids"] == r["about"][:, None]).int().argmax(1)
    hit = (r["ids"] == r["about"][:, None]).any(1)
    share = r["read"].gather(1, first[:, None].long())[:, 0] / r["read"].sum(1)
    slots = r["kept"] // PAGE
    mine = (slots == first[:, None, None]).float().sum(2).mean(1) / (r["keep"] - r["asked"])
    print("question  passage  found  share of the passages' attention  share of the kept passage slots")
    for b in range(len(hit)):
        print(f"{b:8d} {int(r['about'][b]):8d} {'yes' if hit[b] else 'no':>6} {float(share[b]):33.2f} {float(mine[b]):32.2f}")
    print(f"slots after {int(r['lens'][0]) - r['keep']} more tokens: {r['lens'].tolist()}")


if __name__ == "__main__":
    main()
