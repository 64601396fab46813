"""Operators of prompts over a paged K/V cache, as the dense engine runs them.

A request's first tokens may lie in the cache already (a shared system prompt, the
chunk of a long prompt that went before). Its next ones come as a chunk of rows, the
chunks of all requests one behind the other: their cache rows are laid out, their
keys and values written, and every new token attends to all that the cache holds
before it and to itself. The kinds of case:

attend  attention of the chunks' rows over the paged cache; a chunk may be a
        single token, nothing may be cached yet
slots   block tables, positions and cache rows of the chunks, from the requests'
        lengths and a list of free pages
"""

import math

import torch

own = False

DEVICE = "cuda"
# query heads, kv heads and head size of the model registry
HEADS = [(8, 2, 64), (14, 2, 64), (12, 2, 128), (28, 4, 128), (32, 8, 128),
         (40, 8, 128), (64, 8, 128)]


# ------------------------------------------------------------------ cases

def _attend(heads, block, requests, new, cached, singles=0):
    h, kv, d = heads
    return {"kind": "attend", "heads": h, "kv_heads": kv, "dim": d, "block": block,
            "requests": requests, "new_least": new[0], "new_most": new[1],
            "cached_least": cached[0], "cached_most": cached[1], "singles": singles}


def _slots(block, requests, new, cached):
    return {"kind": "slots", "block": block, "requests": requests, "new_least": new[0],
            "new_most": new[1], "cached_least": cached[0], "cached_most": cached[1]}


def listed():
    return [
        # a server's request on the 0.5B model: a few words behind a cached
        # system prompt
        {"name": "attend_one_tail", **_attend((14, 2, 64), 16, 1, (5, 5), (1040, 1040))},
        # a batch of requests on the 7B model whose tails differ
        {"name": "attend_tails", **_attend((28, 4, 128), 16, 16, (20, 121), (1040, 1040))},
        # bench.py's prompts on the 7B model, nothing cached
        {"name": "attend_prompts", **_attend((28, 4, 128), 16, 10, (200, 350), (0, 0))},
        # a step that carries chats' single tokens beside two prompts' chunks
        {"name": "attend_mixed_step", **_attend((32, 8, 128), 16, 32, (512, 512), (400, 2900),
                                                singles=30)},
        # single tokens of a few long histories: little to compute, all to read
        {"name": "attend_long_singles", **_attend((40, 8, 128), 16, 6, (1, 1), (20011, 32111))},
        # the last chunk of one long document
        {"name": "attend_deep_chunk", **_attend((28, 4, 128), 16, 1, (2048, 2048),
                                                (14336, 14336))},
        # chunks of a 72B model's long prompts, larger pages
        {"name": "attend_large", **_attend((64, 8, 128), 64, 2, (4096, 4096), (8192, 8192))},
        # a server's step of a few requests
        {"name": "slots_few", **_slots(16, 4, (1, 37), (900, 1100))},
        # bench.py's round: 30 prompts x 16 candidates, one prompt each
        {"name": "slots_round", **_slots(16, 480, (200, 350), (0, 0))},
        # long chunks of many requests
        {"name": "slots_large", **_slots(16, 1000, (100, 4001), (0, 8000))},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _span(rng, low, high):
    a, b = sorted((_spread(rng, low, high), _spread(rng, low, high)))
    return a, b


def draw(rng):
    block = rng.choice([8, 16, 16, 16, 24, 32, 64])
    if rng.random() < 0.3:
        requests = _spread(rng, 1, 1000)
        most = min(8000, max(2, 2_000_000 // requests))
        return _slots(block, requests, _span(rng, 1, most),
                      rng.choice([(0, 0), _span(rng, 1, 8000)]))
    heads = rng.choice(HEADS)
    while True:
        requests, new = _spread(rng, 1, 64), rng.choice([(1, 1), _span(rng, 1, 4096)])
        cached = rng.choice([(0, 0), _span(rng, 1, 30000)])
        # the plain form holds all scores of the batch, padded, in 32 bits
        pairs = requests * heads[0] * new[1] * (new[1] + cached[1])
        if pairs <= 2 * 64 * 4096 * 12288 and requests * cached[1] <= 400_000:
            singles = rng.choice([0, 0, requests // 2])
            return _attend(heads, block, requests, new, cached, singles)


def _lengths(case):
    """New and cached tokens of every request, fixed by the case's values."""
    n = case["requests"]

    def between(low, high, step):
        return [low + (i * step + 11) % (high - low + 1) for i in range(n)]

    new = between(case["new_least"], case["new_most"], 7919)
    cached = between(case["cached_least"], case["cached_most"], 6151)
    return [1] * case.get("singles", 0) + new[case.get("singles", 0):], cached


def work(case):
    new, cached = _lengths(case)
    pages = sum(-(-(c + n) // case["block"]) for n, c in zip(new, cached))
    if case["kind"] == "slots":
        held = sum(-(-c // case["block"]) for c in cached)
        # a page that a token goes to but does not open is read from the table
        return {"bytes": 12 * sum(new) + 8 * (pages - held) + 28 * len(new), "flops": 0}
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    seen = sum(n * c + n * (n + 1) // 2 for n, c in zip(new, cached))
    rows = sum(new)
    return {"bytes": 2 * 2 * rows * h * d + 2 * 2 * (rows + sum(cached)) * kv * d + 4 * pages
            + 12 * len(new), "flops": 4 * h * d * seen}


# ----------------------------------------------------------------- inputs

def _tensor(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    new, cached = _lengths(case)
    block = case["block"]
    held = [-(-c // block) for c in cached]
    needed = [-(-(c + n) // block) for n, c in zip(new, cached)]
    total = sum(needed)
    order = torch.randperm(total + 3, generator=gen, device=DEVICE)[:total].to(torch.int32)
    # a request's pages one behind the other, as rows of its table
    width = max(needed)
    column = torch.arange(width, device=DEVICE)
    there = column < _tensor(needed)[:, None]
    tables = torch.zeros(len(new), width, dtype=torch.int32, device=DEVICE)
    tables[there] = order
    state = {"case": case, "rows": sum(new), "longest": max(new), "block": block}
    if case["kind"] == "slots":
        opened = there & (column >= _tensor(held)[:, None])
        pages = tables[opened]
        tables[opened] = -1
        return {**state, "tables": tables, "pages": pages, "cached": _tensor(cached),
                "new": _tensor(new)}
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=DEVICE, dtype=torch.float32)

    packed = normal(sum(new), (h + 2 * kv) * d).to(torch.bfloat16)
    cache = [torch.empty(total + 3, block, kv, d, dtype=torch.bfloat16, device=DEVICE)
             .normal_(generator=gen) for _ in range(2)]
    ends = torch.tensor([0] + new, dtype=torch.int64).cumsum(0).tolist()
    return {**state, "q": packed[:, :h * d].unflatten(1, (h, d)), "key": cache[0],
            "value": cache[1], "tables": tables, "cu": _tensor(ends),
            "context": _tensor([n + c for n, c in zip(new, cached)]), "scale": d ** -0.5}


# -------------------------------------------------------------------- run

def run(state):
    if state["case"]["kind"] == "slots":
        return _own_slots(state) if own else _plain_slots(state)
    return _own_attend(state) if own else _plain_attend(state)


def _own_attend(s):
    from distrl_llm_amd.ops import functional as OF
    return OF.paged_attention_chunk(s["q"], s["key"], s["value"], s["tables"], s["cu"],
                                    s["context"], s["scale"], s["longest"])


def _own_slots(s):
    from distrl_llm_amd.ops import functional as OF
    plan = OF.chunk_slots(s["tables"], s["cached"], s["new"], s["pages"], s["block"], s["rows"])
    return {"positions": plan.positions, "slots": plan.slots, "cu": plan.cu,
            "context": plan.context_lens, "last": plan.last, "tables": s["tables"]}


def _plain_attend(s):
    q, tables, cu, context = s["q"], s["tables"].long(), s["cu"].long(), s["context"].long()
    kv, d = s["key"].shape[2:]
    h = q.shape[1]
    new, longest = cu[1:] - cu[:-1], s["longest"]
    row = torch.arange(longest, device=q.device)
    at = (cu[:-1, None] + row).clamp(max=q.shape[0] - 1)                # (B, longest)
    qp = q[at].float().unflatten(2, (kv, h // kv)).permute(0, 2, 3, 1, 4)
    qp = qp.reshape(len(new), kv, -1, d)                                # rows: head, token
    kp = s["key"][tables].flatten(1, 2).permute(0, 2, 3, 1).float()     # (B, kv, d, keys)
    vp = s["value"][tables].flatten(1, 2).permute(0, 2, 1, 3).float()
    p = torch.matmul(qp * s["scale"], kp).unflatten(2, (h // kv, longest))
    seen = context[:, None] - new[:, None] + row                        # a row's position
    hidden = torch.arange(kp.shape[3], device=q.device) > seen[:, :, None]
    p.masked_fill_(hidden[:, None, None], float("-inf"))
    p.sub_(p.amax(-1, keepdim=True)).exp_()
    p.div_(p.sum(-1, keepdim=True))
    o = torch.matmul(p.flatten(2, 3), vp).unflatten(2, (h // kv, longest))
    o = o.permute(0, 3, 1, 2, 4).flatten(2, 3)                          # (B, longest, h, d)
    return o[row < new[:, None]].to(q.dtype)


def _plain_slots(s):
    tables, cached, new, block = s["tables"], s["cached"].long(), s["new"].long(), s["block"]
    context = cached + new
    held, needed = (cached + block - 1) // block, (context + block - 1) // block
    column = torch.arange(tables.shape[1], device=tables.device)
    opened = (column >= held[:, None]) & (column < needed[:, None])
    tables[opened] = s["pages"]
    cu = torch.cat([new.new_zeros(1), new.cumsum(0)])
    request = torch.repeat_interleave(new, output_size=s["rows"])
    position = torch.arange(s["rows"], device=tables.device) - cu[request] + cached[request]
    slot = tables[request, position // block].long() * block + position % block
    return {"positions": position.to(torch.int32), "slots": slot, "cu": cu.to(torch.int32),
            "context": context.to(torch.int32), "last": cu[1:] - 1, "tables": tables}


# ------------------------------------------------------------------ exact

def exact(case, seed):
    """Attention in 64 bits, request by request and kv head by kv head."""
    if case["kind"] == "slots":
        return None
    s = prepare(case, seed)
    new, cached = _lengths(case)
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    group, block = h // kv, case["block"]
    out = torch.empty(sum(new), h, d, dtype=torch.float64, device=DEVICE)
    first = 0
    for b, (n, c) in enumerate(zip(new, cached)):
        place = torch.arange(n + c, device=DEVICE)
        line = s["tables"][b].long()[place // block] * block + place % block
        later = place[None, :] > place[c:, None]
        for g in range(kv):
            key = s["key"].view(-1, kv, d)[line, g].double()
            value = s["value"].view(-1, kv, d)[line, g].double()
            for i in range(g * group, (g + 1) * group):
                score = s["q"][first:first + n, i].double() @ key.T / math.sqrt(d)
                score[later] = -math.inf
                out[first:first + n, i] = score.softmax(1) @ value
        first += n
    return out
