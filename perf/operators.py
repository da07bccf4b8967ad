"""The decoding operators, measured: a chunk's attention over a paged cache and the write that feeds it, beam
search's choice of tokens and the move of the beams' caches that follows it.

`own` False: the operators' plain forms, elementary torch operations in 32 bits.  `own` True: the framework's
entry points, as a decoding loop calls them.
"""
import math
import random

import torch

own = False

DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
DEV = "cuda"


def listed():
    return [
        # one request, one token: a step of GPT-2 124M (12 heads of 64) in the middle of its 1024 positions
        {"name": "attend_one_token", "op": "attend", "seqs": 1, "heads": 12, "kv_heads": 12, "dim": 64, "page": 16,
         "chunk": 1, "ctx": 700, "ragged": 0, "window": 0, "type": "f16", "head_major": False},
        # a serving batch of the XL shape (25 heads of 64), one token each, contexts of all lengths up to 1024
        {"name": "attend_batch_tokens", "op": "attend", "seqs": 48, "heads": 25, "kv_heads": 25, "dim": 64,
         "page": 16, "chunk": 1, "ctx": 1024, "ragged": 3, "window": 0, "type": "f16", "head_major": False},
        # long contexts with four query heads to a cache head: the cache's bytes are the cost
        {"name": "attend_long_grouped", "op": "attend", "seqs": 24, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "chunk": 1, "ctx": 24000, "ragged": 5, "window": 0, "type": "bf16", "head_major": False},
        # a few drafted tokens a request, checked at once: ragged chunks, eight query heads to a cache head
        {"name": "attend_draft_check", "op": "attend", "seqs": 16, "heads": 32, "kv_heads": 4, "dim": 128,
         "page": 32, "chunk": 6, "ctx": 6001, "ragged": 7, "window": 0, "type": "bf16", "head_major": True},
        # whole prompts of different lengths, packed, nothing cached before (GPT-2 124M heads)
        {"name": "attend_packed_prompts", "op": "attend", "seqs": 9, "heads": 12, "kv_heads": 12, "dim": 64,
         "page": 16, "chunk": 1023, "ctx": 1023, "ragged": 9, "window": 0, "type": "f16", "head_major": False},
        # a chunk of a long prompt behind what is cached of it: the largest
        {"name": "attend_prompt_chunk", "op": "attend", "seqs": 1, "heads": 16, "kv_heads": 4, "dim": 128,
         "page": 128, "chunk": 4096, "ctx": 16384, "ragged": 0, "window": 0, "type": "bf16", "head_major": True},
        # one token of each of 64 beams written to the cache, out of the c_attn product's f32 rows (XL shape)
        {"name": "append_tokens", "op": "append", "seqs": 64, "heads": 25, "kv_heads": 25, "dim": 64, "page": 16,
         "chunk": 1, "ctx": 1000, "ragged": 3, "source": "f32", "type": "f16", "head_major": False},
        # prompts written to the cache, grouped heads
        {"name": "append_prompts", "op": "append", "seqs": 7, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "chunk": 3001, "ctx": 3001, "ragged": 5, "source": "f32", "type": "bf16", "head_major": True},
        # one request with four beams, GPT-2's vocabulary, twice the beams kept (some may end)
        {"name": "select_one_request", "op": "select", "batch": 1, "beams": 4, "keep": 8, "vocab": 50257,
         "type": "f32", "finished": False},
        # a serving batch of beam searches, some beams ended
        {"name": "select_batch", "op": "select", "batch": 32, "beams": 8, "keep": 16, "vocab": 50257,
         "type": "f32", "finished": True},
        # one request's four beams follow their parents (GPT-2 124M: 12 layers, 12 heads of 64)
        {"name": "reorder_one_request", "op": "reorder", "batch": 1, "beams": 4, "layers": 12, "kv_heads": 12,
         "dim": 64, "page": 16, "prompt": 300, "made": 27, "type": "f16", "head_major": False},
        # the same for 32 requests of eight beams
        {"name": "reorder_batch", "op": "reorder", "batch": 32, "beams": 8, "layers": 12, "kv_heads": 12,
         "dim": 64, "page": 16, "prompt": 500, "made": 43, "type": "f16", "head_major": False},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "select", "reorder"])
    dim = rng.choice([64, 64, 128, 128, 80, 32])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 12, 25])
    page = rng.choice([8, 16, 32, 64, 128])
    kind = rng.choice(["f16", "bf16"])
    major = rng.random() < 0.5
    if op == "attend":
        group = rng.choice([1, 1, 2, 4, 7, 8])
        if rng.random() < 0.55:  # steps: few rows, many keys
            chunk = rng.choice([1, 1, 1, _log(rng, 2, 12)])
            seqs, ctx = _log(rng, 1, 64), _log(rng, 17, 20000)
            while seqs * ctx * kv_heads * dim > 3.0e8:
                ctx = max(chunk, ctx // 2)
            ctx = max(ctx, chunk)
        else:  # prompts, whole or a chunk behind a cached part
            chunk = _log(rng, 30, 4096)
            ctx = chunk if rng.random() < 0.5 else chunk + _log(rng, 1, 12000)
            seqs = _log(rng, 1, 8)
            while seqs * kv_heads * group * chunk * ctx > 1.0e9 and seqs > 1:
                seqs -= 1
            while seqs * kv_heads * group * chunk * ctx > 1.0e9:
                chunk = max(1, chunk * 3 // 4)
                ctx = max(chunk, ctx * 3 // 4)
        window = 0 if rng.random() < 0.75 else _log(rng, 16, 4096)
        return {"op": op, "seqs": seqs, "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "page": page,
                "chunk": chunk, "ctx": ctx, "ragged": rng.randrange(1000), "window": window, "type": kind,
                "head_major": major}
    if op == "append":
        seqs = _log(rng, 1, 64)
        chunk = 1 if rng.random() < 0.4 else _log(rng, 2, 3000)
        while seqs * chunk > 16000:
            chunk //= 2
        return {"op": op, "seqs": seqs, "heads": kv_heads * rng.choice([1, 2, 4]), "kv_heads": kv_heads, "dim": dim,
                "page": page, "chunk": chunk, "ctx": chunk + _log(rng, 1, 2000), "ragged": rng.randrange(1000),
                "source": rng.choice(["f32", "f32", kind]), "type": kind, "head_major": major}
    if op == "select":
        beams = _log(rng, 1, 16)
        batch = _log(rng, 1, 32)
        vocab = _log(rng, 1000, 200000)
        while batch * beams * vocab > 1.3e7:
            batch = max(1, batch // 2)
            vocab = vocab * 3 // 4
        return {"op": op, "batch": batch, "beams": beams, "keep": min(64, beams * rng.choice([1, 2, 2, 3])),
                "vocab": vocab, "type": rng.choice(["f32", "f32", "f16", "bf16"]), "finished": rng.random() < 0.5}
    layers = _log(rng, 1, 24)
    batch = _log(rng, 1, 32)
    while batch * layers * kv_heads * dim * page > 3.0e6:
        batch, layers = max(1, batch // 2), max(1, layers * 3 // 4)
        kv_heads = max(1, kv_heads * 3 // 4)
    return {"op": op, "batch": batch, "beams": _log(rng, 2, 12), "layers": layers, "kv_heads": kv_heads, "dim": dim,
            "page": page, "prompt": _log(rng, 5, 900), "made": _log(rng, 1, 200), "type": kind, "head_major": major}


# ---------------------------------------------------------------- shapes that a case stands for
def lengths(case):
    """(new tokens, tokens in the cache with them) of each sequence."""
    r = random.Random(case["ragged"] * 1009 + case["seqs"])
    new, ctx = [], []
    for s in range(case["seqs"]):
        if case["ragged"] == 0 or s == 0:  # the first one is the longest: the bounds are met
            n, c = case["chunk"], case["ctx"]
        else:
            n = r.randint(max(1, case["chunk"] // 4), case["chunk"])
            c = n + r.randint((case["ctx"] - case["chunk"]) // 5, case["ctx"] - case["chunk"])
        new.append(n)
        ctx.append(c)
    return new, ctx


def _visible(n, c, window):
    """(row, key) pairs that a sequence's rows see."""
    if window <= 0:
        return n * (c - n) + n * (n + 1) // 2
    return sum(min(window, c - n + i + 1) for i in range(n))


def work(case):
    if case["op"] == "select":
        rows = case["batch"] * case["beams"]
        logits = rows * case["vocab"]
        return {"bytes": logits * SIZE[case["type"]] + 4 * rows + 16 * case["batch"] * case["keep"],
                "flops": 4 * logits}
    if case["op"] == "reorder":
        rows, fill = case["batch"] * case["beams"], (case["prompt"] + case["made"]) % case["page"]
        cols, pages = _columns(case), _pool(case)
        token = 2 * case["layers"] * case["kv_heads"] * case["dim"] * SIZE[case["type"]]
        return {"bytes": 2 * (rows - _survivors(case) * case["batch"]) * fill * token + 8 * rows * cols + 8 * pages + 12 * rows,
                "flops": 0}
    new, ctx = lengths(case)
    width, token = SIZE[case["type"]], case["kv_heads"] * case["dim"]
    if case["op"] == "append":
        rows = sum(new)
        moved = rows * (2 * token + case["heads"] * case["dim"])
        return {"bytes": moved * (SIZE[case["source"]] + width), "flops": 0}
    keys = sum(c if case["window"] <= 0 else min(c, n + case["window"] - 1) for n, c in zip(new, ctx))
    rows = sum(new) * case["heads"]
    return {"bytes": 2 * keys * token * width + rows * (2 * case["dim"] * width + 4),
            "flops": 4 * case["heads"] * case["dim"] * sum(_visible(n, c, case["window"]) for n, c in zip(new, ctx))}


def _columns(case):
    return -(-(case["prompt"] + case["made"] + 1) // case["page"]) + 2


def _survivors(case):
    """Beams of a request that live on: the others' places go to second children."""
    return max(1, (case["beams"] + 1) // 2)


def _pool(case):
    shared = case["prompt"] // case["page"]
    mine = -(-(case["prompt"] + case["made"]) // case["page"]) - shared
    rows = case["batch"] * case["beams"]
    return case["batch"] * shared + rows * mine + 2 * rows + 3


# ---------------------------------------------------------------- inputs
def _pages(shape, head_major, kind, gen):
    """[..., pages, page, heads, dim], stored token-major or head-major inside a page."""
    if head_major:
        stored = shape[:-3] + (shape[-2], shape[-3], shape[-1])
        return torch.randn(stored, device=DEV, dtype=DTYPE[kind], generator=gen).transpose(-3, -2)
    return torch.randn(shape, device=DEV, dtype=DTYPE[kind], generator=gen)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed * 7919 + 13)
    if case["op"] == "select":
        rows, vocab = case["batch"] * case["beams"], case["vocab"]
        # a language model's logits: a wide body, and some tens of tokens that stand out, less and less
        x = torch.randn(rows, vocab, device=DEV, generator=gen) * 2.0
        best = torch.randint(0, vocab, (rows, 40), device=DEV, generator=gen)
        up = torch.rand(rows, 40, device=DEV, generator=gen) * torch.linspace(14.0, 4.0, 40, device=DEV)
        x.scatter_add_(1, best, up)
        scores = -20.0 * torch.rand(rows, device=DEV, generator=gen) / case["beams"]
        done = None
        if case["finished"]:
            done = torch.rand(rows, device=DEV, generator=gen) < 0.15
        return {"case": case, "logits": x.to(DTYPE[case["type"]]), "scores": scores, "finished": done,
                "eos": vocab - 1}
    page, kv, dim = case["page"], case["kv_heads"], case["dim"]
    if case["op"] == "reorder":
        batch, beams = case["batch"], case["beams"]
        rows, total, cols = batch * beams, case["prompt"] + case["made"], _columns(case)
        shared, pool = case["prompt"] // page, _pool(case)
        mine = -(-total // page) - shared
        order = torch.randperm(pool, device=DEV, generator=gen).to(torch.int32)
        table = torch.full((batch, beams, cols), -1, dtype=torch.int32, device=DEV)
        table[:, :, :shared] = order[:batch * shared].view(batch, 1, shared)
        table[:, :, shared:shared + mine] = order[batch * shared:batch * shared + rows * mine].view(batch, beams, mine)
        table = table.view(rows, cols)
        refs = torch.zeros(pool, dtype=torch.int32, device=DEV)
        refs[order[:batch * shared].long()] = beams
        refs[order[batch * shared:batch * shared + rows * mine].long()] = 1
        # each request: `survivors` beams chosen at random, every one of them a parent, the rest second children
        alive = _survivors(case)
        pick = torch.rand(batch, beams, device=DEV, generator=gen).argsort(1)[:, :alive]
        child = torch.arange(beams, device=DEV) % alive
        parents = pick[:, child] + torch.arange(batch, device=DEV)[:, None] * beams
        shuffle = torch.rand(batch, beams, device=DEV, generator=gen).argsort(1)
        parents = parents.gather(1, shuffle).reshape(rows).to(torch.int32)
        shape = (case["layers"], pool, page, kv, dim)
        return {"case": case, "table": table, "lens": _ints([total] * rows), "parents": parents, "refs": refs,
                "k": _pages(shape, case["head_major"], case["type"], gen),
                "v": _pages(shape, case["head_major"], case["type"], gen)}
    new, ctx = lengths(case)
    cols = -(-max(ctx) // page)
    held = [-(-c // page) for c in ctx]
    pool = sum(held) + 5
    order = torch.randperm(pool, device=DEV, generator=gen).to(torch.int32)
    starts = [sum(held[:s]) for s in range(len(held))]
    at = _ints(starts)[:, None] + torch.arange(cols, device=DEV, dtype=torch.int32)
    inside = torch.arange(cols, device=DEV)[None] < _ints(held)[:, None]
    table = torch.where(inside, order[at.clamp(max=pool - 1).long()], torch.full_like(at, -1))
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    shape = (pool, page, kv, dim)
    state = {"case": case, "table": table, "ctx": _ints(ctx), "cu": _ints(cu), "rows": cu[-1], "max_q": max(new),
             "max_ctx": max(ctx), "k": _pages(shape, case["head_major"], case["type"], gen),
             "v": _pages(shape, case["head_major"], case["type"], gen)}
    if case["op"] == "append":
        # the rows of the projection before: [q | k | v], heads side by side
        wide = torch.randn(cu[-1], (case["heads"] + 2 * kv) * dim, device=DEV, generator=gen).to(DTYPE[case["source"]])
        q, k, v = wide.split([case["heads"] * dim, kv * dim, kv * dim], 1)
        state |= {"q": q.unflatten(1, (case["heads"], dim)), "new_k": k.unflatten(1, (kv, dim)),
                  "new_v": v.unflatten(1, (kv, dim))}
    else:
        state["q"] = (torch.randn(cu[-1], case["heads"], dim, device=DEV, generator=gen) * 1.5).to(DTYPE[case["type"]])
    return state


# ---------------------------------------------------------------- one pass
def run(state):
    return {"attend": _attend, "append": _append, "select": _select, "reorder": _reorder}[state["case"]["op"]](state)


def _places(cu, ctx, rows):
    """(sequence, row in its chunk, position) of each packed row."""
    at = torch.arange(rows, device=cu.device)
    seq = torch.searchsorted(cu[1:].contiguous(), at, right=True)
    row = at - cu[seq]
    return seq, row, ctx[seq] - (cu[seq + 1] - cu[seq]) + row


def _attend(s):
    case = s["case"]
    if own:
        from tokenvector.inference_b200.generation import paged_attention
        out, lse = paged_attention(s["q"], s["k"], s["v"], s["table"], s["ctx"], s["cu"], max_q=s["max_q"],
                                   window=case["window"], return_lse=True)
        return {"out": out, "lse": lse}
    q, ctx, cu = s["q"], s["ctx"], s["cu"]
    heads, kv, dim, most = case["heads"], case["kv_heads"], case["dim"], s["max_q"]
    group = heads // kv
    seqs = ctx.numel()
    # the cache as [seqs, kv, keys, dim], what lies behind a sequence's end as zeros
    pages = s["table"][:, :-(-s["max_ctx"] // case["page"])].clamp(min=0).long()
    keys = pages.shape[1] * case["page"]
    at = torch.arange(keys, device=q.device)
    there = (at[None] < ctx[:, None])[:, None, :, None]
    k = s["k"][pages].reshape(seqs, keys, kv, dim).transpose(1, 2).float().masked_fill_(~there, 0.0)
    v = s["v"][pages].reshape(seqs, keys, kv, dim).transpose(1, 2).float().masked_fill_(~there, 0.0)
    # the chunks as [seqs, kv, group * most, dim]
    new = cu[1:] - cu[:-1]
    row = torch.arange(most, device=q.device)
    packed = (cu[:-1, None] + row[None]).clamp(max=s["rows"] - 1)
    qs = q[packed].float().view(seqs, most, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(seqs, kv, group * most, dim)
    score = torch.matmul(qs * (1.0 / math.sqrt(dim)), k.transpose(2, 3)).view(seqs, kv, group, most, keys)
    pos = (ctx - new)[:, None] + row[None]
    seen = at[None, None] <= pos[:, :, None]
    if case["window"] > 0:
        seen = seen & (at[None, None] > pos[:, :, None] - case["window"])
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    low = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = score.sub_(low).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(seqs, kv, group * most, keys), v).view(seqs, kv, group, most, dim)
    out = out / torch.where(total == 0, torch.ones_like(total), total)
    lse = (low + total.log())[..., 0]
    seq, row, _ = _places(cu, ctx, s["rows"])
    return {"out": out[seq, :, :, row].reshape(s["rows"], heads, dim).to(q.dtype),
            "lse": lse[seq, :, :, row].reshape(s["rows"], heads)}


def _append(s):
    if own:
        from tokenvector.inference_b200.generation import paged_append
        q = paged_append(s["new_k"], s["new_v"], s["k"], s["v"], s["table"], s["ctx"], s["cu"], q=s["q"])
        return {"q": q, "k": s["k"], "v": s["v"]}
    page, kind = s["case"]["page"], s["k"].dtype
    seq, _, pos = _places(s["cu"], s["ctx"], s["rows"])
    at, slot = s["table"][seq, pos // page].long(), pos % page
    s["k"][at, slot] = s["new_k"].float().to(kind)
    s["v"][at, slot] = s["new_v"].float().to(kind)
    return {"q": s["q"].float().to(kind).contiguous(), "k": s["k"], "v": s["v"]}


def _select(s):
    case = s["case"]
    if own:
        from tokenvector.inference_b200.generation import beam_select
        scores, tokens, parents = beam_select(s["logits"], s["scores"], case["beams"], case["keep"],
                                              finished=s["finished"], eos=s["eos"])
        return {"scores": scores, "tokens": tokens, "parents": parents}
    batch, beams, keep, vocab = case["batch"], case["beams"], case["keep"], case["vocab"]
    x = s["logits"].float() + 0.0
    x = torch.where(x.isnan(), torch.full_like(x, -math.inf), x)
    token = torch.arange(vocab, device=x.device)
    if s["finished"] is not None:
        only = torch.where(token == s["eos"], 0.0, -math.inf)
        x = torch.where(s["finished"][:, None], only[None], x)
    top = x.amax(1, keepdim=True)
    z = (x - top).exp().sum(1, keepdim=True).log()
    # each beam's best, ties to the lowest token: the value's bits in its order above, the token's place below
    bits = x.view(torch.int32).long()
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) * (1 << 32) + ((1 << 32) - 1 - token)
    mine = order.topk(keep, 1).indices
    total = s["scores"][:, None] + ((x.gather(1, mine) - top) - z)
    total = torch.where(total.isnan(), torch.full_like(total, -math.inf), total).view(batch, beams * keep)
    best = torch.sort(total, dim=1, descending=True, stable=True).indices[:, :keep]
    return {"scores": total.gather(1, best), "tokens": mine.view(batch, beams * keep).gather(1, best),
            "parents": (best // keep).to(torch.int32)}


def _reorder(s):
    if own:
        from tokenvector.inference_b200.generation import beam_reorder
        table, lens, refs, status = beam_reorder(s["table"], s["lens"], s["parents"], s["refs"], s["k"], s["v"])
        return {"table": table, "lens": lens, "refs": refs, "status": status, "k": s["k"], "v": s["v"]}
    table, lens, refs, k, v = s["table"], s["lens"], s["refs"], s["k"], s["v"]
    page, (rows, cols), pool = s["case"]["page"], table.shape, refs.numel()
    live = s["parents"] >= 0
    src = s["parents"].clamp(min=0).long()
    size = torch.where(live, lens[src], torch.zeros_like(lens[src]))
    col = torch.arange(cols, device=table.device)

    def holds(t, n):  # how often the tables hold each page
        inside = col[None] < ((n + page - 1) // page)[:, None]
        where = torch.where(inside & (t >= 0), t, torch.full_like(t, pool)).long().view(-1)
        return torch.zeros(pool + 1, dtype=torch.int32, device=t.device).scatter_add_(
            0, where, torch.ones_like(where, dtype=torch.int32))[:pool]

    moved = torch.where(col[None] < ((size + page - 1) // page)[:, None], table[src], torch.full_like(table[src], -1))
    before = holds(table, lens)
    at, fill = (size // page).long(), size % page
    tail = moved.gather(1, at.clamp(max=cols - 1)[:, None])[:, 0].clamp(min=0).long()
    part = live & (fill > 0)
    same = (tail[:, None] == tail[None]) & part[:, None] & part[None]
    keeps = part & ~same.tril(-1).any(1) & (refs[tail] == before[tail])
    fresh = live & ~keeps & (at < cols)
    free = torch.argsort((refs != 0).to(torch.int32), stable=True)
    turn = torch.cumsum(fresh, 0) - 1
    got = fresh & (turn < (refs == 0).sum())
    taken = torch.where(got, free[turn.clamp(0, pool - 1)], torch.full_like(tail, -1))
    moved = torch.where(fresh[:, None] & (col[None] == at[:, None]), taken[:, None].to(torch.int32), moved)
    # rows that copy nothing write their tail onto itself
    copies = got & part
    dst = torch.where(copies, taken, tail)
    slot = torch.arange(page, device=table.device)[None] < fill[:, None]
    for cache in (k, v):
        cache[:, dst] = torch.where((slot & copies[:, None])[None, :, :, None, None], cache[:, tail], cache[:, dst])
    full = torch.where(got, size + 1, size)
    return {"table": moved, "lens": size, "refs": refs - before + holds(moved, full), "k": k, "v": v,
            "status": torch.stack([got.sum(), (live & ~keeps & ~got).sum()]).to(torch.int32)}


# ---------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "reorder":
        return None  # it computes no numbers: everything is moved or counted
    if case["op"] == "append":
        return {"q": s["q"].double(), "k": None, "v": None}
    if case["op"] == "select":
        x = s["logits"].double()
        if s["finished"] is not None:
            x[s["finished"]] = -math.inf
            x[s["finished"], s["eos"]] = 0.0
        total = (torch.log_softmax(x, 1) + s["scores"].double()[:, None]).view(case["batch"], -1)
        return {"scores": total.topk(case["keep"], 1).values, "tokens": None, "parents": None}
    new, ctx = lengths(case)
    group, page = case["heads"] // case["kv_heads"], case["page"]
    out = torch.zeros(s["rows"], case["heads"], case["dim"], dtype=torch.float64, device=DEV)
    lse = torch.full((s["rows"], case["heads"]), -math.inf, dtype=torch.float64, device=DEV)
    first = 0
    for i, (n, c) in enumerate(zip(new, ctx)):
        pages = s["table"][i, :-(-c // page)].long()
        pos = torch.arange(c - n, c, device=DEV)[:, None]
        j = torch.arange(c, device=DEV)[None]
        hidden = (j > pos) | ((j <= pos - case["window"]) if case["window"] > 0 else (j < 0))
        for g in range(case["kv_heads"]):
            k = s["k"][pages, :, g].reshape(-1, case["dim"])[:c].double()
            v = s["v"][pages, :, g].reshape(-1, case["dim"])[:c].double()
            for h in range(g * group, (g + 1) * group):
                a = (s["q"][first:first + n, h].double() @ k.T) / math.sqrt(case["dim"])
                a[hidden] = -math.inf
                lse[first:first + n, h] = torch.logsumexp(a, 1)
                out[first:first + n, h] = torch.softmax(a, 1) @ v
        first += n
    return {"out": out, "lse": lse}
