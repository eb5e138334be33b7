"""Timed cases of the operators for language models: attention whose scores are changed by a formula and masked by rules, and what
generation token by token needs next to it (page tables, the 8-bit cache's writes, attention over that cache).

  scored   `scored_attention`: tanh cap, distance bias (slopes or a table), document / prefix / causal / window / padding masks
  cache    `cache_attention`: one or a few tokens per request over a paged 8-bit cache with a scale per page and head
  append   `cache_append`: new keys and values quantised into their slots
  tables   `page_tables`: block tables and slot maps from request lengths, pages taken from and given back to a stack

`run` computes the plain form in elementary torch operations, or, where `own` is set, calls the framework.
"""
import functools
import math
import os
import random
import sys

import torch

own = False

SCORED = {"batch": 1, "heads": 12, "kv_heads": 12, "seq": 128, "past": 0, "dim": 64, "dtype": "fp16", "causal": True, "window": 0, "softcap": 0.0,
          "bias": "", "documents": False, "prefix": False, "padded": False}
CACHE = {"requests": 1, "heads": 12, "kv_heads": 12, "dim": 64, "dtype": "fp16", "cache": "int8", "page": 16, "longest": 1024, "tokens": 1,
         "window": 0, "softcap": 0.0, "bias": ""}


def listed():
    return [
        # one short prompt of a small model with linear distance bias: latency
        {"name": "scored 1x12x200 slopes", "kind": "scored", **SCORED, "seq": 200, "bias": "slopes"},
        # an encoder batch of short texts packed into rows, every text attending to itself alone
        {"name": "scored 4x12x1120 documents", "kind": "scored", **SCORED, "batch": 4, "seq": 1120, "causal": False, "documents": True},
        # a padded encoder batch with a learned bias per head and clipped distance
        {"name": "scored 8x16x1001 table padded", "kind": "scored", **SCORED, "batch": 8, "heads": 16, "kv_heads": 16, "seq": 1001, "causal": False,
         "bias": "table", "padded": True},
        # a local layer of a model with capped scores: window, shared K/V heads, a prompt's second half on top of its first
        {"name": "scored 2x32x2048+2048 window cap", "kind": "scored", **SCORED, "batch": 2, "heads": 32, "kv_heads": 8, "seq": 2048, "past": 2048,
         "dim": 128, "dtype": "bf16", "window": 1024, "softcap": 50.0},
        # the largest: a long prompt through a global layer with capped scores, its first part visible to all
        {"name": "scored 1x32x8192 cap prefix", "kind": "scored", **SCORED, "heads": 32, "kv_heads": 8, "seq": 8192, "dim": 128, "dtype": "bf16",
         "softcap": 50.0, "prefix": True},
        # one request being answered: latency
        {"name": "cache 1x32x4000 int8", "kind": "cache", **CACHE, "heads": 32, "kv_heads": 8, "dim": 128, "longest": 4000},
        # a small model's batch, four tokens guessed ahead, linear distance bias
        {"name": "cache 16x12x2048 4 tokens", "kind": "cache", **CACHE, "requests": 16, "longest": 2048, "tokens": 4, "page": 64, "bias": "slopes"},
        # the largest: a full serving batch of uneven requests
        {"name": "cache 96x32x16000 e4m3 cap", "kind": "cache", **CACHE, "requests": 96, "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16",
         "cache": "e4m3", "page": 32, "longest": 16000, "softcap": 30.0},
        # the tokens of one step of a serving batch
        {"name": "append 64x1", "kind": "append", "requests": 64, "kv_heads": 8, "dim": 128, "dtype": "bf16", "page": 16, "held": 2000, "new": 1},
        # prompts: whole pages and ragged ends
        {"name": "append 9x2000", "kind": "append", "requests": 9, "kv_heads": 8, "dim": 128, "dtype": "fp16", "page": 32, "held": 0, "new": 2000},
        # a step of a serving batch: a token each, now and then a page, some requests done
        {"name": "tables 256 step", "kind": "tables", "requests": 256, "page": 16, "longest": 8000, "prompts": False},
        # a batch of prompts comes in while others leave
        {"name": "tables 1000 prompts", "kind": "tables", "requests": 1000, "page": 32, "longest": 2000, "prompts": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["scored", "scored", "cache", "cache", "append", "tables"])
    dtype = rng.choice(["fp16", "bf16"])
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 4])
    dim = rng.choice([64, 128])
    bias = rng.choice(["", "", "slopes", "table"])
    softcap = rng.choice([0.0, 0.0, 30.0, 50.0])
    if kind == "scored":
        seq, past = _log(rng, 1, 6000), rng.choice([0, 0, _log(rng, 1, 2000)])
        batch = max(1, min(_log(rng, 1, 16), int(1.5e9 / (heads * seq * (seq + past)))))
        causal = rng.random() < 0.7
        return {"kind": kind, "batch": batch, "heads": heads, "kv_heads": kv, "seq": seq, "past": past, "dim": dim, "dtype": dtype, "causal": causal,
                "window": _log(rng, 16, 2000) if rng.random() < 0.3 else 0, "softcap": softcap, "bias": bias, "documents": rng.random() < 0.3,
                "prefix": causal and rng.random() < 0.3, "padded": rng.random() < 0.3}
    if kind == "cache":
        longest = _log(rng, 1, 16000)
        return {"kind": kind, "requests": max(1, min(_log(rng, 1, 128), int(1e9 / (longest * kv * dim)))), "heads": heads, "kv_heads": kv, "dim": dim,
                "dtype": dtype, "cache": rng.choice(["int8", "e4m3"]), "page": rng.choice([16, 32, 64, 128]), "longest": longest,
                "tokens": min(longest, rng.choice([1, 1, 1, 2, 5])), "window": _log(rng, 16, 4000) if rng.random() < 0.2 else 0, "softcap": softcap,
                "bias": bias}
    if kind == "append":
        prompts = rng.random() < 0.5
        return {"kind": kind, "requests": _log(rng, 1, 16 if prompts else 256), "kv_heads": kv, "dim": dim, "dtype": dtype, "page": rng.choice([16, 32, 64, 128]),
                "held": rng.choice([0, _log(rng, 1, 500)]) if prompts else _log(rng, 1, 2000), "new": _log(rng, 16, 1500) if prompts else rng.choice([1, 1, 3])}
    return {"kind": kind, "requests": _log(rng, 1, 1024), "page": rng.choice([16, 32, 64, 128]), "longest": _log(rng, 64, 4000), "prompts": rng.random() < 0.5}


# ------------------------------------------------------------------------------------------
# what a case stands for beyond its sizes: lengths and documents (the same for every seed)
# ------------------------------------------------------------------------------------------
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TABLE_RADIUS = 128                     # distances beyond it share the table's outermost entries


def _key_lens(case):
    total = case["seq"] + case["past"]
    r = random.Random(total)
    return [total] + [r.randint((total + 1) // 2, total) for _ in range(case["batch"] - 1)]


def _prefix_lens(case):
    r = random.Random(case["seq"] + 1)
    return [r.randint(0, max(1, (case["seq"] + case["past"]) // 4)) for _ in range(case["batch"])]


def _documents(case):
    """(batch, keys) document numbers: texts of 20 to 400 tokens back to back."""
    total = case["seq"] + case["past"]
    g = torch.Generator().manual_seed(total)
    ends = torch.randint(20, 401, (case["batch"], total // 20 + 1), generator=g).cumsum(1)
    return torch.searchsorted(ends, torch.arange(total).expand(case["batch"], total).contiguous(), right=True).int()


def _request_lengths(case):
    r = random.Random(case["longest"])
    return [case["longest"]] + [r.randint(max(case["tokens"], case["longest"] // 8), case["longest"]) for _ in range(case["requests"] - 1)]


def _held_and_lengths(case):
    r = random.Random(case["requests"])
    if case["prompts"]:                # every third request leaves, every third comes in, the others take a token
        held = [0 if i % 3 == 1 else r.randint(1, case["longest"] - 1) for i in range(case["requests"])]
        return held, [h + 1 if i % 3 == 0 else r.randint(1, case["longest"]) if i % 3 == 1 else 0 for i, h in enumerate(held)]
    held = [r.randint(1, case["longest"] - 1) for i in range(case["requests"])]
    return held, [0 if i % 50 == 49 else h + 1 for i, h in enumerate(held)]


def _random(seed, device="cuda"):
    return torch.Generator(device=device).manual_seed(seed)


def prepare(case, seed):
    g = _random(seed)
    kind = case["kind"]
    state = {"case": case}
    if kind == "scored":
        b, h, n, d, t = case["batch"], case["heads"], case["kv_heads"], case["dim"], TYPES[case["dtype"]]
        total = case["seq"] + case["past"]
        # the layout that a projection leaves: (batch, tokens, heads, dim), seen as (batch, heads, tokens, dim)
        state["q"] = (torch.randn(b, case["seq"], h, d, generator=g, device="cuda") * 2).to(t).transpose(1, 2)
        state["k"] = torch.randn(b, total, n, d, generator=g, device="cuda").to(t).transpose(1, 2)
        state["v"] = torch.randn(b, total, n, d, generator=g, device="cuda").to(t).transpose(1, 2)
        state["documents"] = _documents(case).cuda() if case["documents"] else None
        state["prefix_lens"] = torch.tensor(_prefix_lens(case), dtype=torch.int32, device="cuda") if case["prefix"] else None
        state["key_lens"] = torch.tensor(_key_lens(case), dtype=torch.int32, device="cuda") if case["padded"] else None
    elif kind == "cache":
        h, n, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
        lengths = torch.tensor(_request_lengths(case), dtype=torch.int32, device="cuda")
        width = -(-case["longest"] // page)
        blocks = (lengths + page - 1) // page
        pages = sum(-(-x // page) for x in _request_lengths(case)) + 7
        order = torch.randperm(pages, generator=g, device="cuda").int()
        start = (blocks.cumsum(0) - blocks).unsqueeze(1)
        at = torch.arange(width, device="cuda").unsqueeze(0)
        state["block_table"] = torch.where(at < blocks.unsqueeze(1), order[(start + at).clamp(max=pages - 1)], 0).int()
        state["lengths"] = lengths
        spread, most = (32.0, 127.0) if case["cache"] == "int8" else (110.0, 448.0)
        state["k_pages"] = (torch.randn(pages, n, page, d, generator=g, device="cuda") * spread).clamp_(-most, most).round_().to(TYPES[case["cache"]])
        state["v_pages"] = (torch.randn(pages, n, page, d, generator=g, device="cuda") * spread).clamp_(-most, most).round_().to(TYPES[case["cache"]])
        state["k_scales"] = (torch.rand(pages, n, generator=g, device="cuda") + 0.5) / spread
        state["v_scales"] = (torch.rand(pages, n, generator=g, device="cuda") + 0.5) / spread
        state["q"] = (torch.randn(case["requests"], case["tokens"], h, d, generator=g, device="cuda") * 2).to(TYPES[case["dtype"]])
    elif kind == "append":
        n, d, page, r = case["kv_heads"], case["dim"], case["page"], case["requests"]
        width = -(-(case["held"] + case["new"]) // page)
        pages = r * width + 5
        table = torch.randperm(pages, generator=g, device="cuda")[:r * width].view(r, width)
        at = case["held"] + torch.arange(case["new"], device="cuda")
        state["slots"] = (table[:, at // page] * page + at % page).view(-1).int()
        state["k_pages"] = (torch.randn(pages, n, page, d, generator=g, device="cuda") * 110).clamp_(-448, 448).to(torch.float8_e4m3fn)
        state["v_pages"] = (torch.randn(pages, n, page, d, generator=g, device="cuda") * 110).clamp_(-448, 448).to(torch.float8_e4m3fn)
        state["k_scales"] = (torch.rand(pages, n, generator=g, device="cuda") + 0.5) / 110
        state["v_scales"] = (torch.rand(pages, n, generator=g, device="cuda") + 0.5) / 110
        # keys and values as slices of one projection's rows
        kv = torch.randn(r * case["new"], 2, n, d, generator=g, device="cuda").to(TYPES[case["dtype"]])
        state["k"], state["v"] = kv[:, 0], kv[:, 1]
    else:
        held, lengths = _held_and_lengths(case)
        page, r = case["page"], case["requests"]
        width = -(-case["longest"] // page) + 1
        have = torch.tensor([-(-x // page) for x in held], device="cuda")
        pages = r * width
        order = torch.randperm(pages, generator=g, device="cuda").int()
        start = (have.cumsum(0) - have).unsqueeze(1)
        at = torch.arange(width, device="cuda").unsqueeze(0)
        used = sum(-(-x // page) for x in held)
        state["block_table"] = torch.where(at < have.unsqueeze(1), order[(start + at).clamp(max=pages - 1)], -1).int()
        state["free_pages"] = torch.cat((order[used:], torch.zeros(used, dtype=torch.int32, device="cuda")))
        state["free_count"] = torch.tensor([pages - used], dtype=torch.int32, device="cuda")
        state["held"] = torch.tensor(held, dtype=torch.int32, device="cuda")
        state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        state["new_tokens"] = sum(max(0, b - a) for a, b in zip(held, lengths))
    bias = case.get("bias", "")
    state["slopes"] = torch.exp2(-8.0 * torch.arange(1, case["heads"] + 1, device="cuda") / case["heads"]) if bias == "slopes" else None
    state["distance_bias"] = torch.randn(case["heads"], 2 * TABLE_RADIUS + 1, generator=g, device="cuda") if bias == "table" else None
    return state


# ------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------
def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"scored": _scored_own, "cache": _cache_own, "append": _append_own, "tables": _tables_own}[kind](state, state["case"])
    return {"scored": _scored, "cache": _cache, "append": _append, "tables": _tables}[kind](state, state["case"])


@functools.cache
def _framework():
    sys.path.insert(0, os.path.join(os.getcwd(), "sc25-stof-ad_b200"))
    import stof_b200
    return stof_b200


def _scored_own(s, c):
    return _framework().scored_attention(s["q"], s["k"], s["v"], causal=c["causal"], window=c["window"] or None, softcap=c["softcap"] or None,
                                         slopes=s["slopes"], distance_bias=s["distance_bias"], documents=s["documents"], prefix_lens=s["prefix_lens"],
                                         key_lens=s["key_lens"])


def _cache_own(s, c):
    return _framework().cache_attention(s["q"], s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"], s["block_table"], s["lengths"],
                                        window=c["window"] or None, softcap=c["softcap"] or None, slopes=s["slopes"], distance_bias=s["distance_bias"])


def _append_own(s, c):
    _framework().cache_append(s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"], s["k"], s["v"], s["slots"])
    return s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"]


def _tables_own(s, c):
    slots, starts, free_count, missing = _framework().page_tables(s["lengths"], s["held"], s["block_table"], s["free_pages"], s["free_count"], c["page"],
                                                                  s["new_tokens"])
    return s["block_table"], slots, starts, s["free_pages"], free_count, missing


def _changed(x, distance, s, c):
    """Cap and bias: x (..., heads, queries, keys), distance = key position - query position, broadcastable to x without its heads."""
    if c["softcap"]:
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    if s["slopes"] is not None:
        x = x - s["slopes"].view(-1, 1, 1) * distance.abs().unsqueeze(-3)
    if s["distance_bias"] is not None:
        at = distance.clamp(-TABLE_RADIUS, TABLE_RADIUS) + TABLE_RADIUS
        x = x + s["distance_bias"][:, at].movedim(0, -3)
    return x


def _attend(x, visible, v):
    """softmax over the visible keys, times v; rows without any give zeros.  x (batch, heads, queries, keys), v (batch, kv heads, keys, dim)"""
    x = x.masked_fill(~visible, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    b, h, q, n = p.shape
    o = torch.matmul(p.view(b, v.shape[1], -1, n), v).view(b, h, q, -1)
    return torch.where(total > 0, o / total, 0.0)


def _scores(q, k):
    """(batch, heads, queries, dim) x (batch, kv heads, keys, dim) -> scaled products, heads sharing a K/V head side by side"""
    b, h, n, d = q.shape
    return torch.matmul(q.reshape(b, k.shape[1], -1, d) * d ** -0.5, k.transpose(-1, -2)).view(b, h, n, -1)


def _scored(s, c):
    pos = torch.arange(c["past"], c["past"] + c["seq"], device="cuda")
    key = torch.arange(c["past"] + c["seq"], device="cuda")
    distance = key.unsqueeze(0) - pos.unsqueeze(1)
    x = _changed(_scores(s["q"].float(), s["k"].float()), distance, s, c)
    visible = distance <= 0 if c["causal"] else torch.ones_like(distance, dtype=torch.bool)
    if c["window"]:
        visible = visible & (distance.abs() < c["window"])
    visible = visible.expand(c["batch"], -1, -1)
    if c["prefix"]:
        visible = visible | (key < s["prefix_lens"].view(-1, 1, 1))
    if c["documents"]:
        visible = visible & (s["documents"][:, c["past"]:].unsqueeze(2) == s["documents"].unsqueeze(1))
    if c["padded"]:
        visible = visible & (key < s["key_lens"].view(-1, 1, 1))
    return _attend(x, visible.unsqueeze(1), s["v"].float()).to(s["q"].dtype)


def _cache(s, c):
    b, width, page, d = c["requests"], s["block_table"].shape[1], c["page"], c["dim"]
    at = s["block_table"].long()
    k = (s["k_pages"].view(torch.int8)[at].view(s["k_pages"].dtype).float() * s["k_scales"][at][..., None, None]).transpose(1, 2).reshape(b, -1, width * page, d)
    v = (s["v_pages"].view(torch.int8)[at].view(s["v_pages"].dtype).float() * s["v_scales"][at][..., None, None]).transpose(1, 2).reshape(b, -1, width * page, d)
    key = torch.arange(width * page, device="cuda")
    pos = s["lengths"].view(-1, 1) - c["tokens"] + torch.arange(c["tokens"], device="cuda")
    distance = key - pos.unsqueeze(2)
    x = _changed(_scores(s["q"].float().transpose(1, 2), k), distance, s, c)
    visible = distance <= 0
    if c["window"]:
        visible = visible & (distance > -c["window"])
    return _attend(x, visible.unsqueeze(1), v).transpose(1, 2).to(s["q"].dtype)


def _append(s, c):
    page, slots = c["page"], s["slots"].long()
    first = slots % page == 0
    first[0] = True
    first[1:] |= slots[1:] != slots[:-1] + 1
    run_of = first.long().cumsum(0) - 1                          # tokens of consecutive slots inside a page
    lead = slots[first.nonzero().view(-1)]
    in_page, before = lead // page, lead % page
    live = (torch.arange(page, device="cuda") < before.view(-1, 1)).view(-1, 1, page, 1)

    def write(pages, scales, x):
        x = x.float()
        top = torch.zeros(lead.numel(), x.shape[1], device="cuda").scatter_reduce_(0, run_of.view(-1, 1).expand(-1, x.shape[1]), x.abs().amax(-1), "amax")
        old = scales[in_page]
        new = top * (1 / 448.0)
        new = torch.where(before.view(-1, 1) > 0, torch.maximum(new, old), new)
        grown = (before.view(-1, 1) > 0) & (new > old)
        raw = pages.view(torch.uint8)
        was = raw[in_page]
        again = (was.view(pages.dtype).float() * (old / new)[..., None, None]).to(pages.dtype).view(torch.uint8)
        raw[in_page] = torch.where(live & grown[..., None, None], again, was)
        scales[in_page] = new
        factor = torch.where(new > 0, 1 / new, 0.0)[run_of].unsqueeze(-1)
        raw[slots // page, :, slots % page] = (x * factor).clamp(-448, 448).to(pages.dtype).view(torch.uint8)

    write(s["k_pages"], s["k_scales"], s["k"])
    write(s["v_pages"], s["v_scales"], s["v"])
    return s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"]


def _tables(s, c):
    page, table, stack, n = c["page"], s["block_table"], s["free_pages"], s["free_count"]
    width, room = table.shape[1], stack.numel()
    need, have = (s["lengths"].long() + page - 1) // page, (s["held"].long() + page - 1) // page
    take, give = (need - have).clamp(min=0), (have - need).clamp(min=0)
    top = n + give.sum()
    missing = (take.sum() - top).clamp(min=0) + (need - width).clamp(min=0).sum()
    good = missing == 0
    at = torch.arange(width, device="cuda").unsqueeze(0)
    gives = good & (at >= need.unsqueeze(1)) & (at < have.unsqueeze(1))
    to = n + (give.cumsum(0) - give - need).unsqueeze(1) + at
    stack.copy_(torch.cat((stack, stack[:1])).scatter_(0, torch.where(gives, to, room).view(-1), table.reshape(-1))[:room])
    takes = good & (at >= have.unsqueeze(1)) & (at < need.unsqueeze(1))
    come = top - 1 - ((take.cumsum(0) - take - have).unsqueeze(1) + at)
    table.copy_(torch.where(takes, stack[come.clamp(0, room - 1)], table))
    new = (s["lengths"] - s["held"]).long().clamp(min=0)
    starts = torch.cat((torch.zeros(1, dtype=torch.long, device="cuda"), new.cumsum(0)))
    t = torch.arange(s["new_tokens"], device="cuda")
    r = torch.searchsorted(starts[1:].contiguous(), t, right=True).clamp(max=new.numel() - 1)
    pos = s["held"][r] + t - starts[r]
    slots = torch.where(good & (t < starts[-1]), table[r, (pos // page).clamp(max=width - 1)].long() * page + pos % page, -1)
    left = torch.where(good, top - take.sum(), n.long())
    return table, slots.int(), starts.int(), stack, left.int(), missing.int()


# ------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "scored":
        total = case["seq"] + case["past"]
        pos, key = torch.arange(case["past"], total).unsqueeze(1), torch.arange(total).unsqueeze(0)
        pairs = 0
        for b in range(case["batch"]):
            on = torch.ones(case["seq"], total, dtype=torch.bool)
            if case["causal"]:
                on &= key <= pos
            if case["window"]:
                on &= (key - pos).abs() < case["window"]
            if case["prefix"]:
                on |= key < _prefix_lens(case)[b]
            if case["documents"]:
                doc = _documents(case)[b]
                on &= doc[case["past"]:].unsqueeze(1) == doc.unsqueeze(0)
            if case["padded"]:
                on &= key < _key_lens(case)[b]
            pairs += int(on.sum())
        moved = 2 * case["batch"] * case["dim"] * (2 * case["heads"] * case["seq"] + 2 * case["kv_heads"] * total)
        return {"bytes": moved, "flops": 4.0 * case["dim"] * case["heads"] * pairs}
    if kind == "cache":
        n, pairs, keys, blocks = case["tokens"], 0, 0, 0
        for length in _request_lengths(case):
            seen = min(length, case["window"] + n - 1) if case["window"] else length
            keys += seen
            blocks += -(-seen // case["page"])
            pairs += sum(min(length - n + t + 1, case["window"] or length) for t in range(n))
        moved = 2 * keys * case["kv_heads"] * case["dim"] + blocks * (8 * case["kv_heads"] + 4) + 4 * case["requests"] * (n * case["heads"] * case["dim"] + 1)
        return {"bytes": moved, "flops": 4.0 * case["dim"] * case["heads"] * pairs}
    if kind == "append":
        tokens = case["requests"] * case["new"]
        touched = case["requests"] * (-(-(case["held"] + case["new"]) // case["page"]) - case["held"] // case["page"])
        return {"bytes": tokens * (6 * case["kv_heads"] * case["dim"] + 4) + 16 * touched * case["kv_heads"], "flops": 8.0 * tokens * case["kv_heads"] * case["dim"]}
    held, lengths = _held_and_lengths(case)
    moves = sum(abs(-(-a // case["page"]) + (-b // case["page"])) for a, b in zip(held, lengths))
    fresh = sum(max(0, b - a) for a, b in zip(held, lengths))
    # a request's two lengths and its start, a page's way from or to the stack, the slots
    return {"bytes": 12 * case["requests"] + 8 * moves + 4 * fresh + 16, "flops": 0}


# ------------------------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ------------------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    return {"scored": _scored_exact, "cache": _cache_exact, "append": _append_exact, "tables": lambda s, c: None}[case["kind"]](state, case)


def _row_exact(q, k, v, pos, head, s, c, seen):
    """One head of one sequence: q (n, dim) at positions pos, k and v (m, dim), seen (n, m)."""
    x = q.double() @ k.double().T / math.sqrt(c["dim"])
    away = torch.arange(k.shape[0], device="cuda")[None] - pos[:, None]
    if c["softcap"] > 0:
        x = torch.tanh(x / c["softcap"]) * c["softcap"]
    if c["bias"] == "slopes":
        x = x - s["slopes"][head].double() * away.abs().double()
    if c["bias"] == "table":
        radius = s["distance_bias"].shape[1] // 2
        x = x + s["distance_bias"][head].double()[(away + radius).clamp(0, 2 * radius)]
    x[~seen] = -math.inf
    some = seen.any(1)
    out = torch.zeros(q.shape[0], c["dim"], dtype=torch.float64, device="cuda")
    out[some] = torch.softmax(x[some], 1) @ v.double()
    return out


def _scored_exact(s, c):
    total, group = c["seq"] + c["past"], c["heads"] // c["kv_heads"]
    if c["batch"] * c["heads"] * c["seq"] * total > 3e9:
        return None
    pos, key = torch.arange(c["past"], total, device="cuda"), torch.arange(total, device="cuda")
    out = torch.empty(c["batch"], c["heads"], c["seq"], c["dim"], dtype=torch.float64, device="cuda")
    for b in range(c["batch"]):
        seen = torch.full((c["seq"], total), True, device="cuda")
        if c["causal"]:
            seen.tril_(c["past"])
        if c["window"]:
            seen &= torch.ones_like(seen).triu_(c["past"] - c["window"] + 1) & torch.ones_like(seen).tril_(c["past"] + c["window"] - 1)
        if c["prefix"]:
            seen[:, :int(s["prefix_lens"][b])] = True
        if c["padded"]:
            seen[:, int(s["key_lens"][b]):] = False
        if c["documents"]:
            seen &= s["documents"][b][pos][:, None] == s["documents"][b][key][None]
        for h in range(c["heads"]):
            out[b, h] = _row_exact(s["q"][b, h], s["k"][b, h // group], s["v"][b, h // group], pos, h, s, c, seen)
    return out


def _cache_exact(s, c):
    if sum(_request_lengths(c)) * c["heads"] * c["tokens"] > 2e8 or c["requests"] * c["heads"] > 4096:
        return None
    n, group = c["tokens"], c["heads"] // c["kv_heads"]
    out = torch.empty(c["requests"], n, c["heads"], c["dim"], dtype=torch.float64, device="cuda")
    for b, length in enumerate(s["lengths"].tolist()):
        pages = s["block_table"][b, :-(-length // c["page"])].long()
        k = s["k_pages"].view(torch.int8)[pages].view(s["k_pages"].dtype).double() * s["k_scales"][pages].double()[:, :, None, None]
        v = s["v_pages"].view(torch.int8)[pages].view(s["v_pages"].dtype).double() * s["v_scales"][pages].double()[:, :, None, None]
        pos = torch.arange(length - n, length, device="cuda")
        away = pos[:, None] - torch.arange(length, device="cuda")[None]
        seen = (away >= 0) & (away < (c["window"] or length))
        for h in range(c["heads"]):
            one = (k[:, h // group].reshape(-1, c["dim"])[:length], v[:, h // group].reshape(-1, c["dim"])[:length])
            out[b, :, h] = _row_exact(s["q"][b, :, h], *one, pos, h, s, c, seen)
    return out


def _append_exact(s, c):
    page, slots, out = c["page"], s["slots"].tolist(), []
    runs, begin = [], 0
    for t in range(1, len(slots) + 1):
        if t == len(slots) or slots[t] != slots[t - 1] + 1 or slots[t] % page == 0:
            runs.append((begin, t))
            begin = t
    for pages, scales, x in ((s["k_pages"], s["k_scales"], s["k"]), (s["v_pages"], s["v_scales"], s["v"])):
        values, scale = pages.double(), scales.double()
        for a, b in runs:
            p, o = slots[a] // page, slots[a] % page
            rows = x[a:b].double().transpose(0, 1)                                # (heads, tokens, dim)
            need = rows.abs().amax((1, 2)) / 448
            if o > 0:
                kept = torch.maximum(need, scale[p])
                grown = (kept > scale[p])[:, None, None]
                front = values[p, :, :o]
                values[p, :, :o] = torch.where(grown, (front * (scale[p] / kept)[:, None, None]).to(torch.float8_e4m3fn).double(), front)
                need = kept
            scale[p] = need
            values[p, :, o:o + b - a] = (rows / need[:, None, None]).clamp(-448, 448).to(torch.float8_e4m3fn).double()
        out.append((values, scale))
    return out[0][0], out[1][0], out[0][1], out[1][1]
