"""A serving batch whose requests share prompts, operator by operator: the step's page tables, its attention over shared
prefixes, and the adjustments of its scores before a token is drawn.

``tables``     positions, sequence numbers, cache slots and block tables of a step from the requests' lengths;
``attention``  queries over a paged cache in which the requests of a group have their first keys in common;
``logits``     repeat, presence and frequency penalties, biases and allowed-token masks on rows of scores.

Lengths come from the case alone (``lengths`` seeds them), everything else from the seed.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
HEADS = ((24, 2), (36, 4), (48, 4), (16, 4), (16, 16), (8, 1))      # query heads on KV heads, of this repository's configurations


def listed():
    return [
        # eight chats decoding, contexts of the stock limit of 4,096: launch time
        {"name": "tables of 8 decoding", "op": "tables", "seqs": 8, "portions": 0, "portion": 1, "page": 16, "context": 4096,
         "shared": 0, "window": 0, "lengths": 1},
        # a step of a server under load: decoding requests, some of one system prompt, and prompt portions of 512
        {"name": "tables of 61 and 3 portions", "op": "tables", "seqs": 64, "portions": 3, "portion": 512, "page": 32,
         "context": 16384, "shared": 1024, "window": 4096, "lengths": 2},
        # offline generation: 1,024 requests, long contexts, a table of 4 thousand entries a request
        {"name": "tables of 1024 long", "op": "tables", "seqs": 1024, "portions": 0, "portion": 1, "page": 16,
         "context": 65536, "shared": 2048, "window": 0, "lengths": 3},
        # a few chats that just began under one system prompt
        {"name": "attention of 4", "op": "attention", "seqs": 4, "groups": 1, "portion": 1, "shared": 512, "own": 64,
         "heads": 24, "kv_heads": 2, "dim": 128, "page": 16, "window": 0, "dtype": "bfloat16", "lengths": 4},
        # an assistant's system prompt and tool descriptions, under the sliding window of the 7B sizes
        {"name": "attention of 32, window", "op": "attention", "seqs": 32, "groups": 1, "portion": 1, "shared": 2048,
         "own": 3000, "heads": 36, "kv_heads": 4, "dim": 128, "page": 16, "window": 4096, "dtype": "bfloat16", "lengths": 5},
        # many questions about one long document
        {"name": "attention of 128 on 32k", "op": "attention", "seqs": 128, "groups": 1, "portion": 1, "shared": 32768,
         "own": 2048, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "window": 0, "dtype": "bfloat16", "lengths": 6},
        # the first step after admission: each request brings the rest of its own prompt; three prefixes, small heads
        {"name": "attention of 12 portions", "op": "attention", "seqs": 12, "groups": 3, "portion": 40, "shared": 2500,
         "own": 500, "heads": 16, "kv_heads": 4, "dim": 64, "page": 8, "window": 0, "dtype": "bfloat16", "lengths": 7},
        # the 32-bit path
        {"name": "attention of 24 in float", "op": "attention", "seqs": 24, "groups": 2, "portion": 1, "shared": 1500,
         "own": 300, "heads": 24, "kv_heads": 2, "dim": 128, "page": 16, "window": 0, "dtype": "float32", "lengths": 8},
        # one chat
        {"name": "logits of 1", "op": "logits", "rows": 1, "vocab": 32768, "tokens": 200, "biases": 4, "masked": 0.0,
         "allowed": 1.0, "dtype": "float32", "lengths": 9},
        # a server's step, half of the requests under a grammar
        {"name": "logits of 64", "op": "logits", "rows": 64, "vocab": 49152, "tokens": 2048, "biases": 32, "masked": 0.5,
         "allowed": 0.5, "dtype": "float32", "lengths": 10},
        # scores as a 16-bit head leaves them
        {"name": "logits of 24 in bfloat16", "op": "logits", "rows": 24, "vocab": 65537, "tokens": 500, "biases": 300,
         "masked": 0.25, "allowed": 0.1, "dtype": "bfloat16", "lengths": 11},
        # structured output offline: every row masked, long histories, a vocabulary that no vector width divides
        {"name": "logits of 256", "op": "logits", "rows": 256, "vocab": 131071, "tokens": 8192, "biases": 16, "masked": 1.0,
         "allowed": 0.3, "dtype": "float32", "lengths": 12},
    ]


def draw(rng):
    def span(low, high):                       # over the logarithm
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    case = {"op": rng.choice(("tables", "attention", "attention", "logits")), "lengths": rng.randrange(1 << 20)}
    if case["op"] == "tables":
        case["seqs"] = span(1, 1024)
        case["portions"] = rng.choice((0, 0, 1, min(case["seqs"], 5)))
        case["portion"] = span(2, 1024) if case["portions"] else 1
        case["page"] = rng.choice((8, 16, 32))
        case["context"] = span(64, 65536)
        case["shared"] = rng.choice((0, span(8, max(8, case["context"] // 2))))
        case["window"] = rng.choice((0, 0, span(16, 8192)))
    elif case["op"] == "attention":
        case["seqs"] = span(1, 128)
        case["groups"] = min(case["seqs"], rng.choice((1, 1, 2, 5)))
        case["portion"] = rng.choice((1, 1, 1, 2, 17, 60)) if case["seqs"] <= 32 else 1
        case["heads"], case["kv_heads"] = rng.choice(HEADS)
        case["dim"] = rng.choice((128, 128, 128, 64, 80))
        case["page"] = rng.choice((8, 16, 16, 32))
        case["window"] = rng.choice((0, 0, 0, span(100, 8192)))
        case["dtype"] = rng.choice(("bfloat16", "bfloat16", "bfloat16", "float32"))
        case["shared"] = span(8, 4096 if case["dtype"] == "float32" or case["portion"] > 1 else 16384)
        case["own"] = span(1, 400 if case["dtype"] == "float32" else 900)
    else:
        case["rows"] = span(1, 256)
        case["vocab"] = span(1000, 131071)
        case["tokens"] = rng.choice((0, span(1, 8192)))
        case["biases"] = rng.choice((0, span(1, 300)))
        case["masked"] = rng.choice((0.0, 0.5, 1.0))
        case["allowed"] = rng.choice((0.01, 0.3, 0.9))
        case["dtype"] = rng.choice(("float32", "float32", "bfloat16"))
    return case


# ------------------------------------------------------------------------------------------ lengths, from the case alone
def _tables_lengths(case):
    r = np.random.RandomState(case["lengths"])
    n, page = case["seqs"], case["page"]
    shared_pages = case["shared"] // page
    context = np.minimum(np.exp(r.uniform(0, math.log(case["context"]), n)).astype(np.int64), case["context"])
    joins = np.zeros(n, bool) if shared_pages == 0 else r.rand(n) < 0.5
    if shared_pages:
        joins[0] = False                        # the first request holds the prefix's pages
        context[0] = max(context[0], shared_pages * page)
    context = np.where(joins, np.maximum(context, shared_pages * page), context)
    q = np.ones(n, np.int64)
    q[n - case["portions"]:] = r.randint(1, case["portion"] + 1, case["portions"])
    width = -(-int((context + q).max()) // page) + 1
    return context, q, joins, shared_pages, width


def _attention_lengths(case):
    """Tokens that each request brings, keys of its own before them, the requests of each group, its prefix."""
    r = np.random.RandomState(case["lengths"])
    n, g = case["seqs"], case["groups"]
    q = r.randint(1, case["portion"] + 1, n)
    before = r.randint(0, case["own"] + 1, n)
    cuts = np.sort(r.choice(np.arange(1, n), g - 1, replace=False)) if g > 1 else np.zeros(0, np.int64)
    first = np.concatenate([[0], cuts, [n]])
    pages = np.maximum(1, (case["shared"] * r.uniform(0.5, 1.0, g) if g > 1 else np.full(g, case["shared"])) // case["page"])
    return q, before, first.astype(np.int64), (pages * case["page"]).astype(np.int64)


def _seen(case):
    """Per token, the keys of the prefix and of its own that it sees; per group and per request, the keys that any sees."""
    q, before, first, shared = _attention_lengths(case)
    prefix_of = np.repeat(shared, np.diff(first))
    position = np.concatenate([p + b + np.arange(k) for p, b, k in zip(prefix_of, before, q)])
    seq = np.repeat(np.arange(len(q)), q)
    low = np.maximum(0, position - case["window"] + 1) if case["window"] else np.zeros_like(position)
    in_prefix = np.maximum(0, prefix_of[seq] - low)
    in_own = position + 1 - np.maximum(low, prefix_of[seq])
    group = np.repeat(np.arange(len(shared)), np.diff(first))[seq]
    union_prefix = np.array([in_prefix[group == i].max() for i in range(len(shared))])
    union_own = np.array([(prefix_of[s] + before[s] + q[s]) - max(prefix_of[s], low[seq == s].min()) for s in range(len(q))])
    return in_prefix, in_own, union_prefix, union_own


def _logits_lengths(case):
    r = np.random.RandomState(case["lengths"])
    rows = case["rows"]
    tokens = r.randint(case["tokens"] // 2, case["tokens"] + 1, rows)
    biases = r.randint(case["biases"] // 2, case["biases"] + 1, rows)
    masked = np.arange(rows) < round(case["masked"] * rows)
    return tokens, biases, masked


def work(case):
    if case["op"] == "tables":
        context, q, joins, shared_pages, width = _tables_lengths(case)
        page = case["page"]
        used = -(-(context + q) // page)
        taken = int((used - -(-context // page)).sum())
        reads = 5 * 4 * case["seqs"] + 4 * int(used.sum())
        writes = 4 * (case["seqs"] * width + 3 * int(q.sum()) + case["seqs"] + taken)
        return {"bytes": reads + writes, "flops": 0}
    if case["op"] == "attention":
        in_prefix, in_own, union_prefix, union_own = _seen(case)
        width = 2 if case["dtype"] == "bfloat16" else 4
        keys = int(union_prefix.sum() + union_own.sum())
        rows = len(in_prefix) * case["heads"] * case["dim"]
        return {"bytes": width * (2 * keys * case["kv_heads"] * case["dim"] + 2 * rows),
                "flops": 4 * case["dim"] * case["heads"] * int(in_prefix.sum() + in_own.sum())}
    tokens, biases, masked = _logits_lengths(case)
    width = 2 if case["dtype"] == "bfloat16" else 4
    read = float((np.where(masked, case["allowed"], 1.0) * case["vocab"] * width).sum())     # masked scores need not be read
    return {"bytes": read + 4 * case["rows"] * case["vocab"] + 4 * int(tokens.sum()) + 8 * int(biases.sum())
            + int(masked.sum()) * (case["vocab"] + 31) // 32 * 4, "flops": 4 * case["rows"] * case["vocab"]}


# ------------------------------------------------------------------------------------------------------------- inputs
def _ints(values):
    return torch.from_numpy(np.ascontiguousarray(values, dtype=np.int32)).to(DEVICE)


def prepare(case, seed):
    return {"tables": _prepare_tables, "attention": _prepare_attention, "logits": _prepare_logits}[case["op"]](case, seed)


def _prepare_tables(case, seed):
    r = np.random.RandomState(seed % (1 << 32))
    context, q, joins, shared_pages, width = _tables_lengths(case)
    n, page = case["seqs"], case["page"]
    have = -(-context // page)
    need = -(-(context + q) // page) - have
    n_rows = n + 3
    rows = r.permutation(n_rows)[:n]
    held = int((have - np.where(joins, shared_pages, 0)).sum())
    n_pages = held + int(need.sum()) + 64
    pages = r.permutation(n_pages).astype(np.int32)
    tables = np.full((n_rows, width), -1, np.int32)
    at = 0
    for s in range(n):
        begin = shared_pages if joins[s] else 0
        count = int(have[s]) - begin
        tables[rows[s], begin:begin + count] = pages[at:at + count]
        at += count
    total = int(q.sum())
    return {"case": case, "q_lens": _ints(q), "context_lens": _ints(context), "rows": _ints(rows), "tables": _ints(tables),
            "free_pages": _ints(pages[at:]), "n_free": _ints([n_pages - at]), "n_pages": n_pages,
            "shared_rows": _ints(np.where(joins, rows[0], -1)), "shared_pages": _ints(np.where(joins, shared_pages, 0)),
            "n_tokens": -(-total // 8) * 8, "status": _ints([0])}


def _prepare_attention(case, seed):
    r = np.random.RandomState(seed % (1 << 32))
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = getattr(torch, case["dtype"])
    q_lens, before, first, shared = _attention_lengths(case)
    page, dim, heads, kv_heads = case["page"], case["dim"], case["heads"], case["kv_heads"]
    prefix_of = np.repeat(shared, np.diff(first))
    context = prefix_of + before
    total = -(-(context + q_lens) // page)
    n_pages = int((shared // page).sum() + (total - prefix_of // page).sum()) + 5
    pages = r.permutation(n_pages)
    tables = np.full((len(q_lens), int(total.max())), -1, np.int64)
    at = 0
    for g in range(len(shared)):
        count = int(shared[g]) // page
        tables[first[g]:first[g + 1], :count] = pages[at:at + count]
        at += count
    for s in range(len(q_lens)):
        begin, end = int(prefix_of[s]) // page, int(total[s])
        tables[s, begin:end] = pages[at:at + end - begin]
        at += end - begin
    n = int(q_lens.sum())
    # keys of unit-variance numbers, queries somewhat larger: a softmax that prefers some keys
    cache = torch.randn(n_pages, 2, kv_heads, page, dim, generator=gen, device=DEVICE).to(dtype)
    q = (1.5 * torch.randn(n, heads * dim, generator=gen, device=DEVICE)).to(dtype)
    return {"case": case, "q": q, "cache": cache, "block_tables": _ints(tables), "cu_q": _ints(np.concatenate([[0], np.cumsum(q_lens)])),
            "context_lens": _ints(context), "tok_seq": _ints(np.repeat(np.arange(len(q_lens)), q_lens)),
            "positions": _ints(np.concatenate([c + np.arange(k) for c, k in zip(context, q_lens)])),
            "shared_first": _ints(first), "shared_lens": _ints(prefix_of), "n_tokens": n, "max_q_len": int(q_lens.max()),
            "max_shared_len": int(shared.max()), "max_own_len": int((before + q_lens).max()),
            "max_group_tokens": int(np.add.reduceat(q_lens, first[:-1]).max()), "status": _ints([0])}


def _prepare_logits(case, seed):
    r = np.random.RandomState(seed % (1 << 32))
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    rows, vocab = case["rows"], case["vocab"]
    tokens, biases, masked = _logits_lengths(case)
    ids = np.minimum(vocab - 1, (vocab * r.rand(int(tokens.sum())) ** 4).astype(np.int64))        # frequent tokens repeat
    bias_ids = [r.choice(vocab, int(k), replace=False) for k in biases]
    words = (vocab + 31) // 32
    bits = torch.rand(max(1, int(masked.sum())), words * 32, generator=gen, device=DEVICE) < case["allowed"]
    weights = torch.ones(32, dtype=torch.int64, device=DEVICE) << torch.arange(32, device=DEVICE)
    packed = (bits.view(-1, words, 32) * weights).sum(-1)
    packed = (packed - ((packed >> 31) << 32)).to(torch.int32)
    return {"case": case, "logits": (4 * torch.randn(rows, vocab, generator=gen, device=DEVICE)).to(getattr(torch, case["dtype"])),
            "token_offsets": _ints(np.concatenate([[0], np.cumsum(tokens)])), "token_ids": _ints(ids),
            "repeat": torch.from_numpy(r.uniform(1.0, 1.5, rows).astype(np.float32)).to(DEVICE),
            "presence": torch.from_numpy(r.uniform(0.0, 1.0, rows).astype(np.float32)).to(DEVICE),
            "frequency": torch.from_numpy(r.uniform(0.0, 0.3, rows).astype(np.float32)).to(DEVICE),
            "bias_offsets": _ints(np.concatenate([[0], np.cumsum(biases)])),
            "bias_ids": _ints(np.concatenate(bias_ids + [np.zeros(0, np.int64)])),
            "bias_values": torch.from_numpy(r.normal(0, 5, int(biases.sum())).astype(np.float32)).to(DEVICE),
            "mask_words": packed, "mask_rows": _ints(np.where(masked, np.cumsum(masked) - 1, -1)),
            "pending": _ints(np.where(r.rand(rows) < 0.5, r.randint(0, vocab, rows), -1))}


# ------------------------------------------------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return {"tables": _own_tables, "attention": _own_attention, "logits": _own_logits}[op](state)
    return {"tables": _plain_tables, "attention": _plain_attention, "logits": _plain_logits}[op](state)


def _own_tables(s):
    from matricxon_b200.ops import kernels

    n, tokens, width = s["q_lens"].numel(), s["n_tokens"], s["tables"].shape[1]

    def ints(*shape):
        return torch.empty(shape, dtype=torch.int32, device=s["q_lens"].device)

    positions, tok_seq, slots, cu_q, taken, block_tables = ints(tokens), ints(tokens), ints(tokens), ints(n + 1), ints(1), ints(n, width)
    kernels.step_tables(s["q_lens"], s["context_lens"], s["rows"], s["tables"], s["free_pages"], s["n_free"], s["case"]["page"],
                        s["n_pages"], positions, tok_seq, cu_q, slots, block_tables, taken, s["status"],
                        shared_rows=s["shared_rows"], shared_pages=s["shared_pages"], window=s["case"]["window"])
    return {"positions": positions, "tok_seq": tok_seq, "cu_q": cu_q, "slots": slots, "block_tables": block_tables, "taken": taken,
            "tables": s["tables"]}


def _plain_tables(s):
    page, width, n_tok = s["case"]["page"], s["tables"].shape[1], s["n_tokens"]
    q, context, rows = s["q_lens"].long(), s["context_lens"].long(), s["rows"].long()
    shared_rows, shared_pages = s["shared_rows"].long(), s["shared_pages"].long()
    have = (context + page - 1) // page
    end = (context + q + page - 1) // page
    cu = torch.cat([q.new_zeros(1), q.cumsum(0)])
    base = (end - have).cumsum(0) - (end - have)
    k = torch.arange(width, device=q.device)
    mine = s["tables"][rows].long()
    fresh = (base[:, None] + k - have[:, None]).clamp(0, max(0, s["free_pages"].numel() - 1))
    is_new = (k >= have[:, None]) & (k < end[:, None])
    mine = torch.where(is_new, s["free_pages"].long()[fresh], mine)
    s["tables"][rows] = mine.to(torch.int32)                       # the same entries whenever it is called
    full = torch.where(k < shared_pages[:, None], s["tables"][shared_rows.clamp_min(0)].long(), mine)
    visible = k < end[:, None]
    if s["case"]["window"]:
        visible &= k >= ((context - s["case"]["window"] + 1).clamp_min(0) // page)[:, None]
    full = torch.where(visible, full, -1)
    row = torch.arange(n_tok, device=q.device)
    seq = torch.searchsorted(cu[1:].contiguous(), row, right=True)
    real = row < cu[-1]
    at = seq.clamp_max(q.numel() - 1)
    position = torch.where(real, context[at] + row - cu[at], 0)
    slot = mine[at, position // page] * page + position % page
    i32 = torch.int32
    return {"positions": position.to(i32), "tok_seq": torch.where(real, seq, -1).to(i32), "cu_q": cu.to(i32),
            "slots": torch.where(real, slot, -1).to(i32), "block_tables": full.to(i32), "taken": (end - have).sum().view(1).to(i32),
            "tables": s["tables"]}


def _own_attention(s):
    from matricxon_b200.ops import kernels

    c = s["case"]
    out = torch.empty_like(s["q"])
    kernels.paged_attention_shared(s["q"], s["q"].stride(0), s["cache"], s["block_tables"], s["cu_q"], s["context_lens"],
                                   s["tok_seq"], s["positions"], s["shared_first"], s["shared_lens"], s["n_tokens"], c["heads"],
                                   c["kv_heads"], c["dim"], c["window"], c["dim"] ** -0.5, out, s["status"],
                                   max_q_len=s["max_q_len"], max_shared_len=s["max_shared_len"], max_own_len=s["max_own_len"])
    return out


def _pages_of(s, tables, first, count):
    """Keys and values [tables, count * page, kv heads, dim] in float of ``count`` pages from page ``first`` of every table."""
    c = s["case"]
    k = first[:, None] + torch.arange(count, device=first.device)
    ids = torch.gather(tables, 1, k.clamp_max(tables.shape[1] - 1)).clamp_min(0).long()
    pages = s["cache"][ids]                                           # [tables, count, 2, kv heads, page, dim]
    n, kv_heads, page, dim = tables.shape[0], c["kv_heads"], c["page"], c["dim"]
    keys = pages[:, :, 0].float().permute(0, 1, 3, 2, 4).reshape(n, count * page, kv_heads, dim)
    values = pages[:, :, 1].reshape(n, count, kv_heads, dim, page).float().permute(0, 1, 4, 2, 3).reshape(n, count * page, kv_heads, dim)
    return keys, values


def _plain_attention(s):
    """Scores of every group's tokens on its prefix and of every request's tokens on its own keys, one softmax over both."""
    c = s["case"]
    heads, kv_heads, dim, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    n, n_seq, n_group, per = s["n_tokens"], s["context_lens"].numel(), s["shared_first"].numel() - 1, heads // kv_heads
    first, shared = s["shared_first"].long(), s["shared_lens"].long()
    seq, position = s["tok_seq"].long(), s["positions"].long()
    cu = s["cu_q"].long()
    group_of = torch.searchsorted(first[1:].contiguous(), torch.arange(n_seq, device=seq.device), right=True)
    token = torch.arange(n, device=seq.device)
    group = group_of[seq]
    in_group, in_seq = token - cu[first[group]], token - cu[seq]
    q = s["q"].float().view(n, kv_heads, per, dim) * dim ** -0.5

    def scores(where, index, size, width, keys):
        rows = q.new_zeros(where, width, kv_heads, per, dim).index_put((size, index), q)
        return torch.matmul(rows.permute(0, 2, 1, 3, 4).reshape(where, kv_heads, width * per, dim), keys.permute(0, 2, 3, 1))

    def back(values, index, size, width):
        return values.view(-1, kv_heads, width, per, values.shape[-1]).permute(0, 2, 1, 3, 4)[size, index]

    def weighted(part, where, index, size, width, values):
        rows = part.new_zeros(where, width, kv_heads, per, part.shape[-1]).index_put((size, index), part)
        sums = torch.matmul(rows.permute(0, 2, 1, 3, 4).reshape(where, kv_heads, width * per, -1), values.permute(0, 2, 1, 3))
        return back(sums, index, size, width)

    low = (position - c["window"] + 1).clamp_min(0) if c["window"] else torch.zeros_like(position)
    n_shared, n_own = -(-s["max_shared_len"] // page), -(-s["max_own_len"] // page) + 1
    zero = torch.zeros(n_group, dtype=torch.int64, device=seq.device)
    pk, pv = _pages_of(s, s["block_tables"][first[:-1]], zero, n_shared)
    ok, ov = _pages_of(s, s["block_tables"], shared // page, n_own)
    most_group, most_q = s["max_group_tokens"], s["max_q_len"]
    on_prefix = back(scores(n_group, in_group, group, most_group, pk), in_group, group, most_group)
    on_own = back(scores(n_seq, in_seq, seq, most_q, ok), in_seq, seq, most_q)
    kp = torch.arange(n_shared * page, device=seq.device)
    ko = torch.arange(n_own * page, device=seq.device) + shared[seq][:, None]
    see_prefix = (kp < shared[seq][:, None]) & (kp >= low[:, None])
    see_own = (ko <= position[:, None]) & (ko >= low[:, None])
    both = torch.cat([on_prefix.masked_fill(~see_prefix[:, None, None], -math.inf),
                      on_own.masked_fill(~see_own[:, None, None], -math.inf)], -1)
    top = both.amax(-1, keepdim=True)
    weights = torch.exp(both - top)
    weights = weights / weights.sum(-1, keepdim=True)
    cut = n_shared * page
    result = (weighted(weights[..., :cut], n_group, in_group, group, most_group, pv)
              + weighted(weights[..., cut:], n_seq, in_seq, seq, most_q, ov))
    return result.reshape(n, heads * dim).to(s["q"].dtype)


def _own_logits(s):
    from matricxon_b200.ops import kernels

    out = torch.empty(s["logits"].shape, dtype=torch.float32, device=s["logits"].device)
    kernels.adjust_logits(s["logits"], out, s["token_offsets"], s["token_ids"], s["repeat"], s["presence"], s["frequency"],
                          bias_offsets=s["bias_offsets"], bias_ids=s["bias_ids"], bias_values=s["bias_values"],
                          mask_words=s["mask_words"], mask_rows=s["mask_rows"], pending_ids=s["pending"])
    return out


def _plain_logits(s):
    rows, vocab = s["logits"].shape
    device = s["logits"].device
    x = s["logits"].float()
    row = torch.arange(rows, device=device)

    def flat(offsets, ids):
        r = torch.searchsorted(offsets[1:].contiguous(), torch.arange(ids.numel(), dtype=torch.int32, device=device), right=True)
        return r * vocab + ids.long()

    counts = torch.zeros(rows * vocab, device=device)
    counts.index_add_(0, flat(s["token_offsets"], s["token_ids"]), torch.ones(s["token_ids"].numel(), device=device))
    pending = s["pending"].long()
    counts.index_add_(0, row * vocab + pending.clamp_min(0), (pending >= 0).float())
    counts = counts.view(rows, vocab)
    seen = counts > 0
    x = torch.where(seen, torch.where(x > 0, x / s["repeat"][:, None], x * s["repeat"][:, None]), x)
    x = x - (s["frequency"][:, None] * counts + s["presence"][:, None] * seen)
    bias = torch.zeros(rows * vocab, device=device)
    bias[flat(s["bias_offsets"], s["bias_ids"])] = s["bias_values"]
    x = x + bias.view(rows, vocab)
    words = s["mask_words"][s["mask_rows"].long().clamp_min(0)]
    allowed = (words[:, :, None] >> torch.arange(32, dtype=torch.int32, device=device)) & 1
    allowed = allowed.view(rows, -1)[:, :vocab].bool() | (s["mask_rows"] < 0)[:, None]
    return x.masked_fill(~allowed, -math.inf)


# --------------------------------------------------------------------------------------- the same from the definitions
def exact(case, seed):
    s = prepare(case, seed)
    return {"tables": _exact_tables, "attention": _exact_attention, "logits": _exact_logits}[case["op"]](s)


def _exact_tables(s):
    """Request by request, on the host."""
    c = s["case"]
    page = c["page"]
    host = {k: v.cpu().numpy() for k, v in s.items() if isinstance(v, torch.Tensor)}
    tables, free = host["tables"].copy(), list(host["free_pages"])
    cu, positions, tok_seq, slots = [0], [], [], []
    n, width = len(host["q_lens"]), tables.shape[1]
    block_tables = np.full((n, width), -1, np.int32)
    at = 0
    for i in range(n):
        context, q, row = int(host["context_lens"][i]), int(host["q_lens"][i]), int(host["rows"][i])
        k = -(-context // page)
        while k * page < context + q:
            tables[row, k] = free[at]
            at, k = at + 1, k + 1
        for p in range(context, context + q):
            positions.append(p)
            tok_seq.append(i)
            slots.append(int(tables[row, p // page]) * page + p % page)
        cu.append(cu[-1] + q)
    for i in range(n):
        context, q, row = int(host["context_lens"][i]), int(host["q_lens"][i]), int(host["rows"][i])
        used = -(-(context + q) // page)
        block_tables[i, :used] = tables[row, :used]
        h = int(host["shared_pages"][i])
        if h:
            block_tables[i, :h] = tables[int(host["shared_rows"][i]), :h]
        if c["window"]:
            block_tables[i, :max(0, context - c["window"] + 1) // page] = -1
    pad = s["n_tokens"] - len(positions)
    return {"positions": np.array(positions + [0] * pad, np.int32), "tok_seq": np.array(tok_seq + [-1] * pad, np.int32),
            "cu_q": np.array(cu, np.int32), "slots": np.array(slots + [-1] * pad, np.int32), "block_tables": block_tables,
            "taken": np.array([at], np.int32), "tables": tables}


def _exact_attention(s):
    """Request by request and KV head by KV head over all of its keys, as if nothing were shared."""
    c = s["case"]
    heads, kv_heads, dim, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    per = heads // kv_heads
    cu, context = s["cu_q"].tolist(), s["context_lens"].tolist()
    out = torch.empty(s["n_tokens"], heads, dim, dtype=torch.float64, device=s["q"].device)
    for i in range(len(context)):
        a, b = cu[i], cu[i + 1]
        length = context[i] + b - a
        pages = s["cache"][s["block_tables"][i, :-(-length // page)].long()]
        p = torch.arange(context[i], length, device=out.device)[:, None]
        j = torch.arange(length, device=out.device)[None]
        hidden = j > p
        if c["window"]:
            hidden = hidden | (j <= p - c["window"])
        for h in range(kv_heads):
            keys = pages[:, 0, h].double().reshape(-1, dim)[:length]
            values = pages[:, 1, h].reshape(-1, dim, page).double().transpose(1, 2).reshape(-1, dim)[:length]
            q = s["q"][a:b].view(b - a, heads, dim)[:, h * per:(h + 1) * per].double()
            score = torch.einsum("thd,kd->htk", q, keys) / math.sqrt(dim)
            out[a:b, h * per:(h + 1) * per] = torch.einsum("htk,kd->thd", torch.softmax(score.masked_fill(hidden, -math.inf), -1), values)
    return out.view(s["n_tokens"], heads * dim)


def _exact_logits(s):
    """Row by row."""
    rows, vocab = s["logits"].shape
    out = torch.empty(rows, vocab, dtype=torch.float64, device=s["logits"].device)
    t, b = s["token_offsets"].tolist(), s["bias_offsets"].tolist()
    pending, mask_rows = s["pending"].tolist(), s["mask_rows"].tolist()
    shifts = torch.arange(32, device=out.device)
    for r in range(rows):
        counts = torch.bincount(s["token_ids"][t[r]:t[r + 1]].long(), minlength=vocab).double()
        if pending[r] >= 0:
            counts[pending[r]] += 1
        x = s["logits"][r].double()
        repeat, presence, frequency = (float(s[k][r]) for k in ("repeat", "presence", "frequency"))
        at = counts > 0
        x[at] = torch.where(x[at] > 0, x[at] / repeat, x[at] * repeat) - frequency * counts[at] - presence
        x[s["bias_ids"][b[r]:b[r + 1]].long()] += s["bias_values"][b[r]:b[r + 1]].double()
        if mask_rows[r] >= 0:
            bits = (s["mask_words"][mask_rows[r]].long()[:, None] >> shifts) & 1
            x[bits.reshape(-1)[:vocab] == 0] = -math.inf
        out[r] = x
    return out
