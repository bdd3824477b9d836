"""Cases of the operators around a paged key-value cache, each in a plain form and as the package's own calls.

A server that keeps many requests of unknown length holds keys and values in pages of a pool instead of one
contiguous cache per row.  One step of its loop is four operators, and every case is one of them:

* ``reserve``  ``paged_reserve``: room for the new tokens of every request, built on the device from the request
               lengths: block tables, slots, positions.  A pass reserves and then takes the same tokens back (a step
               whose speculated tokens were rejected), which leaves the tables as they were.
* ``append``   ``paged_append``: keys and values of new tokens into their slots.
* ``decode``   ``paged_kv_attention``: one new token a request; its key and value are appended on the way.
* ``prompt``   ``paged_prefill_attention``: several new tokens a request (whole prompts, or a chunk after a cached
               prefix), already appended.

Head layouts are those of the package's presets (9/3 and 14/2 heads of 64, 32/8 and 32/32 of 64, 8/1 of 256) and
generic 128-wide ones; up to 64 requests in a decode step, contexts of 1 to 131,072 keys, chunks of 1 to 8,192 tokens,
tables of up to 1,024 requests; pages of 8 to 128 tokens scattered over the pool.
"""

from __future__ import annotations

import math

import torch

own = False

HEADS = ((9, 3, 64), (14, 2, 64), (32, 8, 64), (32, 32, 64), (8, 1, 256), (32, 8, 128), (16, 16, 128), (28, 4, 128),
         (40, 8, 128), (32, 2, 128), (24, 1, 64), (16, 4, 256))
MAX_CACHE = 64 * 8192 * 8 * 128   # values of keys (and of values) that a decode step reads
MAX_SCORES = 32 * 8192 * 8192     # scores of a prompt pass, padded to its longest request


def _reserve(name, mix, requests, tokens, page, *, tight=False):
    return {"name": name, "kind": "reserve", "mix": mix, "requests": requests, "tokens": tokens, "page": page,
            "tight": tight}


def _append(name, tokens, kv_heads, dim, page, *, dtype="bfloat16", padded=False):
    return {"name": name, "kind": "append", "tokens": tokens, "kv_heads": kv_heads, "dim": dim, "page": page,
            "dtype": dtype, "padded": padded}


def _decode(name, batch, keys, heads, page, *, ragged=False, dtype="bfloat16", layout="nhd"):
    return {"name": name, "kind": "decode", "batch": batch, "keys": keys, "heads": heads[0], "kv_heads": heads[1],
            "dim": heads[2], "page": page, "ragged": ragged, "dtype": dtype, "layout": layout}


def _prompt(name, requests, tokens, cached, heads, page, *, dtype="bfloat16", layout="nhd"):
    return {"name": name, "kind": "prompt", "requests": requests, "tokens": tokens, "cached": cached,
            "heads": heads[0], "kv_heads": heads[1], "dim": heads[2], "page": page, "dtype": dtype, "layout": layout}


def listed():
    return [
        # one decode step of a small server: a token for each of 32 requests
        _reserve("reserve-step-r32", "step", 32, 700, 64),
        # requests come and go at once: one in three ends, the others go on; long tables of small pages
        _reserve("reserve-churn-r256", "churn", 256, 1500, 16),
        # the smallest append: one token of one request
        _append("append-1", 1, 3, 64, 64),
        # the prompts of a full batch, padded to a fixed number of rows
        _append("append-16384", 16384, 8, 128, 64, padded=True),
        # the smallest attention: a chat turn of one user, all latency
        _decode("decode-b1-k33", 1, 33, (9, 3, 64), 64),
        # one user with a very long document: the cache's length is all there is to share out
        _decode("decode-b1-k131071", 1, 131071, (32, 8, 128), 64),
        # continuous batching at different depths, idle places in the batch, small pages
        _decode("decode-b37-ragged-k4099", 37, 4099, (14, 2, 64), 16, ragged=True),
        # the largest: a full batch over long contexts
        _decode("decode-b64-k8192", 64, 8192, (32, 8, 128), 64),
        # a one-line prompt
        _prompt("prompt-t19", 1, 19, 0, (9, 3, 64), 64),
        # ragged prompts that are admitted together
        _prompt("prompt-r7-ragged-t1031", 7, 1031, 0, (32, 8, 64), 16, dtype="float16"),
        # a chunk of a long prompt after a cached prefix, 256-wide heads
        _prompt("prompt-chunk-t509-c16000", 1, 509, 16000, (8, 1, 256), 128, layout="hnd"),
        # the largest: a whole long prompt
        _prompt("prompt-t8192", 1, 8192, 0, (32, 8, 128), 64),
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choices(("reserve", "append", "decode", "prompt"), (2, 2, 4, 4))[0]
    page = rng.choice((8, 16, 16, 32, 64, 64, 128))
    dtype = rng.choice(("bfloat16", "bfloat16", "float16"))
    layout = rng.choice(("nhd", "nhd", "hnd"))
    heads = rng.choice(HEADS)
    if kind == "reserve":
        requests = _log_uniform(rng, 1, 1024)
        case = _reserve("", rng.choice(("step", "churn", "admit")), requests,
                        _log_uniform(rng, 2, max(2, min(8192, 400000 // requests))), page, tight=rng.random() < 0.2)
    elif kind == "append":
        case = _append("", _log_uniform(rng, 1, 16384), rng.choice((1, 2, 3, 4, 5, 8)), rng.choice((64, 128)), page,
                       dtype=dtype, padded=rng.random() < 0.5)
    elif kind == "decode":
        batch = _log_uniform(rng, 1, 64)
        most = min(131071, MAX_CACHE // (batch * heads[1] * heads[2]))
        case = _decode("", batch, _log_uniform(rng, 1, most), heads, page, ragged=rng.random() < 0.5, dtype=dtype,
                       layout=layout)
    else:
        requests = rng.choice((1, 1, 2, 3, 5, 9))
        tokens = _log_uniform(rng, 1, 8192 // requests)
        cached = rng.choice((0, _log_uniform(rng, 1, 30000)))
        while requests * heads[0] * tokens * (tokens + cached) > MAX_SCORES:
            tokens, cached = tokens // 2, cached // 2
        case = _prompt("", requests, tokens, cached, heads, page, dtype=dtype, layout=layout)
    del case["name"]
    return case


# ---------------------------------------------------------------------------------------
# Lengths: a function of the case alone
# ---------------------------------------------------------------------------------------
def _spread(most, count, low=1):
    """`most` down to a fraction of it."""
    return [max(low, most - i * most // (count + 1)) for i in range(count)]


def _reserve_lengths(case):
    """(tokens held, tokens asked for or given back) of every request."""
    requests, tokens = case["requests"], case["tokens"]
    held = _spread(tokens, requests, 0)
    if case["mix"] == "admit":
        return [0] * requests, held
    if case["mix"] == "step":
        return held, [0 if i % 11 == 10 else 1 for i in range(requests)]
    return held, [-held[i] if i % 3 == 2 else 1 for i in range(requests)]


def _decode_lengths(case):
    """Keys of every token's request, its new one among them; 0 in an idle place."""
    if not case["ragged"]:
        return [case["keys"]] * case["batch"]
    return _spread(case["keys"], case["batch"]) + [0] * (1 + case["batch"] // 8)


def _prompt_lengths(case):
    """(new tokens, keys of the request, the new ones among them) of every request."""
    new = _spread(case["tokens"], case["requests"])
    cached = _spread(case["cached"], case["requests"], 0)
    return new, [n + c for n, c in zip(new, cached)]


def _pages(tokens, page):
    return (tokens + page - 1) // page


# ---------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------
def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _table(lengths, width, page, pages, g):
    """Pages of the pool in random order, dealt out to the requests; -1 where a request has none."""
    held = torch.tensor([_pages(n, page) for n in lengths], device="cuda")
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    column = torch.arange(width, device="cuda")
    index = (held.cumsum(0) - held)[:, None] + column
    table = torch.where(column < held[:, None], order[index.clamp(max=pages - 1)], torch.full_like(index, -1,
                                                                                                 dtype=torch.int32))
    return table.contiguous(), order, sum(_pages(n, page) for n in lengths)


def _pool(case, pages, g, dtype):
    shape = (pages, case["page"], case["kv_heads"], case["dim"])
    if case.get("layout") == "hnd":   # every head of a page in one piece
        shape = (shape[0], shape[2], shape[1], shape[3])
    pools = [torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=g) for _ in range(2)]
    return [p.transpose(1, 2) for p in pools] if case.get("layout") == "hnd" else pools


def _normal(shape, g, dtype):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=g)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    page, kind = case["page"], case["kind"]
    if kind == "reserve":
        held, counts = _reserve_lengths(case)
        after = [max(0, n + c) for n, c in zip(held, counts)]
        need = sum(_pages(max(a, b), page) for a, b in zip(held, after))
        width = max(_pages(max(a, b), page) for a, b in zip(held, after)) + 2
        used = sum(_pages(n, page) for n in held)
        pages = max(1, used + (need - used) // 2 if case["tight"] else need + need // 4 + 4)
        table, order, _ = _table(held, width, page, pages, g)
        stack = torch.cat([order[used:], torch.zeros(used, dtype=torch.int32, device="cuda")])
        # which request holds how much is a matter of chance
        deal = torch.randperm(case["requests"], generator=g, device="cuda")
        return {"kind": kind, "page": page, "counts": _int32(counts)[deal], "lengths": _int32(held)[deal],
                "table": table[deal].contiguous(), "stack": stack, "free": _int32([pages - used]),
                "most": sum(abs(c) for c in counts) + 3}
    dtype = getattr(torch, case["dtype"])
    if kind == "append":
        tokens = case["tokens"]
        pages = _pages(tokens, page) + 3
        pools = _pool(case, pages, g, dtype)
        slots = torch.randperm(pages, generator=g, device="cuda")[:, None] * page + torch.arange(page, device="cuda")
        slots = slots.flatten()[:tokens].contiguous()
        if case["padded"]:
            slots[tokens - tokens // 8:] = -1
        # keys and values come as parts of one projection's rows
        rows = _normal((tokens, 2, case["kv_heads"], case["dim"]), g, dtype)
        return {"kind": kind, "key": rows[:, 0], "value": rows[:, 1], "pools": pools, "slots": slots}
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    if kind == "decode":
        lengths = _decode_lengths(case)
        tokens = len(lengths)
        total = sum(_pages(n, page) for n in lengths)
        table, _, _ = _table(lengths, _pages(max(lengths), page) + 3, page, total + total // 8 + 2, g)
        pools = _pool(case, total + total // 8 + 2, g, dtype)
        rows = None
        if case["ragged"]:   # token t belongs to request rows[t]; idle places have none
            deal = torch.randperm(tokens, generator=g, device="cuda")
            rows = torch.argsort(deal).to(torch.int32)
            rows[torch.tensor(lengths, device="cuda") == 0] = -1
            table, lengths = table[deal].contiguous(), _int32(lengths)[deal]
        else:
            lengths = _int32(lengths)
        qkv = _normal((tokens, heads + 2 * kv_heads, dim), g, dtype)
        return {"kind": kind, "query": qkv[:, :heads], "key": qkv[:, heads:heads + kv_heads],
                "value": qkv[:, heads + kv_heads:], "pools": pools, "table": table, "lengths": lengths, "rows": rows}
    new, lengths = _prompt_lengths(case)
    total = sum(_pages(n, page) for n in lengths)
    table, _, _ = _table(lengths, _pages(max(lengths), page) + 3, page, total + total // 8 + 2, g)
    pools = _pool(case, total + total // 8 + 2, g, dtype)
    offsets = [0]
    for n in new:
        offsets.append(offsets[-1] + n)
    return {"kind": kind, "query": _normal((offsets[-1] + 5, heads, dim), g, dtype), "pools": pools, "table": table,
            "lengths": _int32(lengths), "offsets": _int32(offsets), "longest": max(new)}


# ---------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------
def run(state):
    if state["kind"] == "reserve":
        names = ("lengths", "table", "stack", "free")
        if own:
            from megabake_b200 import paged_reserve
        else:
            paged_reserve = _plain_reserve
        tables = [state[n] for n in names]
        first = paged_reserve(state["counts"], *tables, state["page"], state["most"])
        back = paged_reserve(-first[4], *tables, state["page"], state["most"])
        return {"first": list(first), "back": list(back), "tables": tables}
    if state["kind"] == "append":
        args = (state["key"], state["value"], *state["pools"], state["slots"])
        if own:
            from megabake_b200 import paged_append
            paged_append(*args)
        else:
            _plain_append(*args)
        return state["pools"]
    if state["kind"] == "decode":
        args = (state["query"], state["key"], state["value"], *state["pools"], state["table"], state["lengths"],
                state["rows"])
        if own:
            from megabake_b200 import paged_kv_attention
            return [paged_kv_attention(*args), *state["pools"]]
        return [_plain_decode(*args), *state["pools"]]
    args = (state["query"], *state["pools"], state["table"], state["lengths"], state["offsets"])
    if own:
        from megabake_b200 import paged_prefill_attention
        return paged_prefill_attention(*args)
    return _plain_prompt(*args, state["longest"])


# ---------------------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------------------
def _plain_reserve(counts, lengths, table, stack, free, page, most):
    width, pages = table.shape[1], stack.numel()
    column = torch.arange(width, device=table.device)
    c, old = counts.long(), lengths.long().clamp(0, width * page)
    # give back: rows and pages from the last to the first, so that the first page lies on top
    keep = torch.where(c < 0, (old + c).clamp(min=0), old)
    held, kept = _pages(old, page)[:, None], _pages(keep, page)[:, None]
    gone = (column >= kept) & (column < held)
    backwards = gone.flatten().flip(0)
    place = torch.where(backwards, free.long() + backwards.cumsum(0) - 1, pages).clamp(max=pages)
    padded = torch.cat([stack, stack.new_zeros(1)])
    padded.scatter_(0, place, table.flatten().flip(0))
    stack.copy_(padded[:pages])
    entries = torch.where(gone, -1, table.long())
    available = free.long() + gone.sum()
    # grant, in order
    need = torch.where(c > 0, _pages(keep + c, page) - kept[:, 0], 0)
    fits = (c > 0) & (keep + c <= width * page)
    tokens, wanted = torch.where(fits, c, 0), torch.where(fits, need, 0)
    granted = fits & (tokens.cumsum(0) <= most) & ((need == 0) | (wanted.cumsum(0) <= available))
    got, pages_got = torch.where(granted, c, 0), torch.where(granted, need, 0)
    index = available - 1 - ((pages_got.cumsum(0) - pages_got)[:, None] + column - kept)
    takes = (column >= kept) & (column < kept + pages_got[:, None])
    table.copy_(torch.where(takes, stack[index.clamp(0, pages - 1)].long(), entries))
    lengths.copy_(keep + got)
    free.copy_(available - pages_got.sum())
    # where every token goes
    offsets = torch.cat([got.new_zeros(1), got.cumsum(0)])
    token = torch.arange(most, device=table.device)
    row = torch.searchsorted(offsets[1:].contiguous(), token, right=True).clamp(max=counts.numel() - 1)
    valid = token < offsets[-1]
    position = torch.where(valid, keep[row] + token - offsets[row], 0)
    slot = table[row, position // page].long() * page + position % page
    return (offsets.int(), torch.where(valid, slot, -1), position, torch.where(valid, row, -1).int(),
            torch.where(c < 0, keep - old, got).int())


def _plain_append(key, value, key_pages, value_pages, slots):
    page = key_pages.shape[1]
    valid = slots >= 0
    # what belongs nowhere repeats the first token, which has a slot
    token = torch.where(valid, torch.arange(slots.numel(), device=slots.device), 0)
    place = slots[token]
    for rows, pages in ((key, key_pages), (value, value_pages)):
        pages[place // page, place % page] = rows[token]


def _plain_decode(query, key, value, key_pages, value_pages, table, lengths, rows):
    page = key_pages.shape[1]
    tokens, heads, dim = query.shape
    row = torch.arange(tokens, device=query.device) if rows is None else rows.long().clamp(min=0)
    length = lengths[row].long()
    if rows is not None:
        length = torch.where(rows < 0, 0, length)
    table = table[row].long()
    last = (length - 1).clamp(min=0)
    slot = table.gather(1, (last // page)[:, None])[:, 0] * page + last % page
    _plain_append(key, value, key_pages, value_pages, torch.where(length > 0, slot, -1))
    kv_heads = key_pages.shape[2]
    keys, values = (p[table.clamp(min=0)].flatten(1, 2).float() for p in (key_pages, value_pages))
    seen = (torch.arange(keys.shape[1], device=query.device) < length[:, None])[:, None, None]
    grouped = query.float().reshape(tokens, kv_heads, heads // kv_heads, dim)
    scores = torch.einsum("tkgd,tlkd->tkgl", grouped, keys) * dim ** -0.5
    scores = torch.where(seen, scores, -torch.inf)
    highest = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(highest == -torch.inf, 0, highest))
    mixed = torch.einsum("tkgl,tlkd->tkgd", weights, values) / weights.sum(-1, keepdim=True).clamp(min=1e-30)
    return mixed.reshape(tokens, heads, dim).to(query.dtype)


def _plain_prompt(query, key_pages, value_pages, table, lengths, offsets, longest):
    count, heads, dim = query.shape
    kv_heads, requests = key_pages.shape[2], lengths.numel()
    keys, values = (p[table.long().clamp(min=0)].flatten(1, 2).float() for p in (key_pages, value_pages))
    step = torch.arange(longest, device=query.device)
    new = (offsets[1:] - offsets[:-1]).long()[:, None]
    place = torch.where(step < new, offsets[:-1].long()[:, None] + step, count)   # the row behind the last takes the rest
    padded = torch.cat([query, query.new_zeros(1, heads, dim)])[place].float()
    grouped = padded.reshape(requests, longest, kv_heads, heads // kv_heads, dim)
    scores = torch.einsum("rtkgd,rlkd->rkgtl", grouped, keys).mul_(dim ** -0.5)
    last = (lengths.long()[:, None] - new + step).clamp(min=0)     # the position of every query
    unseen = torch.arange(keys.shape[1], device=query.device) > last[:, :, None]
    scores.masked_fill_(unseen[:, None, None], -torch.inf)
    weights = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    mixed = torch.einsum("rkgtl,rlkd->rtkgd", weights / weights.sum(-1, keepdim=True), values)
    out = query.new_zeros(count + 1, heads, dim)
    out[place.flatten()] = mixed.reshape(-1, heads, dim).to(query.dtype)
    out[count] = 0
    return out[:count]


# ---------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------
def work(case):
    page = case["page"]
    if case["kind"] == "reserve":
        # twice: what is asked for; lengths and what is granted, offsets; pages given or taken, on both sides; 20 bytes
        # for every place of a token
        held, counts = _reserve_lengths(case)
        moved = sum(abs(_pages(n + c, page) - _pages(n, page)) for n, c in zip(held, counts))
        return {"bytes": 2 * (20 * case["requests"] + 12 * moved + 20 * (sum(abs(c) for c in counts) + 3)), "flops": 0}
    row = case["kv_heads"] * case["dim"] * 2
    if case["kind"] == "append":
        written = case["tokens"] - (case["tokens"] // 8 if case["padded"] else 0)
        return {"bytes": 4 * written * row + 8 * case["tokens"], "flops": 0}
    query_row = case["heads"] * case["dim"] * 2
    if case["kind"] == "decode":
        lengths = _decode_lengths(case)
        used = sum(n > 0 for n in lengths)
        return {"bytes": 2 * row * (sum(lengths) + used) + 2 * query_row * len(lengths)
                + 4 * sum(_pages(n, page) for n in lengths),
                "flops": 4 * sum(lengths) * case["heads"] * case["dim"]}
    new, lengths = _prompt_lengths(case)
    pairs = sum(n * (length - n) + n * (n + 1) // 2 for n, length in zip(new, lengths))
    return {"bytes": 2 * row * sum(lengths) + 2 * query_row * sum(new) + 4 * sum(_pages(n, page) for n in lengths),
            "flops": 4 * pairs * case["heads"] * case["dim"]}


# ---------------------------------------------------------------------------------------
# The definition, in 64 bits
# ---------------------------------------------------------------------------------------
def exact(case, seed):
    if case["kind"] == "reserve":
        return None   # whole numbers
    state = prepare(case, seed)
    key_pages, value_pages = state["pools"]
    page = case["page"]
    if case["kind"] == "append":
        kept = (state["slots"] >= 0).nonzero()[:, 0]
        for pages, rows in ((key_pages, state["key"]), (value_pages, state["value"])):
            flat = pages.flatten(0, 1)    # a view: the pages follow one another
            flat.index_copy_(0, state["slots"][kept], rows[kept])
        return [key_pages, value_pages]
    group, lengths, table = case["heads"] // case["kv_heads"], state["lengths"].tolist(), state["table"].long()

    def context(request, pages, head):
        count = _pages(lengths[request], page)
        return pages[table[request, :count], :, head].flatten(0, 1)[:lengths[request]].double()

    def attend(queries, request, head):
        """`queries` [n, D] of one head, the last n positions of the request."""
        scores = queries.double() @ context(request, key_pages, head // group).T / math.sqrt(case["dim"])
        n, total = scores.shape
        future = torch.ones(n, total, dtype=torch.bool, device=scores.device).triu(total - n + 1)
        weights = scores.masked_fill(future, -torch.inf).softmax(-1)
        return weights @ context(request, value_pages, head // group)

    query = state["query"]
    out = torch.zeros(query.shape, dtype=torch.float64, device=query.device)
    if case["kind"] == "decode":
        rows = range(len(lengths)) if state["rows"] is None else state["rows"].tolist()
        for token, request in enumerate(rows):
            if request < 0 or lengths[request] == 0:
                continue
            last = lengths[request] - 1
            at = int(table[request, last // page])
            key_pages[at, last % page] = state["key"][token]
            value_pages[at, last % page] = state["value"][token]
            for head in range(case["heads"]):
                out[token, head] = attend(query[token, head:head + 1], request, head)[0]
        return [out, key_pages, value_pages]
    offsets = state["offsets"].tolist()
    for request in range(len(lengths)):
        first, last = offsets[request], offsets[request + 1]
        for head in range(case["heads"]):
            out[first:last, head] = attend(query[first:last, head], request, head)
    return out
