"""Cases, plain forms and 64-bit values of the operators around a paged KV cache.

A serving loop that admits and finishes requests keeps K and V rows in pages of a pool. Each step
makes room for the new tokens of every sequence and gives back what finished requests held (table:
block tables, slot maps), stores the new rows (append), and attends with each new token over its
sequence's pages (attend), or over the few pages that a cheap score selects for it (sparse). Shapes
are those of the BaseLM backbone (16 query heads of 128 on 2 KV heads, contexts of 64 to 4096 for 16
streams and up to 32768 for one), of the one-layer model with heads of 64, and generic ones.

The pool is [pages][kv_heads][2: K, V][page rows][head_dim] in fp16 or bf16. ``table`` int32
[sequences][pages of one] names the pages of each sequence in order, -1 where it holds none; ``rows``
int32 [sequences] says how many rows it holds; ``free`` int32 [pages] is a stack of free pages whose
height is ``pool[0]``. Freed pages are pushed in the order of sequences and table entries, and the
pages that a step hands out are the topmost ones, in the order in which they lie in the stack. A step's
``slots`` say where each new token's row goes (page * page rows + row), its ``positions`` and
``sequences`` whose it is, and its ``runs`` the new rows page by page: first token, page, first row, rows.

The summary of a page is, per KV head and channel, the smallest and the largest K of its rows. The
score of a page for a query is the largest sum of its heads' products with K that the summary allows:
the sum over channels and heads of max(q * smallest, q * largest), in 64 bits. The first ``sinks`` and
the last ``recent`` pages of a query's rows are always selected, then those of the highest scores.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
FULL, NO_PAGES, BAD_COUNT = 1, 2, 4     # status of a sequence's last step


# --------------------------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------------------------
def listed():
    backbone = {"heads": 16, "kv_heads": 2, "head_dim": 128}
    return [
        # one token for each of 16 streams, one of which has finished and is followed by a prompt of 40 (latency)
        {"name": "table_step", "op": "table", "seqs": 16, "page": 64, "low": 64, "high": 4096, "finished": 1, "prompt": 40,
         "short": 0},
        # 256 streams with pages of 16 rows: 16 finish and are followed by prompts of 512, for the last of which no page is left
        {"name": "table_admit", "op": "table", "seqs": 256, "page": 16, "low": 64, "high": 4096, "finished": 16,
         "prompt": 512, "short": 40},
        # a new batch: 1024 prompts of 128 tokens after as many finished requests
        {"name": "table_batch", "op": "table", "seqs": 1024, "page": 32, "low": 16, "high": 1024, "finished": 1024,
         "prompt": 128, "short": 0},
        # one row for each of 16 streams, with the summaries that page selection reads (latency)
        {"name": "append_step", "op": "append", "seqs": 16, "tokens": 1, "kv_heads": 2, "head_dim": 128, "page": 64,
         "low": 64, "high": 4096, "dtype": "f32", "cache": "f16", "summaries": True},
        # the prompts of 16 requests, about 4096 tokens each, 8 KV heads
        {"name": "append_prompts", "op": "append", "seqs": 16, "tokens": 4097, "kv_heads": 8, "head_dim": 128, "page": 16,
         "low": 0, "high": 100, "dtype": "bf16", "cache": "bf16", "summaries": True},
        # the one-layer model's single token after 512 cached rows: the smallest call (latency)
        {"name": "attend_one", "op": "attend", "seqs": 1, "tokens": 1, "heads": 16, "kv_heads": 2, "head_dim": 64,
         "page": 16, "low": 513, "high": 513, "dtype": "f32", "cache": "f16"},
        # a decode step of 16 streams at ragged contexts, 32-bit activations
        {"name": "attend_streams", "op": "attend", "seqs": 16, "tokens": 1, **backbone, "page": 64, "low": 64,
         "high": 4096, "dtype": "f32", "cache": "f16"},
        # 5 drafted tokens of 16 streams
        {"name": "attend_draft", "op": "attend", "seqs": 16, "tokens": 5, **backbone, "page": 32, "low": 64,
         "high": 4096, "dtype": "f16", "cache": "f16"},
        # a decode step of 16 streams deep in long contexts, 16-bit activations
        {"name": "attend_long", "op": "attend", "seqs": 16, "tokens": 1, **backbone, "page": 64, "low": 24001,
         "high": 32768, "dtype": "bf16", "cache": "bf16"},
        # one long session that reads 2048 of its 32768 rows (latency)
        {"name": "sparse_one", "op": "sparse", "seqs": 1, "tokens": 1, **backbone, "page": 16, "low": 32768,
         "high": 32768, "budget": 128, "sinks": 1, "recent": 4, "dtype": "f32", "cache": "f16"},
        # 16 streams deep in long contexts that read 4096 rows each
        {"name": "sparse_streams", "op": "sparse", "seqs": 16, "tokens": 1, **backbone, "page": 64, "low": 24001,
         "high": 32768, "budget": 64, "sinks": 1, "recent": 2, "dtype": "bf16", "cache": "bf16"},
        # 16 sessions of 131072 rows and pages of 16
        {"name": "sparse_long", "op": "sparse", "seqs": 16, "tokens": 1, **backbone, "page": 16, "low": 131072,
         "high": 131072, "budget": 512, "sinks": 2, "recent": 16, "dtype": "f16", "cache": "f16"},
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["table", "append", "attend", "attend", "sparse"])
    page = rng.choice([16, 16, 32, 64, 128])
    if op == "table":
        while True:
            n, high = _log(rng, 1, 1024), _log(rng, 16, 8192)
            c = {"op": op, "seqs": n, "page": page, "low": rng.randrange(0, high), "high": high,
                 "finished": rng.randrange(0, n + 1), "prompt": _log(rng, 1, 4096), "short": rng.choice([0, 0, _log(rng, 1, 64)])}
            if n * high <= 1 << 21 and c["finished"] * c["prompt"] <= 1 << 17:
                return c
    cache = rng.choice(["f16", "bf16"])
    dtype = rng.choice(["f32", cache, cache])
    if op == "append":
        while True:
            high = _log(rng, 1, 4096)
            c = {"op": op, "seqs": _log(rng, 1, 64), "tokens": _log(rng, 1, 4097), "kv_heads": rng.choice([1, 2, 3, 8]),
                 "head_dim": rng.choice([64, 128]), "page": page, "low": rng.randrange(0, high), "high": high,
                 "dtype": dtype, "cache": cache, "summaries": rng.random() < 0.6}
            if c["seqs"] * (c["tokens"] + high) * c["kv_heads"] * c["head_dim"] <= 16 * 4097 * 1024:
                return c
    while True:
        heads, kv_heads = rng.choice([(16, 2), (8, 2), (2, 1), (12, 2), (8, 8), (32, 2), (6, 3), (16, 1)])
        c = {"op": op, "seqs": _log(rng, 1, 64), "tokens": 1, "heads": heads, "kv_heads": kv_heads,
             "head_dim": rng.choice([64, 128, 128]), "page": page}
        if op == "attend":
            c["tokens"] = rng.choice([1, 1, rng.randrange(2, 9)])
        high = _log(rng, 4 * page if op == "sparse" else 16, 32768)
        c.update(low=rng.randrange(c["tokens"], high + 1), high=high)
        if op == "sparse":
            budget = rng.randrange(2, max(3, high // page))
            sinks = rng.randrange(0, min(4, budget))
            c.update(budget=budget, sinks=sinks, recent=rng.randrange(0, min(17, budget - sinks + 1)))
        c.update(dtype=dtype, cache=cache)
        if c["seqs"] * c["tokens"] * high * kv_heads * c["head_dim"] <= 16 * 32768 * 256 and \
                c["seqs"] * c["tokens"] * high * heads <= 1 << 25:
            return c


def _lengths(case):
    """Rows held by each sequence: spread over [low, high], in a mixed order."""
    n, low, high = case["seqs"], case["low"], case["high"]
    if n == 1:
        return [high]
    step = next(k for k in range(max(1, n * 5 // 8), n + 2) if math.gcd(k, n) == 1)
    return [low + (high - low) * (i * step % n) // (n - 1) for i in range(n)]


def _pages(rows, page):
    return -(-rows // page)


def _news(case):
    """New rows of each sequence (append: about `tokens` each, mixed lengths; table: prompts where a request has finished,
    else one)."""
    n = case["seqs"]
    if case["op"] == "table":
        return [case["prompt"] if _finished(case, i) else 1 for i in range(n)]
    return [case["tokens"] - (i * 7 % 16) * (case["tokens"] // 64) for i in range(n)]


def _finished(case, i):
    n, f = case["seqs"], case["finished"]
    return (i + 1) * f // n > i * f // n


def work(case):
    op = case["op"]
    lengths = _lengths(case)
    if op == "table":
        page, news = case["page"], _news(case)
        kept = [0 if _finished(case, i) else r for i, r in enumerate(lengths)]
        freed = sum(_pages(r, page) - _pages(k, page) for r, k in zip(lengths, kept))
        taken = max(0, sum(_pages(k + c, page) - _pages(k, page) for k, c in zip(kept, news)) - case["short"])
        runs = sum(_pages(k + c, page) - k // page for k, c in zip(kept, news))
        # rows, keep and counts in; rows, status and starts out; three words a token, four a run; page numbers out of
        # the table into the stack and the other way
        return {"bytes": 24 * len(lengths) + 12 * sum(news) + 16 * runs + 12 * freed + 8 * taken, "flops": 8 * sum(news)}
    size = torch.empty(0, dtype=DTYPES[case["dtype"]]).element_size()
    wide, page = case["kv_heads"] * case["head_dim"], case["page"]
    if op == "append":
        news = _news(case)
        b = 2 * sum(news) * wide * (size + 2)
        if case["summaries"]:     # the K rows that the first page of each holds already, and a summary of each page
            b += sum(r % page for r in lengths) * wide * 2
            b += sum(_pages(r + c, page) - r // page for r, c in zip(lengths, news)) * wide * 4
        return {"bytes": b, "flops": 2 * sum(news) * wide}
    n, t, group = case["seqs"], case["tokens"], case["heads"] // case["kv_heads"]
    q = 2 * n * t * case["heads"] * case["head_dim"] * size
    if op == "attend":
        pairs = sum(t * (m - t) + t * (t + 1) // 2 for m in lengths)
        return {"bytes": 4 * sum(lengths) * wide + q, "flops": 4 * pairs * wide * group}
    chosen = [min(case["budget"], _pages(m, page)) for m in lengths]
    scored = [_pages(m, page) if _pages(m, page) > case["budget"] else 0 for m in lengths]
    rows = sum(c * page for c in chosen)
    return {"bytes": 4 * sum(scored) * wide + 4 * rows * wide + q + 4 * sum(chosen) * case["kv_heads"],
            "flops": 4 * sum(scored) * wide + 4 * rows * wide * group}


# --------------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed & 0x7FFFFFFF)


def _normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _ints(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def _state(s, g, lengths, most, spare):
    """Tables of sequences that hold `lengths` rows, with pages in a mixed order: room for `most` rows each, `spare` free
    pages. Buffers have one page more than the pool, where plain forms put what goes nowhere."""
    page = s["page"]
    wide = max(1, _pages(most, page))
    held = torch.tensor([_pages(r, page) for r in lengths]).cuda()
    pages = s["pages"] = int(sum(_pages(r, page) for r in lengths)) + spare
    order = torch.randperm(pages, generator=g, device="cuda").int()
    col = torch.arange(wide, device="cuda")
    place = (held.cumsum(0) - held)[:, None] + col
    s["table"] = torch.where(col < held[:, None], order[place.clamp_max(pages - 1)], -1)
    s["rows"] = _ints(lengths)
    s["status"] = torch.zeros_like(s["rows"])
    s["free"] = torch.cat((order[pages - spare:], order.new_zeros(pages - spare)))
    s["pool"] = _ints([spare, 0])
    s["seq_pages"] = wide


def _fill(s, g):
    """A pool of K and V rows, and the summaries of its pages: K drifts from page to page and a few of its channels are
    large, as in trained models."""
    h, d, page, dtype = s["kv_heads"], s["head_dim"], s["page"], DTYPES[s["cache"]]
    s["data"] = torch.empty(s["pages"] + 1, h, 2, page, d, dtype=dtype, device="cuda")
    # 16 bits at a time: a normal of every value would take as long as the measurement
    s["data"].normal_(generator=g)
    gain = _normal(g, 1, h, 1, d).mul(0.8).exp().to(dtype)
    s["data"][:, :, 0] = (s["data"][:, :, 0] + _normal(g, s["pages"] + 1, h, 1, d, dtype=dtype)).mul_(gain)


def prepare(case, seed):
    g = _generator(seed)
    s = dict(case)
    lengths = _lengths(case)
    page = case["page"]
    if case["op"] in ("table", "append"):
        news = _news(case)
        kept = [0 if case["op"] == "table" and _finished(case, i) else r for i, r in enumerate(lengths)]
        freed = sum(_pages(r, page) - _pages(k, page) for r, k in zip(lengths, kept))
        need = sum(_pages(k + c, page) - _pages(k, page) for k, c in zip(kept, news))
        spare = max(0, need - freed - case.get("short", 0))
        _state(s, g, lengths, max(max(k + c for k, c in zip(kept, news)), max(lengths)), spare)
        s["news"], s["kept"] = _ints(news), _ints(kept)
        s["total"] = sum(news) + (5 if case["op"] == "table" else 0)    # rows of the step's buffers: some are padding
    if case["op"] == "append":
        shape = s["total"], case["kv_heads"], case["head_dim"]
        s["k"], s["v"] = (_normal(g, *shape, dtype=DTYPES[case["dtype"]]) for _ in "kv")
        s["data"] = torch.zeros(s["pages"] + 1, case["kv_heads"], 2, page, case["head_dim"], dtype=DTYPES[case["cache"]],
                                device="cuda")
        # what the pages hold before: only rows that share a page with new ones matter
        at = (torch.arange(len(lengths), device="cuda"), (s["rows"].long() // page).clamp_max(s["seq_pages"] - 1))
        first = s["table"][at].long()
        first = torch.where(first < 0, s["pages"], first)
        s["data"][first] = _normal(g, len(lengths), *s["data"].shape[1:], dtype=s["data"].dtype)
        s["summaries_of"] = torch.zeros(s["pages"] + 1, case["kv_heads"], 2, case["head_dim"], dtype=s["data"].dtype,
                                        device="cuda") if case["summaries"] else None
        s["step"] = _plain_table(s)     # the step that this append belongs to
    elif case["op"] in ("attend", "sparse"):
        _state(s, g, lengths, max(lengths), 3)
        _fill(s, g)
        n, t = case["seqs"], case["tokens"]
        s["q"] = _normal(g, n * t, case["heads"], case["head_dim"]).mul(1.5).to(DTYPES[case["dtype"]])
        s["sequences"] = torch.arange(n, device="cuda").repeat_interleave(t).int()
        s["positions"] = s["rows"][s["sequences"].long()] - t + torch.arange(t, device="cuda").repeat(n).int()
        if case["op"] == "sparse":
            k = s["data"][:, :, 0]
            s["summaries_of"] = torch.stack((k.amin(2), k.amax(2)), 2)
            # rows that a sequence's last page has room for are not held: their values are in no summary
            at = (torch.arange(n, device="cuda"), ((s["rows"].long() - 1) // page))
            last = s["table"][at].long()
            past = (torch.arange(page, device="cuda") >= (s["rows"].long()[:, None] - 1) % page + 1)[:, None, :, None]
            k = s["data"][last][:, :, 0]
            s["summaries_of"][last] = torch.stack((k.masked_fill(past, math.inf).amin(2),
                                                   k.masked_fill(past, -math.inf).amax(2)), 2)
    return s


# --------------------------------------------------------------------------------------------
# the framework's operators
# --------------------------------------------------------------------------------------------
def _objects(s):
    """The table and cache objects over the buffers in hand, kept as a program keeps them."""
    if "objects" not in s:
        from voxgen_b200.paged import PagedCache, PageTable
        table = PageTable(s["seqs"], s["pages"], s["page"], s["seq_pages"], table=s["table"], rows=s["rows"],
                          status=s["status"], free=s["free"], pool=s["pool"])
        cache = None
        if "data" in s:
            cache = PagedCache(table, s["kv_heads"], s["head_dim"], dtype=s["data"].dtype, data=s["data"][:-1],
                               summaries=None if s.get("summaries_of") is None else s["summaries_of"][:-1])
        if s["op"] == "append":
            from voxgen_b200.paged import Step
            s["step_of"] = Step.of(table, **s["step"])
        s["objects"] = table, cache
    return s["objects"]


def _run_own(s):
    table, cache = _objects(s)
    if s["op"] == "table":
        step = table.step(s["news"], s["total"], keep=s["kept"])
        return {"table": s["table"], "rows": s["rows"], "status": s["status"], "free": s["free"], "pool": s["pool"],
                "starts": step.starts, "slots": step.slots, "positions": step.positions, "sequences": step.sequences,
                "runs": step.runs}
    if s["op"] == "append":
        cache.append(s["step_of"], s["k"], s["v"])
        out = {"data": s["data"][:-1]}
        return {**out, "summaries": s["summaries_of"][:-1]} if s["summaries"] else out
    which = (None, None) if s["tokens"] == 1 else (s["sequences"], s["positions"])
    if s["op"] == "attend":
        return {"out": cache.attention(s["q"], sequences=which[0], positions=which[1])}
    chosen = cache.select(s["q"], s["budget"], sinks=s["sinks"], recent=s["recent"])
    return {"chosen": chosen, "out": cache.attention(s["q"], chosen=chosen)}


# --------------------------------------------------------------------------------------------
# plain forms
# --------------------------------------------------------------------------------------------
def _plain_table(s):
    page, t, wide, pages = s["page"], s["total"], s["seq_pages"], s["pages"]
    rows, counts = s["rows"].long(), s["news"].long()
    kept = torch.where(s["kept"] < 0, rows, torch.minimum(s["kept"].long(), rows))
    bad = (counts < 0) | (counts > t)
    counts = torch.where(bad, 0, counts)
    starts = torch.cat((counts.new_zeros(1), counts.cumsum(0)))
    bad |= starts[1:] > t
    full = kept + counts > wide * page
    held, stay = _pages(rows, page), _pages(kept, page)
    # freed pages, onto the stack
    col = torch.arange(wide, device="cuda")
    freed = held - stay
    height = s["pool"][0].long()
    on_stack = height + (freed.cumsum(0) - freed)[:, None] + col - stay[:, None]
    frees = (col >= stay[:, None]) & (col < held[:, None])
    stack = torch.cat((s["free"], s["free"].new_zeros(1)))
    stack.scatter_(0, torch.where(frees, on_stack, pages).flatten(), s["table"].flatten())
    s["free"].copy_(stack[:-1])
    height = height + freed.sum()
    # pages for what fits, off its top
    need = torch.where(bad | full, 0, _pages(kept + counts, page) - stay)
    before = need.cumsum(0) - need
    short = (need > 0) & (before + need > height)
    ok = ~(bad | full | short)
    need = torch.where(ok, need, 0)
    height = height - need.sum()
    takes = (col >= stay[:, None]) & (col < (stay + need)[:, None])
    taken = s["free"][(height + before[:, None] + col - stay[:, None]).clamp(0, pages - 1)]
    s["table"].copy_(torch.where(takes, taken, torch.where(col < stay[:, None], s["table"], -1)))
    new = torch.where(ok, counts, 0)
    s["rows"].copy_(kept + new)
    s["status"].copy_(torch.where(bad, BAD_COUNT, torch.where(full, FULL, torch.where(short, NO_PAGES, 0))))
    s["pool"][0] = height
    # the tokens of the step
    i = torch.arange(t, device="cuda")
    seq = torch.searchsorted(starts[1:].contiguous(), i, right=True).clamp_max(s["seqs"] - 1)
    valid = (i < starts[-1]) & ok[seq]
    pos = torch.where(valid, kept[seq] + i - starts[seq], 0)
    slot = s["table"][seq, pos // page] * page + pos % page
    token = {"slots": slot, "positions": pos, "sequences": seq}
    token = {k: torch.where(valid, x, -1).int() for k, x in token.items()}
    # its new rows page by page
    first = kept // page
    count = torch.where(new > 0, (kept + new - 1) // page - first + 1, 0)
    upto = count.cumsum(0)
    i = torch.arange(min(t, t // page + 2 * s["seqs"]), device="cuda")
    seq = torch.searchsorted(upto, i, right=True).clamp_max(s["seqs"] - 1)
    col = (first[seq] + i - (upto - count)[seq]).clamp(0, wide - 1)
    a, b = torch.maximum(kept[seq], col * page), torch.minimum((kept + new)[seq], (col + 1) * page)
    runs = torch.stack((starts[seq] + a - kept[seq], s["table"][seq, col].long(), a % page, b - a), 1)
    runs = torch.where((i < upto[-1])[:, None], runs, 0)
    return {"starts": starts.clamp_max(t).int(), **token, "runs": runs.int()}


def _table(s):
    step = _plain_table(s)
    return {"table": s["table"], "rows": s["rows"], "status": s["status"], "free": s["free"], "pool": s["pool"], **step}


def _append(s):
    page, dtype = s["page"], s["data"].dtype
    slot = s["step"]["slots"].long()
    at = torch.where(slot < 0, s["pages"], slot // page)     # tokens without a slot go to the page past the pool
    row = slot.clamp_min(0) % page
    s["data"][at, :, 0, row] = s["k"].to(dtype)
    s["data"][at, :, 1, row] = s["v"].to(dtype)
    if not s["summaries"]:
        return {"data": s["data"][:-1]}
    # of a page, its last token of the step knows how many of its rows are held
    last = (at != torch.cat((at[1:], at.new_full((1,), -1)))).nonzero()[:, 0]
    p, n = at[last], row[last] + 1
    past = (torch.arange(page, device="cuda") >= n[:, None])[:, None, :, None]
    k = s["data"][p][:, :, 0].float()
    past = past | k.isnan()
    top = torch.finfo(dtype).max
    low, high = k.masked_fill(past, math.inf).amin(2), k.masked_fill(past, -math.inf).amax(2)
    none = past.expand_as(k).all(2)
    found = torch.stack((low, high), 2).clamp(-top, top).masked_fill(none[:, :, None], 0.0)
    s["summaries_of"][p] = found.to(dtype)
    return {"data": s["data"][:-1], "summaries": s["summaries_of"][:-1]}


def _rows_of(s, page_of):
    """fp32 K and V [queries, kv_heads, listed rows, head_dim] of listed pages [queries, kv_heads, n] (-1: any)."""
    h = torch.arange(s["kv_heads"], device="cuda")[:, None]
    x = s["data"][page_of.long(), h]                  # [queries, kv_heads, n, 2, page, head_dim]
    return x[..., 0, :, :].flatten(2, 3).float(), x[..., 1, :, :].flatten(2, 3).float()


def _softmax_of(s, k, v, hidden):
    """Attention of each query's heads over listed rows; hidden [queries, kv_heads, rows]."""
    group = s["heads"] // s["kv_heads"]
    q = s["q"].float().unflatten(1, (s["kv_heads"], group))
    score = (q / math.sqrt(s["head_dim"])) @ k.transpose(-1, -2)
    score.masked_fill_(hidden[:, :, None], -math.inf)
    p = (score - score.amax(-1, keepdim=True)).exp_()
    out = (p @ v) / p.sum(-1, keepdim=True)
    return out.flatten(1, 2).to(s["q"].dtype)


def _attend(s):
    seq = s["sequences"].long()
    k, v = _rows_of(s, s["table"][seq][:, None].expand(-1, s["kv_heads"], -1))
    hidden = torch.arange(k.shape[2], device="cuda") > s["positions"][:, None]
    return {"out": _softmax_of(s, k, v, hidden[:, None].expand(-1, s["kv_heads"], -1))}


def _sparse(s):
    page, group = s["page"], s["heads"] // s["kv_heads"]
    table = s["table"][s["sequences"].long()]
    count = s["positions"] // page + 1                      # pages of each query's rows
    q = s["q"].double().unflatten(1, (s["kv_heads"], group))
    up, down = q.clamp_min(0).sum(2), q.clamp_max(0).sum(2)     # [queries, kv_heads, head_dim]
    ends = s["summaries_of"][table.long()].permute(0, 2, 1, 3, 4)     # [queries, kv_heads, pages, 2, head_dim]
    score = (torch.matmul(ends[..., 0, :].double(), down[..., None]) + torch.matmul(ends[..., 1, :].double(), up[..., None]))[..., 0]
    col = torch.arange(table.shape[1], device="cuda")
    forced = (col < s["sinks"]) | (col >= count[:, None] - s["recent"])
    score = torch.where(forced[:, None], math.inf, score)
    score = torch.where((col < count[:, None])[:, None], score, -math.inf)
    order = score.argsort(dim=-1, descending=True, stable=True)[..., :s["budget"]]
    order = torch.where(order < count[:, None, None], order, table.shape[1]).sort(-1).values
    chosen = torch.where(order < count[:, None, None], order, -1).int()
    chosen = torch.nn.functional.pad(chosen, (0, s["budget"] - chosen.shape[-1]), value=-1)
    listed_page = table[:, None].expand(-1, s["kv_heads"], -1).gather(2, chosen.clamp_min(0).long())
    k, v = _rows_of(s, listed_page)
    row = chosen[..., None] * page + torch.arange(page, device="cuda")
    hidden = (chosen < 0)[..., None] | (row > s["positions"][:, None, None, None])
    return {"chosen": chosen, "out": _softmax_of(s, k, v, hidden.flatten(2))}


def run(state):
    if own:
        return _run_own(state)
    return {"table": _table, "append": _append, "attend": _attend, "sparse": _sparse}[state["op"]](state)


# --------------------------------------------------------------------------------------------
# 64-bit values
# --------------------------------------------------------------------------------------------
def _exact_append(case, s):
    held, page = s["rows"].tolist(), case["page"]       # rows after the step
    data = s["data"][:-1].double()
    ends = torch.zeros(s["pages"], case["kv_heads"], 2, case["head_dim"], dtype=torch.float64, device="cuda")
    first, table = s["step"]["starts"].tolist(), s["table"].tolist()
    k, v = s["k"].double(), s["v"].double()
    for i, n in enumerate(held):
        start = n - (first[i + 1] - first[i])
        for c in range(start // page, _pages(n, page)):
            a, b = max(start, c * page), min(n, (c + 1) * page)
            token = first[i] + a - start
            p = table[i][c]
            data[p, :, 0, a - c * page:b - c * page] = k[token:token + b - a].transpose(0, 1)
            data[p, :, 1, a - c * page:b - c * page] = v[token:token + b - a].transpose(0, 1)
            if case["summaries"]:
                x = data[p, :, 0, :b - c * page]
                ends[p, :, 0], ends[p, :, 1] = x.min(1)[0], x.max(1)[0]
    return {"data": data, "summaries": ends} if case["summaries"] else {"data": data}


def exact(case, seed):
    if case["op"] == "table":
        return None
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(case, s)
    page, d, group = case["page"], case["head_dim"], case["heads"] // case["kv_heads"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, (seq, pos) in enumerate(zip(s["sequences"].tolist(), s["positions"].tolist())):
        mine = s["table"][seq, :pos // page + 1].long()
        for h in range(case["kv_heads"]):
            q = s["q"][i, h * group:(h + 1) * group].double()
            take = torch.arange(len(mine), device="cuda")
            if case["op"] == "sparse" and len(mine) > case["budget"]:
                ends = s["summaries_of"][mine, h].double()
                bound = torch.zeros(len(mine), dtype=torch.float64, device="cuda")
                for one in q:
                    bound += torch.maximum(one * ends[:, 0], one * ends[:, 1]).sum(-1)
                sure = (take < case["sinks"]) | (take >= len(mine) - case["recent"])
                rest = case["budget"] - int(sure.sum())
                best = bound.masked_fill(sure, -math.inf).topk(rest)[1] if rest else take[:0]
                sure[best] = True
                take = take[sure]
            x = s["data"][mine[take], h].double()
            row = (take[:, None] * page + torch.arange(page, device="cuda")).flatten()
            k, v = (x[:, j].flatten(0, 1)[row <= pos] for j in (0, 1))
            out[i, h * group:(h + 1) * group] = (q @ k.T * d ** -0.5).softmax(-1) @ v
    return {"out": out} if case["op"] == "attend" else {"chosen": None, "out": out}
