"""Cases, plain forms and 64-bit results of the serving operators over a paged 8-bit KV cache.

The operators of one serving step: ``append`` writes new keys and values into
pages with one scale for each page and head, ``attend`` reads them, the page
operations (copy-on-write fork, free, compaction) keep the book of who holds
which page, and ``verify`` checks drafted tokens.  ``run`` computes them in
plain torch operations, or, with ``own`` set, through ``cuda_b200``.

The cache is the tensors a serving program holds: pools ``k_pages`` and
``v_pages`` (layers, pages, kv_heads, page, head_size) of int8 or e4m3,
``k_scale`` and ``v_scale`` (layers, pages, kv_heads) float32, and one int32
``book``: the table (slots, columns) of page ids, the lengths (slots), the
reference counts (pages), the stack of free pages (pages) and its height.
"""

import math
import sys

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
STORAGE = {"int8": torch.int8, "float8_e4m3": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "float8_e4m3": 448.0}
TINY = 2.0 ** -110  # a block whose scale would be smaller holds zeros
UNIT = 2.0 ** 40  # fixed-point one of the sampling weights
#: query heads, kv heads and head size: the tiny, TinyLlama and Llama-3 shapes, no sharing, and one shared head
HEADS = ((8, 2, 32), (32, 4, 64), (32, 8, 128), (16, 16, 64), (32, 1, 128))


# ---- the cases ---------------------------------------------------------------


def attend(name, batch, tokens, heads, kv_heads, head_size, context, page, storage, dtype, ragged, idle):
    return {"name": name, "op": "attend", "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
            "head_size": head_size, "context": context, "page": page, "storage": storage, "dtype": dtype,
            "ragged": ragged, "idle": idle}


def append(name, batch, tokens, kv_heads, head_size, context, page, storage, dtype, ragged):
    return {"name": name, "op": "append", "batch": batch, "tokens": tokens, "kv_heads": kv_heads,
            "head_size": head_size, "context": context, "page": page, "storage": storage, "dtype": dtype,
            "ragged": ragged}


def pages(name, what, batch, shared, context, layers, kv_heads, head_size, page, spare):
    return {"name": name, "op": "pages", "what": what, "batch": batch, "shared": shared, "context": context,
            "layers": layers, "kv_heads": kv_heads, "head_size": head_size, "page": page, "spare": spare}


def verify(name, batch, tokens, vocab, dtype):
    return {"name": name, "op": "verify", "batch": batch, "tokens": tokens, "vocab": vocab, "dtype": dtype}


def listed():
    return [
        # one user's next token late in a short chat: the smallest call, all latency (float32, the graphs' own type)
        attend("attend_one", 1, 1, 32, 4, 64, 384, 16, "int8", "float32", False, False),
        # a batch of chats of all lengths, one slot idle
        attend("attend_batch", 32, 1, 32, 8, 128, 4096, 64, "int8", "bfloat16", True, True),
        # two very long documents: few rows, a long axis, an odd end
        attend("attend_long", 2, 1, 32, 8, 128, 131067, 64, "float8_e4m3", "bfloat16", False, False),
        # a block of four drafted tokens and the one before them, checked by the target model
        attend("attend_draft", 16, 5, 32, 8, 128, 8191, 32, "int8", "float16", True, False),
        # one new token for each of a batch: latency, and now and then a page whose scale grows
        append("append_token", 32, 1, 8, 128, 1024, 64, "int8", "bfloat16", True),
        # eight prompts of 2048 tokens, as the prefill leaves them
        append("append_prompt", 8, 2048, 8, 128, 2048, 64, "float8_e4m3", "bfloat16", False),
        # chunks of prompts of unlike lengths behind what the slots hold already
        append("append_ragged", 6, 517, 4, 64, 2048, 16, "int8", "float32", True),
        # four prompts continued four ways each: tables forked, then a token's room with copies of the open pages
        pages("fork", "fork", 4, 4, 1001, 22, 4, 64, 16, 64),
        # half of a batch that shares its system prompt ends
        pages("free", "free", 64, 32, 2040, 1, 4, 64, 16, 256),
        # half of the sequences have ended; the rest moves to the front of the pool
        pages("compact", "compact", 32, 0, 2048, 16, 8, 128, 32, 0),
        # four drafted tokens of one user
        verify("verify_one", 1, 4, 32000, "float32"),
        # seven drafted tokens for each of a large batch, a large vocabulary
        verify("verify_batch", 64, 7, 128256, "float32"),
    ]


def draw(rng):
    def spread(lo, hi):
        n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        return n + 1 if n == 3072 else n

    op = rng.choice(("attend", "attend", "append", "append", "pages", "verify"))
    heads, kv_heads, head_size = rng.choice(HEADS)
    page = rng.choice((16, 32, 64, 128))
    storage = rng.choice(sorted(STORAGE))
    dtype = rng.choice(sorted(DTYPES))
    if op == "attend":
        batch, tokens = spread(1, 64), rng.choice((1, 1, 2, 3, 4, 5, 7, 8))
        top = max(256, min(131072, 200_000_000 // (batch * kv_heads * head_size * max(1, tokens * heads // kv_heads // 8))))
        case = attend("", batch, tokens, heads, kv_heads, head_size, spread(tokens, top), page, storage, dtype,
                      rng.random() < 0.7, rng.random() < 0.3)
    elif op == "append":
        batch, tokens = spread(1, 64), spread(1, 2048)
        tokens = min(tokens, max(1, 16384 // batch))
        case = append("", batch, tokens, kv_heads, head_size, tokens + spread(1, 2048), page, storage, dtype,
                      rng.random() < 0.5)
    elif op == "pages":
        what = rng.choice(("fork", "free", "compact"))
        if what == "fork":
            case = pages("", what, spread(1, 8), spread(1, 8), spread(2, 2048), spread(1, 22), kv_heads, head_size,
                         page, spread(64, 256))
        elif what == "free":
            case = pages("", what, spread(2, 64), spread(1, 64), spread(64, 4096), 1, kv_heads, head_size, page,
                         spread(16, 256))
        else:
            case = pages("", what, spread(2, 32), 0, spread(64, 2048), spread(1, 16), kv_heads, head_size, page,
                         spread(1, 64))
    else:
        case = verify("", spread(1, 64), rng.randint(1, 8), spread(500, 128256), dtype)
    del case["name"]
    return case


def lengths_of(case):
    """Tokens of each slot: the context, or for ragged ones a spread below it that starts with the context."""
    new = case.get("tokens", 1)
    if not case.get("ragged"):
        return [case["context"]] * case["batch"]
    share = [0.2 + 0.8 * (1.0 - (b * 0.6180339887498949) % 1.0) for b in range(case["batch"])]
    return [max(new, int(case["context"] * f)) for f in share]


def counts_of(case):
    """New tokens of each slot (the last ones of its length): all, and for appended chunks of ragged ones fewer."""
    if case["op"] == "append" and case["ragged"]:
        return [max(1, case["tokens"] - b * 37 % case["tokens"]) for b in range(case["batch"])]
    if case["op"] == "attend" and case["idle"] and case["batch"] > 1:
        return [0 if b == 1 else case["tokens"] for b in range(case["batch"])]
    return [case["tokens"]] * case["batch"]


def held(case):
    """Lengths with the idle slot empty."""
    return [0 if n == 0 else m for m, n in zip(lengths_of(case), counts_of(case))]


def ceil_div(a, b):
    return -(-a // b)


# ---- what a program has in hand ------------------------------------------------


def pool(shape, storage, gen):
    """Values of a cache as quantised normal keys and values are; a few at the ends of the range."""
    top = TOP[storage]
    if storage == "int8":
        x = torch.empty(shape, dtype=torch.float16, device="cuda")
        for part in x.view(-1).split(1 << 28):
            part.normal_(generator=gen)
        return x.mul_(36.0).round_().clamp_(-top, top).to(torch.int8)
    x = torch.empty(shape, dtype=torch.float16, device="cuda")
    for part in x.view(-1).split(1 << 28):
        part.normal_(generator=gen)
    return x.mul_(128.0).clamp_(-top, top).to(torch.float8_e4m3fn)


def scales(shape, storage, gen):
    """Scales of blocks whose largest value is about 3.5 deviations, of deviations about one."""
    x = torch.randn(shape, device="cuda", generator=gen)
    return (0.25 * x).exp_() * (3.5 / TOP[storage])


def book_of(table, lengths, refs, free, height):
    """One int32 tensor with the table, lengths, reference counts, free stack and its height one after the other."""
    parts = [table.reshape(-1), lengths, refs, free, torch.tensor([height], device=table.device)]
    return torch.cat([p.to(torch.int32) for p in parts])


def views(s):
    """The parts of the book."""
    slots, columns, total = s["slots"], s["columns"], s["k_pages"].shape[1]
    at = slots * columns
    book = s["book"]
    return (book[:at].view(slots, columns), book[at:at + slots], book[at + slots:at + slots + total],
            book[at + slots + total:at + slots + 2 * total], book[at + slots + 2 * total:])


def simple_book(lens, page, gen, spare=3):
    """A book whose slots hold pages of their own, scattered over the pool."""
    need = torch.tensor([ceil_div(n, page) for n in lens], device="cuda")
    used, columns = int(need.sum()), max(1, int(need.max()))
    total = used + spare
    ids = torch.randperm(total, device="cuda", generator=gen)
    first = need.cumsum(0) - need
    column = torch.arange(columns, device="cuda")
    at = (first[:, None] + column).clamp(max=total - 1)
    table = torch.where(column < need[:, None], ids[at], -1)
    refs = torch.zeros(total, dtype=torch.int64, device="cuda")
    refs[ids[:used]] = 1
    free = torch.zeros(total, dtype=torch.int64, device="cuda")
    free[:spare] = ids[used:]
    return book_of(table, torch.tensor(lens, device="cuda"), refs, free, spare), columns, total


def shared_book(case, gen):
    """A book for the page operations, and the slots that they are called with."""
    page, ctx, batch = case["page"], case["context"], case["batch"]
    need = ceil_div(ctx, page)
    if case["what"] == "fork":  # `batch` parents, and `shared` empty slots for each
        slots, own_pages, prefix = batch * (1 + case["shared"]), need, 0
        lens = [ctx] * batch + [0] * (slots - batch)
        columns = ceil_div(ctx + 1, page)
        spare = case["spare"] + slots * 2
    else:  # the first pages of all slots are the same ones
        prefix = min(case["shared"], need - 1)
        slots, own_pages, spare = batch, need - prefix, case["spare"]
        lens, columns = [ctx] * batch, need
    used = prefix + own_pages * batch
    total = used + spare
    ids = torch.randperm(total, device="cuda", generator=gen)
    row = torch.arange(batch, device="cuda")[:, None]
    column = torch.arange(columns, device="cuda")[None]
    at = torch.where(column < prefix, column + 0 * row, prefix + row * own_pages + column - prefix)
    table = torch.full((slots, columns), -1, dtype=torch.int64, device="cuda")
    table[:batch] = torch.where(column < need, ids[at.clamp(max=total - 1)], -1)
    refs = torch.zeros(total, dtype=torch.int64, device="cuda")
    refs[ids[:used]] = 1
    refs[ids[:prefix]] = batch
    height = spare
    free = torch.zeros(total, dtype=torch.int64, device="cuda")
    free[:spare] = ids[used:]
    if case["what"] == "compact":  # every second slot has ended, and its pages are on the stack
        gone = ids[prefix:used].view(batch, own_pages)[::2].reshape(-1)
        refs[gone] = 0
        free[spare:spare + gone.numel()] = gone
        height += gone.numel()
        table[:batch:2] = -1
        lens = [0 if b % 2 == 0 else n for b, n in enumerate(lens)]
    return book_of(table, torch.tensor(lens, device="cuda"), refs, free, height), slots, columns, total


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case, "op": case["op"]}
    if case["op"] == "verify":
        return s | prepare_verify(case, gen)
    storage = case.get("storage", "int8")
    if case["op"] == "pages":
        s["book"], s["slots"], s["columns"], total = shared_book(case, gen)
        s["saved"] = s["book"].clone()
        layers = case["layers"]
    else:
        s["book"], s["columns"], total = simple_book(held(case), case["page"], gen)
        s["slots"], layers = case["batch"], 1
    shape = (layers, total, case["kv_heads"], case["page"], case["head_size"])
    if case["op"] == "pages":
        s["k_pages"] = torch.randint(-127, 128, shape, dtype=torch.int8, device="cuda", generator=gen)
        s["v_pages"] = torch.randint(-127, 128, shape, dtype=torch.int8, device="cuda", generator=gen)
    else:
        s["k_pages"], s["v_pages"] = pool(shape, storage, gen), pool(shape, storage, gen)
    s["k_scale"], s["v_scale"] = scales(shape[:3], storage, gen), scales(shape[:3], storage, gen)
    dtype = DTYPES[case.get("dtype", "float32")]
    batch = case["batch"]
    if case["op"] == "attend":
        # queries as the rope step leaves them; deviation 2, so that some keys stand out
        shape = (batch, case["tokens"], case["heads"], case["head_size"])
        s["q"] = (2.0 * torch.randn(shape, device="cuda", generator=gen)).to(dtype)
        s["counts"] = torch.tensor(counts_of(case), dtype=torch.int32, device="cuda")
    elif case["op"] == "append":
        # keys and values as slices of the rows that one projection writes
        width = case["kv_heads"] * case["head_size"]
        rows = torch.randn(batch, case["tokens"], 2 * width, device="cuda", generator=gen).to(dtype)
        split = (batch, case["tokens"], case["kv_heads"], case["head_size"])
        s["k"], s["v"] = rows[..., :width].view(split), rows[..., width:].view(split)
        s["counts"] = torch.tensor(counts_of(case), dtype=torch.int32, device="cuda")
    elif case["what"] == "fork":
        parents = torch.arange(batch, dtype=torch.int32, device="cuda")
        s["parents"] = parents.repeat_interleave(case["shared"])
        s["children"] = torch.arange(batch, s["slots"], dtype=torch.int32, device="cuda")
        s["counts"] = torch.ones(s["slots"], dtype=torch.int32, device="cuda")
    elif case["what"] == "free":
        s["ending"] = torch.arange(0, batch, 2, dtype=torch.int32, device="cuda")
    if own:  # the handle that a program keeps with these tensors; it holds them as they are
        s["cache"] = package("paged").PagedCache(s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"], s["book"],
                                                 sequences=s["slots"], pages_per_sequence=s["columns"])
    return s


def prepare_verify(case, gen):
    """Probabilities of two models that mostly agree, tokens drawn from the draft's, and uniform numbers."""
    batch, n, vocab, dtype = case["batch"], case["tokens"], case["vocab"], DTYPES[case["dtype"]]
    logits = 2.5 * torch.randn(batch, n + 1, vocab, device="cuda", generator=gen)
    noise = 0.5 * torch.randn(batch, n, vocab, device="cuda", generator=gen)
    target, draft = torch.softmax(logits, -1), torch.softmax(logits[:, :n] + noise, -1)
    del logits, noise
    tokens = torch.multinomial(draft.view(batch * n, vocab), 1, generator=gen).view(batch, n)
    return {"target": target.to(dtype), "draft": draft.to(dtype), "tokens": tokens,
            "uniforms": torch.rand(batch, n + 1, dtype=torch.float64, device="cuda", generator=gen)}


def package(name):
    """A module of this repository's package."""
    import importlib

    if "chomik-grad_b200" not in sys.path:
        sys.path.insert(0, "chomik-grad_b200")
    return importlib.import_module("cuda_b200." + name)


# ---- one pass ----------------------------------------------------------------


def run(s):
    if s["op"] == "attend":
        if own:
            return s["cache"].attend(0, s["q"], counts=s["counts"])
        return plain_attend(s)
    if s["op"] == "append":
        if own:
            s["cache"].append(0, s["k"], s["v"], counts=s["counts"])
        else:
            plain_append(s)
        return {"k_pages": s["k_pages"], "v_pages": s["v_pages"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if s["op"] == "verify":
        if own:
            return package("speculative").verify(s["target"], s["draft"], s["tokens"], s["uniforms"])
        return plain_verify(s)
    # the book as the scheduler's step finds it, then the step
    s["book"].copy_(s["saved"])
    what = s["case"]["what"]
    if own:
        cache = s["cache"]
        if what == "fork":
            cache.fork(s["parents"], s["children"])
            cache.extend(s["counts"])
        elif what == "free":
            cache.release(s["ending"])
        else:
            cache.compact()
    elif what == "fork":
        plain_fork(s)
        plain_extend(s)
    elif what == "free":
        plain_release(s)
    else:
        plain_compact(s)
    if what == "free":
        return {"book": s["book"]}
    return {"book": s["book"], "k_pages": s["k_pages"], "v_pages": s["v_pages"], "k_scale": s["k_scale"],
            "v_scale": s["v_scale"]}


def raw(pages_):
    """The pool's bytes: what indexing moves."""
    return pages_.view(torch.int8)


def read(pages_, scale, table):
    """float32 (batch, kv_heads, columns * page, head_size) of layer 0's pages of each slot."""
    at = table.clamp(min=0).long()
    x = raw(pages_[0])[at].view(pages_.dtype).float() * scale[0][at][..., None, None]
    return x.transpose(1, 2).flatten(2, 3)


def plain_attend(s):
    q, counts = s["q"], s["counts"].long()
    table, lengths = views(s)[:2]
    k, v = read(s["k_pages"], s["k_scale"], table), read(s["v_pages"], s["v_scale"], table)
    batch, tokens, heads, size = q.shape
    kv_heads, span = k.shape[1], k.shape[2]
    where, t = torch.arange(span, device=q.device), torch.arange(tokens, device=q.device)
    v = torch.where((where < lengths[:, None])[:, None, :, None], v, 0.0)
    limit = torch.where(t < counts[:, None], (lengths - counts)[:, None] + t + 1, 0)
    seen = (where < limit[..., None])[:, None, :, None]  # (batch, 1, tokens, 1, span)
    rows = q.float().view(batch, tokens, kv_heads, heads // kv_heads, size).transpose(1, 2)
    score = (rows.flatten(2, 3) @ k.transpose(2, 3)).view(*rows.shape[:4], span) * (1.0 / math.sqrt(size))
    score = torch.where(seen, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.where(seen, torch.exp(score - torch.where(seen.any(-1, keepdim=True), top, 0.0)), 0.0)
    total = e.sum(-1, keepdim=True)
    out = (e.flatten(2, 3) @ v).view(rows.shape) / torch.where(total == 0, 1.0, total)
    return out.transpose(1, 2).reshape(q.shape).to(q.dtype)


def plain_append(s):
    table, lengths = views(s)[:2]
    plain_append_one(s["k"], s["k_pages"], s["k_scale"], table, lengths, s["counts"])
    plain_append_one(s["v"], s["v_pages"], s["v_scale"], table, lengths, s["counts"])


def plain_append_one(x, pages_, scale, table, lengths, counts):
    storage = "int8" if pages_.dtype == torch.int8 else "float8_e4m3"
    top, page = TOP[storage], pages_.shape[3]
    batch, tokens = x.shape[:2]
    end = lengths.long()
    start = end - counts
    # the pages that the new tokens touch: (batch, slots) of them, and the position of each of their rows
    slot = start[:, None] // page + torch.arange((tokens + page - 2) // page + 1, device=x.device)
    used = slot * page < end[:, None]
    ids = table.gather(1, slot.clamp(max=table.shape[1] - 1).long())[used].long()
    position = slot[..., None] * page + torch.arange(page, device=x.device)
    new = (position >= start[:, None, None]) & (position < end[:, None, None])
    old = position < start[:, None, None]
    at = torch.where(new, position - start[:, None, None], 0)
    b = torch.arange(batch, device=x.device)[:, None, None]
    rows = x[b, at][used].float().transpose(1, 2)  # (pages, kv_heads, page, head_size)
    new, old = new[used][:, None, :, None], old[used][:, None, :, None]
    fine = new & torch.isfinite(rows)
    grown = torch.where(fine, rows.abs(), 0.0).amax((2, 3)) / top
    grown = torch.where(grown < TINY, 0.0, grown)
    before = torch.where(old[:, :, 0, 0], scale[0][ids], 0.0)
    after = torch.maximum(before, grown)
    inverse = torch.where(after == 0, 0.0, 1.0 / after)[..., None, None]
    fresh = torch.where(torch.isnan(rows) | (inverse == 0), 0.0, rows * inverse)
    was = raw(pages_[0])[ids].view(pages_.dtype)
    moved = was.float() * (before[..., None, None] * inverse)
    moved = torch.where((after > before)[..., None, None], moved, was.float())
    value = torch.where(new, fresh, torch.where(old, moved, 0.0)).clamp(-top, top)
    coded = value.round().to(torch.int8) if storage == "int8" else raw(value.to(torch.float8_e4m3fn))
    raw(pages_[0])[ids] = torch.where(new | old, coded, raw(was))
    scale[0][ids] = after


def plain_fork(s):
    table, lengths, refs = views(s)[:3]
    parents, children = s["parents"].long(), s["children"].long()
    rows = table[parents]
    table[children] = rows
    lengths[children] = lengths[parents]
    refs.scatter_add_(0, rows.clamp(min=0).long().view(-1), (rows >= 0).to(torch.int32).view(-1))


def plain_extend(s):
    page = s["k_pages"].shape[3]
    table, lengths, refs, free, height = views(s)
    counts = s["counts"]
    have, need = (lengths + page - 1) // page, (lengths + counts + page - 1) // page
    # an open last page that others hold too is copied; the last of its holders to write keeps it
    open_ = (lengths % page != 0) & (counts > 0)
    last = (have - 1).clamp(min=0).long()[:, None]
    tail = torch.where(open_, table.gather(1, last)[:, 0], -1)
    earlier = ((tail[:, None] == tail[None, :]) & open_[None, :]).tril(-1).sum(1)
    at = tail.clamp(min=0).long()
    copied = open_ & (refs[at] - earlier > 1)
    taken = need - have + copied.int()
    first = taken.cumsum(0) - taken
    column = torch.arange(table.shape[1], device=table.device)
    base = (have - copied.int())[:, None]
    fresh = (column >= base) & (column < need[:, None])
    index = height.long() - 1 - (first[:, None] + column - base)
    popped = free[torch.where(fresh, index, 0).clamp(min=0)]
    table.copy_(torch.where(fresh, popped, table))
    refs.scatter_add_(0, at, -copied.int())
    refs.scatter_add_(0, popped.long().view(-1), fresh.to(torch.int32).view(-1))
    source, target = at[copied], table.gather(1, last)[:, 0][copied].long()
    for_each_pool(s, source, target)
    lengths += counts
    height -= taken.sum().int()


def for_each_pool(s, source, target):
    """Pages `source` copied to `target`, in every layer."""
    s["k_pages"][:, target] = s["k_pages"][:, source]
    s["v_pages"][:, target] = s["v_pages"][:, source]
    s["k_scale"][:, target] = s["k_scale"][:, source]
    s["v_scale"][:, target] = s["v_scale"][:, source]


def plain_release(s):
    table, lengths, refs, free, height = views(s)
    ending = s["ending"].long()
    rows = table[ending]
    valid, ids = (rows >= 0).view(-1), rows.clamp(min=0).long().view(-1)
    refs.scatter_add_(0, ids, -valid.int())
    # a page is pushed at the place of its last holder among the rows, the last place first
    place = torch.arange(ids.numel(), device=ids.device)
    final = torch.full_like(refs, -1, dtype=torch.int64)
    final.scatter_reduce_(0, ids, torch.where(valid, place, -1), "amax")
    pushed = valid & (refs[ids] == 0) & (final[ids] == place)
    rank = pushed.flip(0).cumsum(0).flip(0) - 1
    free[(height.long() + rank)[pushed]] = ids[pushed].int()
    height += pushed.sum().int()
    table[ending] = -1
    lengths[ending] = 0


def plain_compact(s):
    table, lengths, refs, free, height = views(s)
    total = refs.numel()
    ids = torch.arange(total, device=refs.device)
    live = refs > 0
    kept = live.sum()
    source, target = ids[live & (ids >= kept)], ids[~live & (ids < kept)]
    to = ids.clone()
    to[source] = target
    for_each_pool(s, source, target)
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()].int(), table))
    refs[target] = refs[source]
    refs[source] = 0
    free.copy_(torch.where(ids < total - kept, total - 1 - ids, free).int())
    height.copy_(total - kept)


def plain_verify(s):
    target, draft, tokens, uniforms = s["target"], s["draft"], s["tokens"], s["uniforms"]
    batch, n = tokens.shape
    p = target[:, :n].gather(2, tokens[..., None])[..., 0].double()
    q = draft.gather(2, tokens[..., None])[..., 0].double()
    taken = (uniforms[:, :n] * q < p).int().cumprod(1)
    accepted = taken.sum(1)
    b = torch.arange(batch, device=tokens.device)
    here = target[b, accepted].float()
    there = torch.where((accepted < n)[:, None], draft[b, accepted.clamp(max=n - 1)].float(), 0.0)
    rest = fixed(here - there)
    weight = torch.where(rest.sum(1, keepdim=True) > 0, rest, fixed(here))
    running = weight.cumsum(1)
    total = running[:, -1]
    bar = (uniforms[:, n] * total.double()).long().minimum(total - 1)
    token = (running > bar[:, None]).int().argmax(1)
    bad = torch.isnan(here).any(1) | torch.isnan(there).any(1) | (total == 0)
    token = torch.where(bad, -1, token)
    column = torch.arange(n + 1, device=tokens.device)
    padded = torch.cat([tokens, tokens[:, :1]], 1)
    out = torch.where(column < accepted[:, None], padded, torch.where(column == accepted[:, None], token[:, None], -1))
    return accepted.int(), out


def fixed(x):
    """Fixed-point weights: sums of them are exact, whatever their order."""
    return (torch.where(x > 0, x, 0.0).clamp(max=1.0) * UNIT).long()


# ---- in 64 bits ----------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attend":
        return exact_attend(case, s)
    if case["op"] == "append":
        k_pages, k_scale = exact_append(case, s, "k")
        v_pages, v_scale = exact_append(case, s, "v")
        return {"k_pages": k_pages, "v_pages": v_pages, "k_scale": k_scale, "v_scale": v_scale}
    return None  # whole numbers, and bytes that are moved


def exact_attend(case, s):
    q, table = s["q"].double(), s["book"][:s["slots"] * s["columns"]].view(s["slots"], s["columns"])
    out = torch.zeros_like(q)
    group = case["heads"] // case["kv_heads"]
    for b, (length, n) in enumerate(zip(held(case), counts_of(case))):
        used = table[b, :ceil_div(length, case["page"])].long()
        for g in range(case["kv_heads"] if n else 0):
            k = (s["k_pages"][0, used, g].double() * s["k_scale"][0, used, g].double()[:, None, None]).flatten(0, 1)
            v = (s["v_pages"][0, used, g].double() * s["v_scale"][0, used, g].double()[:, None, None]).flatten(0, 1)
            for t in range(n):
                end = length - n + t + 1
                score = q[b, t, g * group:(g + 1) * group] @ k[:end].T / math.sqrt(case["head_size"])
                out[b, t, g * group:(g + 1) * group] = torch.softmax(score, -1) @ v[:end]
    return out


def exact_append(case, s, which):
    """The scales, and for e4m3 the numbers before they are rounded (whole numbers have no such value)."""
    page, top = case["page"], TOP[case["storage"]]
    pages_, scale, rows = s[which + "_pages"].double(), s[which + "_scale"].double(), s[which].double()
    table = s["book"][:s["slots"] * s["columns"]].view(s["slots"], s["columns"]).tolist()
    for b, (length, n) in enumerate(zip(held(case), counts_of(case))):
        start = length - n
        for column in range(start // page, ceil_div(length, page)):
            one = table[b][column]
            lo, hi = max(start, column * page), min(length, (column + 1) * page)
            x = rows[b, lo - start:hi - start].transpose(0, 1)  # (kv_heads, rows, head_size)
            before = scale[0, one].clone() if lo > column * page else torch.zeros_like(scale[0, one])
            after = torch.maximum(before, x.abs().amax((1, 2)) / top)
            pages_[0, one, :, :lo - column * page] *= (before / after)[:, None, None]
            pages_[0, one, :, lo - column * page:hi - column * page] = x / after[:, None, None]
            scale[0, one] = after
    return (None if case["storage"] == "int8" else pages_), scale


# ---- what a pass cannot do without -----------------------------------------------


def work(case):
    item = {"float32": 4, "bfloat16": 2, "float16": 2}[case.get("dtype", "float32")]
    if case["op"] == "attend":
        rows = case["heads"] * case["head_size"]
        tokens, keys = sum(counts_of(case)), sum(held(case))
        blocks = sum(ceil_div(n, case["page"]) for n in held(case))
        size = 2 * keys * case["kv_heads"] * case["head_size"] + blocks * (8 * case["kv_heads"] + 4)
        size += (tokens + case["batch"] * case["tokens"]) * rows * item
        return {"bytes": size, "flops": 4 * sum(n * m for n, m in zip(held(case), counts_of(case))) * rows}
    if case["op"] == "append":
        width = case["kv_heads"] * case["head_size"]
        tokens = sum(counts_of(case))
        blocks = sum(ceil_div(m, case["page"]) - (m - n) // case["page"] for m, n in zip(held(case), counts_of(case)))
        return {"bytes": 2 * tokens * width * (item + 1) + blocks * (8 * case["kv_heads"] + 4),
                "flops": 4 * tokens * width}
    if case["op"] == "verify":
        # the target's row that is drawn from, and the draft's where a token is refused (three of four are accepted)
        rows = case["batch"] * (2.0 - 0.75 ** case["tokens"])
        return {"bytes": rows * case["vocab"] * item + case["batch"] * case["tokens"] * (2 * item + 24),
                "flops": 4 * rows * case["vocab"]}
    need = ceil_div(case["context"], case["page"])
    one = case["layers"] * 2 * case["kv_heads"] * (case["page"] * case["head_size"] + 4)
    if case["what"] == "fork":
        children = case["batch"] * case["shared"]
        copies = children if case["context"] % case["page"] else 0
        return {"bytes": 2 * copies * one + children * need * 12}
    if case["what"] == "free":
        return {"bytes": (case["batch"] + 1) // 2 * need * 16}
    # a live page lies beyond the live ones' number with the share of free pages
    live = case["batch"] // 2 * need
    total = case["batch"] * need + case["spare"]
    return {"bytes": 2 * live * (total - live) / total * one + 4 * (case["batch"] * need * 2 + 3 * total)}
