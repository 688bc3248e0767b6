"""Cases, plain forms and 64-bit results of the operators for many samples of one prompt.

One decoding step of a batch whose sequences begin alike, with small weights and
constrained tokens: ``linear`` multiplies rows by 4-bit weights with group
scales, ``dequantise`` gives the same weights to a prefill's large products,
``attend_shared`` reads the pages that all sequences of a paged 8-bit cache have
in common once for all of them, and ``adjust`` applies penalties, biases and a
grammar's mask to the logits.  ``run`` computes them in plain torch operations,
or, with ``own`` set, through ``cuda_b200``.
"""

import math
import sys

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
TOP = {"int8": 127.0, "float8_e4m3": 448.0}
#: query heads, kv heads and head size: the tiny, TinyLlama and Llama-3 shapes, no sharing, and one shared head
HEADS = ((8, 2, 32), (32, 4, 64), (32, 8, 128), (16, 16, 64), (32, 1, 128))


# ---- the cases ---------------------------------------------------------------


def attend(name, batch, tokens, heads, kv_heads, head_size, prefix, tail, page, storage, dtype, idle):
    return {"name": name, "op": "attend_shared", "batch": batch, "tokens": tokens, "heads": heads,
            "kv_heads": kv_heads, "head_size": head_size, "prefix": prefix, "tail": tail, "page": page,
            "storage": storage, "dtype": dtype, "idle": idle}


def adjust(name, batch, vocab, history, biases, grammar, dtype):
    return {"name": name, "op": "adjust", "batch": batch, "vocab": vocab, "history": history, "biases": biases,
            "grammar": grammar, "dtype": dtype}


def linear(name, rows, inputs, outputs, group, dtype, scales):
    return {"name": name, "op": "linear", "rows": rows, "inputs": inputs, "outputs": outputs, "group": group,
            "dtype": dtype, "scales": scales}


def dequantise(name, inputs, outputs, group, dtype, scales):
    return {"name": name, "op": "dequantise", "inputs": inputs, "outputs": outputs, "group": group, "dtype": dtype,
            "scales": scales}


def listed():
    return [
        # four answers to one short question, just begun: the smallest call, all latency (float32, the graphs' own type)
        attend("shared_few", 4, 1, 32, 4, 64, 500, 40, 16, "int8", "float32", False),
        # 64 samples of one long prompt, of unlike lengths, one slot idle
        attend("shared_samples", 64, 1, 32, 8, 128, 16384, 700, 64, "int8", "bfloat16", True),
        # users of one long document, each with a block of four drafted tokens and the one before them
        attend("shared_drafted", 16, 5, 32, 8, 128, 32700, 500, 32, "float8_e4m3", "float16", False),
        # one user's next token: penalties and a few biases, all latency
        adjust("adjust_one", 1, 32000, 300, 8, False, "float32"),
        # a batch under grammars, long histories, a large vocabulary
        adjust("adjust_grammar", 64, 128256, 4000, 64, True, "bfloat16"),
        # drafted blocks that a grammar filters, an odd vocabulary, no history
        adjust("adjust_odd", 80, 32003, 0, 0, True, "float16"),
        # the query projection of a small model: the smallest product, all latency
        linear("linear_query", 1, 2048, 2048, 32, "bfloat16", "bfloat16"),
        # the widest projection of a larger one, one user
        linear("linear_gate", 1, 4096, 14336, 128, "bfloat16", "bfloat16"),
        # a drafted block of five rows through the narrow end of an MLP, float32 activations
        linear("linear_down", 5, 5632, 2048, 64, "float32", "float16"),
        # the vocabulary's projection for a batch: the largest
        linear("linear_vocabulary", 16, 4096, 128256, 128, "float16", "float16"),
        # weights of a prompt's large products: a small and a large one
        dequantise("dequantise_query", 2048, 2048, 32, "bfloat16", "bfloat16"),
        dequantise("dequantise_gate", 4096, 14336, 128, "bfloat16", "bfloat16"),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(("attend_shared", "attend_shared", "adjust", "linear", "linear", "dequantise"))
    dtype = rng.choice(sorted(DTYPES))
    if op == "attend_shared":
        heads, kv_heads, head_size = rng.choice(HEADS)
        batch, tokens = spread(2, 64), rng.choice((1, 1, 1, 2, 3, 5, 8))
        # no more keys than a pool of the largest case has, and no more products
        keys = min(33_000_000 // (kv_heads * head_size), 10_000_000_000 // (batch * tokens * heads * head_size))
        tail = spread(tokens, max(tokens, min(1000, keys // (4 * batch))))
        page = rng.choice((16, 32, 64, 128))
        prefix = spread(page, max(2 * page, min(65536, keys - tail * batch)))
        case = attend("", batch, tokens, heads, kv_heads, head_size, prefix, tail, page, rng.choice(sorted(TOP)),
                      dtype, rng.random() < 0.3)
    elif op == "adjust":
        history, biases = rng.choice((0, 1)) * spread(1, 4000), rng.choice((0, 1)) * spread(1, 256)
        case = adjust("", spread(1, 64), spread(500, 128256), history, biases,
                      history + biases == 0 or rng.random() < 0.6, dtype)
    else:
        group = rng.choice((32, 64, 128))
        inputs = group * spread(1, 14336 // group)
        outputs = spread(64, min(128256, (58_000_000 if rng.random() < 0.8 else 500_000_000) // inputs))
        scales = rng.choice(("bfloat16", "float16"))
        if op == "linear":
            case = linear("", spread(1, 40), inputs, outputs, group, dtype, scales)
        else:
            case = dequantise("", inputs, min(outputs, 58_000_000 // inputs), group, dtype, scales)
    del case["name"]
    return case


def ceil_div(a, b):
    return -(-a // b)


def counts_of(case):
    """New tokens of each slot: all of them, and none of the second where one is idle."""
    return [0 if case["idle"] and b == 1 else case["tokens"] for b in range(case["batch"])]


def shared_pages(case):
    """Pages that every slot holds: the whole ones of the prefix."""
    return case["prefix"] // case["page"]


def lengths_of(case):
    """Tokens of each slot: the prefix and a tail of its own, from the new tokens alone to the longest."""
    share = [1.0 - (b * 0.6180339887498949) % 1.0 for b in range(case["batch"])]
    return [case["prefix"] + max(case["tokens"], int(case["tail"] * f)) for f in share]


# ---- what a program has in hand ------------------------------------------------


def pool(shape, storage, gen):
    """Values of a cache as quantised normal keys and values are; a few at the ends of the range."""
    top = TOP[storage]
    x = torch.empty(shape, dtype=torch.float16, device="cuda").normal_(generator=gen)
    if storage == "int8":
        return x.mul_(36.0).round_().clamp_(-top, top).to(torch.int8)
    return x.mul_(128.0).clamp_(-top, top).to(torch.float8_e4m3fn)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case, "op": case["op"]}
    if case["op"] == "attend_shared":
        return s | prepare_attend(case, gen)
    if case["op"] == "adjust":
        return s | prepare_adjust(case, gen)
    return s | prepare_weights(case, gen)


def prepare_attend(case, gen):
    batch, page, shared = case["batch"], case["page"], shared_pages(case)
    lengths = torch.tensor(lengths_of(case), device="cuda")
    need = (lengths + page - 1) // page
    mine = need - shared
    columns = max(ceil_div(n, page) for n in lengths_of(case))
    used = shared + sum(ceil_div(n, page) - shared for n in lengths_of(case))
    total = used + 3
    ids = torch.randperm(total, device="cuda", generator=gen)
    column = torch.arange(columns, device="cuda")
    first = shared + mine.cumsum(0) - mine
    at = torch.where(column < shared, column, first[:, None] + column - shared)
    table = torch.where(column < need[:, None], ids[at.clamp(max=total - 1)], -1)
    refs = torch.zeros(total, dtype=torch.int64, device="cuda")
    refs[ids[:used]] = 1
    refs[ids[:shared]] = batch
    free = torch.zeros(total, dtype=torch.int64, device="cuda")
    free[:3] = ids[used:]
    # the book of the cache: table, lengths, reference counts, the stack of free pages and its height
    book = torch.cat([table.reshape(-1), lengths, refs, free, torch.full_like(free[:1], 3)]).to(torch.int32)
    shape = (1, total, case["kv_heads"], page, case["head_size"])
    s = {"book": book, "columns": columns, "k_pages": pool(shape, case["storage"], gen),
         "v_pages": pool(shape, case["storage"], gen)}
    for name in ("k_scale", "v_scale"):  # of blocks whose largest value is about 3.5 deviations, of deviations about one
        s[name] = (0.25 * torch.randn(shape[:3], device="cuda", generator=gen)).exp_() * (3.5 / TOP[case["storage"]])
    # queries as the rope step leaves them; deviation 2, so that some keys stand out
    q = 2.0 * torch.randn(batch, case["tokens"], case["heads"], case["head_size"], device="cuda", generator=gen)
    s["q"] = q.to(DTYPES[case["dtype"]])
    s["counts"] = torch.tensor(counts_of(case), dtype=torch.int32, device="cuda")
    if own:  # the handle that a program keeps with these tensors; it holds them as they are
        s["cache"] = package("paged").PagedCache(s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"], book,
                                                 sequences=batch, pages_per_sequence=columns)
    return s


def prepare_adjust(case, gen):
    """Logits, the tokens so far (a prompt and what followed it, many of them again), biases and a grammar's mask."""
    batch, vocab, room = case["batch"], case["vocab"], case["history"]
    dev = {"device": "cuda", "generator": gen}
    s = {"logits": (3.0 * torch.randn(batch, vocab, **dev)).to(DTYPES[case["dtype"]])}
    s["history"] = s["bias"] = s["allowed"] = None
    if room:
        tokens = (vocab * torch.rand(batch, room, **dev) ** 3).long().clamp(max=vocab - 1).to(torch.int32)
        lengths = torch.randint(room // 2, room + 1, (batch,), **dev).to(torch.int32)
        prompts = (lengths * torch.rand(batch, **dev)).to(torch.int32)
        s["history"] = (tokens, lengths, prompts)
    s["repetition"] = 1.0 + 0.5 * torch.rand(batch, **dev)
    s["frequency"], s["presence"] = 0.5 * torch.rand(batch, **dev), torch.rand(batch, **dev)
    if case["biases"]:
        tokens = torch.randint(0, vocab, (batch, case["biases"]), **dev).to(torch.int32)
        s["bias"] = (tokens, 4.0 * torch.randn(batch, case["biases"], **dev))
    if case["grammar"]:  # one bit for each token, from few tokens allowed to most
        words = ceil_div(vocab, 32)
        bits = torch.rand(batch, words, 32, **dev) < torch.rand(batch, 1, 1, **dev)
        place = torch.arange(32, device="cuda")
        s["allowed"] = (bits.long() << place).sum(-1).sub((bits[..., 31].long() << 32)).to(torch.int32)
    return s


def prepare_weights(case, gen):
    """Codes of normal weights, two to a byte (the even input in the low half, plus 8), and their scales."""
    inputs, outputs, group = case["inputs"], case["outputs"], case["group"]
    dev = {"device": "cuda", "generator": gen}
    packed = torch.empty(outputs, inputs // 2, dtype=torch.uint8, device="cuda")
    for part in packed.split(max(1, (1 << 26) // inputs)):
        x = torch.randn(part.shape[0], inputs, **dev).mul_(2.7).round_().clamp_(-8, 7).add_(8).to(torch.uint8)
        part.copy_(x[:, ::2] | x[:, 1::2] << 4)
    spread = (0.25 * torch.randn(outputs, inputs // group, **dev)).exp_()
    s = {"packed": packed, "scale": (spread * (0.37 / math.sqrt(inputs))).to(DTYPES[case["scales"]])}
    if case["op"] == "linear":
        s["x"] = torch.randn(case["rows"], inputs, **dev).to(DTYPES[case["dtype"]])
    if own:  # the weights as a program keeps them
        s["weights"] = package("quantized").Weights4.pack(packed, s["scale"])
    return s


def package(name):
    """A module of this repository's package."""
    import importlib

    if "chomik-grad_b200" not in sys.path:
        sys.path.insert(0, "chomik-grad_b200")
    return importlib.import_module("cuda_b200." + name)


# ---- one pass ----------------------------------------------------------------


def run(s):
    if s["op"] == "attend_shared":
        if own:
            return s["cache"].attend_shared(0, s["q"], counts=s["counts"])
        return plain_attend(s)
    if s["op"] == "adjust":
        if own:
            return own_adjust(s)
        return plain_adjust(s)
    if s["op"] == "linear":
        if own:
            return s["weights"].linear(s["x"])
        return (s["x"].float() @ plain_weights(s).T).to(s["x"].dtype)
    dtype = DTYPES[s["case"]["dtype"]]
    if own:
        return s["weights"].dequantise(dtype)
    return plain_weights(s).to(dtype)


def own_adjust(s):
    more = {}
    if s["history"] is not None:
        more = dict(zip(("tokens", "lengths", "prompts"), s["history"]))
        more |= {name: s[name] for name in ("repetition", "frequency", "presence")}
    if s["bias"] is not None:
        more["bias_tokens"], more["bias"] = s["bias"]
    if s["allowed"] is not None:
        more["allowed"] = s["allowed"]
    return package("logits").adjust(s["logits"], **more)


def read(pages, scale, table):
    """float32 (..., kv_heads, columns * page, head_size) of layer 0's pages."""
    at = table.clamp(min=0).long()
    x = pages[0].view(torch.int8)[at].view(pages.dtype).float() * scale[0][at][..., None, None]
    return x.transpose(-4, -3).flatten(-3, -2)


def plain_attend(s):
    """Products of all rows with the shared pages, of each slot's rows with its own, and one softmax over both."""
    q, counts, case = s["q"], s["counts"].long(), s["case"]
    batch, tokens, heads, size = q.shape
    kv_heads, shared, page = case["kv_heads"], shared_pages(case), case["page"]
    table = s["book"][:batch * s["columns"]].view(batch, s["columns"])
    lengths = s["book"][batch * s["columns"]:batch * (s["columns"] + 1)].long()
    rows = q.float().view(batch, tokens, kv_heads, heads // kv_heads, size) * (1.0 / math.sqrt(size))
    k, v = (read(s[x + "_pages"], s[x + "_scale"], table[0, :shared]) for x in "kv")  # (kv_heads, keys, size)
    all_rows = rows.permute(2, 0, 1, 3, 4).flatten(1, 3)
    first = all_rows @ k.transpose(1, 2)
    own_k, own_v = (read(s[x + "_pages"], s[x + "_scale"], table[:, shared:]) for x in "kv")
    own_rows = rows.transpose(1, 2).flatten(2, 3)  # (batch, kv_heads, tokens * group, size)
    second = own_rows @ own_k.transpose(2, 3)
    where, t = shared * page + torch.arange(own_k.shape[2], device=q.device), torch.arange(tokens, device=q.device)
    own_v = torch.where((where < lengths[:, None])[:, None, :, None], own_v, 0.0)
    limit = torch.where(t < counts[:, None], (lengths - counts)[:, None] + t + 1, 0)
    limit = limit.repeat_interleave(heads // kv_heads, 1)  # (batch, tokens * group)
    second = torch.where((where < limit[..., None])[:, None], second, -math.inf)
    first = first.view(kv_heads, batch, -1, k.shape[1]).transpose(0, 1)
    real = (limit > 0)[:, None, :, None]
    top = second.amax(-1, keepdim=True)
    top = torch.maximum(top, first.amax(-1, keepdim=True)) if shared else top
    top = torch.where(real, top, 0.0)
    first, second = torch.exp(first - top), torch.exp(second - top)
    total = first.sum(-1, keepdim=True) + second.sum(-1, keepdim=True)
    out = (first.transpose(0, 1).flatten(1, 2) @ v).view(kv_heads, batch, -1, size).transpose(0, 1) + second @ own_v
    out = torch.where(real, out / total, 0.0)
    return out.view(batch, kv_heads, tokens, -1, size).transpose(1, 2).reshape(q.shape).to(q.dtype)


def plain_adjust(s):
    logits = s["logits"]
    x = logits.float()
    if s["history"] is not None:
        tokens, lengths, prompts = s["history"]
        place = torch.arange(tokens.shape[1], device=x.device)
        held = (place < lengths[:, None]).int()
        made = held * (place >= prompts[:, None])
        seen = torch.zeros(x.shape, dtype=torch.int32, device=x.device).scatter_add_(1, tokens.long(), held) > 0
        count = torch.zeros(x.shape, dtype=torch.int32, device=x.device).scatter_add_(1, tokens.long(), made).float()
        r = s["repetition"][:, None]
        x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
        x = x - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0).float()
    if s["bias"] is not None:
        tokens, bias = s["bias"]
        x = x + torch.zeros_like(x).scatter_add_(1, tokens.long(), bias)
    if s["allowed"] is not None:
        place = torch.arange(32, device=x.device, dtype=torch.int32)
        allowed = (s["allowed"][..., None] >> place & 1).flatten(1)[:, :x.shape[1]] != 0
        x = torch.where(allowed, x, -math.inf)
    return x.to(logits.dtype)


def plain_weights(s):
    packed = s["packed"]
    codes = torch.stack([packed & 15, packed >> 4], -1).flatten(1).float() - 8.0
    return codes * s["scale"].float().repeat_interleave(s["case"]["group"], 1)


# ---- in 64 bits ----------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attend_shared":
        return exact_attend(case, s)
    if case["op"] == "adjust":
        return exact_adjust(case, s)
    scale = s["scale"].double()
    x = s["x"].double() if case["op"] == "linear" else None
    out = []
    for at in range(0, case["outputs"], 4096):
        byte = s["packed"][at:at + 4096].long()
        codes = torch.empty(byte.shape[0], case["inputs"], dtype=torch.float64, device="cuda")
        codes[:, 0::2], codes[:, 1::2] = byte % 16 - 8, byte // 16 - 8
        w = codes.view(byte.shape[0], -1, case["group"]) * scale[at:at + 4096, :, None]
        out.append(w.flatten(1) if x is None else x @ w.flatten(1).T)
    return torch.cat(out, 0 if x is None else 1)


def exact_attend(case, s):
    q = s["q"].double()
    table = s["book"][:case["batch"] * s["columns"]].view(case["batch"], s["columns"])
    out = torch.zeros_like(q)
    group = case["heads"] // case["kv_heads"]
    for b, (length, n) in enumerate(zip(lengths_of(case), counts_of(case))):
        used = table[b, :ceil_div(length, case["page"])].long()
        if n == 0:
            continue
        k, v = ((s[x + "_pages"][0, used].double() * s[x + "_scale"][0, used].double()[..., None, None])
                .transpose(0, 1).flatten(1, 2) for x in "kv")  # (kv_heads, keys, size)
        for t in range(n):
            end = length - n + t + 1
            rows = q[b, t].view(case["kv_heads"], group, -1)
            score = rows @ k[:, :end].transpose(1, 2) / math.sqrt(case["head_size"])
            out[b, t] = (torch.softmax(score, -1) @ v[:, :end]).flatten(0, 1)
    return out


def exact_adjust(case, s):
    x = s["logits"].double()
    for b in range(case["batch"]):
        row = x[b]
        if s["history"] is not None:
            tokens, length, prompt = (a[b] for a in s["history"])
            held, made = tokens[:int(length)].long(), tokens[int(prompt):int(length)].long()
            seen = held.unique()
            r = float(s["repetition"][b])
            row[seen] = torch.where(row[seen] > 0, row[seen] / r, row[seen] * r)
            token, count = made.unique(return_counts=True)
            row[token] -= float(s["frequency"][b]) * count.double() + float(s["presence"][b])
        if s["bias"] is not None:
            row.index_add_(0, s["bias"][0][b].long(), s["bias"][1][b].double())
        if s["allowed"] is not None:
            words = s["allowed"][b].long() & 0xFFFFFFFF
            token = torch.arange(case["vocab"], device=row.device)
            row[(words[token // 32] >> token % 32) % 2 == 0] = -math.inf
    return x


# ---- what a pass cannot do without -----------------------------------------------


def work(case):
    item = {"float32": 4, "bfloat16": 2, "float16": 2}[case["dtype"]]
    if case["op"] == "attend_shared":
        rows, wide = case["heads"] * case["head_size"], case["kv_heads"] * case["head_size"]
        live = [(m, n) for m, n in zip(lengths_of(case), counts_of(case)) if n]
        shared = shared_pages(case)
        keys = shared * case["page"] + sum(m - shared * case["page"] for m, _ in live)
        pages = shared + sum(ceil_div(m, case["page"]) - shared for m, _ in live)
        size = 2 * keys * wide + pages * (8 * case["kv_heads"] + 4) + shared * (len(live) - 1) * 4
        size += (sum(n for _, n in live) + case["batch"] * case["tokens"]) * rows * item
        return {"bytes": size, "flops": 4 * sum(n * m for m, n in live) * rows}
    if case["op"] == "adjust":
        values = case["batch"] * case["vocab"]
        size = 2 * values * item + (values // 8 if case["grammar"] else 0)
        return {"bytes": size + case["batch"] * (4 * case["history"] + 8 * case["biases"]), "flops": 4 * values}
    weights = case["inputs"] * case["outputs"]
    size = weights // 2 + 2 * weights // case["group"]
    if case["op"] == "dequantise":
        return {"bytes": size + weights * item, "flops": weights}
    return {"bytes": size + case["rows"] * (case["inputs"] + case["outputs"]) * item,
            "flops": 2 * case["rows"] * weights}
