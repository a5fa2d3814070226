"""The operators of decoding several sequences over one paged cache, as measurable cases, with their plain forms.

Kinds of case:

attention  attention of new tokens, one or a chunk a sequence, over a paged cache (ops.attention_paged).
extend     sequences grow by new tokens: pages taken, and the rows that the tokens get (ops.extend_pages).
fork       sequences that continue others: whole pages shared, the partial last one copied (ops.fork_pages).
compact    sequences end and the pages that stay move together (ops.free_pages, ops.compact_pages).
logits     penalties for repeated tokens, biases and grammar masks (ops.adjust_logits), and the greedy
           token of the result (ops.next_tokens).

Head layouts: "7b" is Qwen2.5-7B's (28 query / 4 KV heads of 128), "0.5b" Qwen2.5-0.5B's (14 / 2 heads of 64), "mha" one
without shared KV heads (8 / 8 of 64).

A paged cache of a layer is (1, Hkv, pages * page, D): page p is the rows [p * page, (p + 1) * page) of every head. table
(sequences, entries) names each sequence's pages in order, -1 past the last; lengths its rows; refs how often each page is named.
"""

import math
import random

import torch

own = False

DEV = "cuda"
HEADS = {"7b": (28, 4, 128), "0.5b": (14, 2, 64), "mha": (8, 8, 64)}
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
MOST_PAIRS = 28 * 4096 * (32832 - 2048)  # (query row, cached row) pairs of the largest listed case


def listed():
    return [
        # one sequence's decoded token after an 8k request: latency
        {"name": "attention_decode_8k", "kind": "attention", "heads": "7b", "page": 64, "seqs": 1, "rows": 8302, "new": 1, "shared": 0, "deal": 0},
        # a step of 32 sequences of all lengths up to 8k, some slots not in use
        {"name": "attention_decode_32", "kind": "attention", "heads": "7b", "page": 64, "seqs": 32, "rows": 8302, "new": 1, "shared": 0, "deal": 5},
        # follow-up questions of up to 250 tokens in twelve conversations on the small model
        {"name": "attention_chunks_12", "kind": "attention", "heads": "0.5b", "page": 32, "seqs": 12, "rows": 2000, "new": 250, "shared": 0, "deal": 3},
        # the last 4096 tokens of a 32k prompt, prefilled in chunks
        {"name": "attention_chunk_4k_of_32k", "kind": "attention", "heads": "7b", "page": 128, "seqs": 1, "rows": 32832, "new": 4096, "shared": 0, "deal": 0},
        # a decode step's rows: latency
        {"name": "extend_step_32", "kind": "extend", "page": 64, "seqs": 32, "rows": 8302, "new": 1, "deal": 2},
        # ragged documents join 16 conversations of up to 500 rows
        {"name": "extend_prompts_16", "kind": "extend", "page": 32, "seqs": 16, "rows": 500, "new": 8302, "deal": 4},
        # three drafts of a short answer on the small model
        {"name": "fork_3_short", "kind": "fork", "heads": "0.5b", "layers": 24, "dtype": "bf16", "page": 32, "seqs": 1, "rows": 1103, "forks": 3, "deal": 0},
        # sixteen continuations of an 8k request
        {"name": "fork_16_of_8k", "kind": "fork", "heads": "7b", "layers": 28, "dtype": "bf16", "page": 64, "seqs": 2, "rows": 8302, "forks": 16, "deal": 0},
        # half of a few short conversations end
        {"name": "compact_short", "kind": "compact", "heads": "0.5b", "layers": 24, "dtype": "f32", "page": 32, "seqs": 8, "rows": 500, "ended": 4, "deal": 1},
        # half of twelve long conversations end: gigabytes of pages are moved
        {"name": "compact_8k", "kind": "compact", "heads": "7b", "layers": 28, "dtype": "bf16", "page": 64, "seqs": 12, "rows": 8302, "ended": 6, "deal": 3},
        # the next token of one sequence after an 8k prompt: latency
        {"name": "logits_token_1", "kind": "logits", "rows": 1, "vocab": 152064, "dtype": "bf16", "prompt": 8302, "generated": 256, "bias": False, "grammar": False, "token": True},
        # 64 sequences under a grammar, with a bias, logits kept for sampling
        {"name": "logits_64", "kind": "logits", "rows": 64, "vocab": 152064, "dtype": "bf16", "prompt": 1103, "generated": 500, "bias": True, "grammar": True, "token": False},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "extend", "fork", "compact", "logits", "logits"])
    c = {"kind": kind, "deal": rng.randint(0, 1 << 20)}
    if kind == "logits":
        c.update(rows=_log_int(rng, 1, 64), vocab=rng.choice([152064, _log_int(rng, 300, 152064)]), dtype=rng.choice(["bf16", "bf16", "f32"]),
                 prompt=rng.choice([0, _log_int(rng, 1, 8302)]), generated=rng.choice([0, _log_int(rng, 1, 1000)]),
                 bias=rng.random() < 0.4, grammar=rng.random() < 0.4, token=rng.random() < 0.5)
        return c
    c["page"] = rng.choice([32, 64, 128])
    if kind == "extend":
        c["seqs"] = _log_int(rng, 1, 64)
        c["new"] = rng.choice([1, _log_int(rng, 1, 4000)])
        c["rows"] = _log_int(rng, 1, 8302)
        return c
    c["heads"] = rng.choice(["7b", "7b", "0.5b", "mha"])
    if kind == "attention":
        hq = HEADS[c["heads"]][0]
        c["rows"] = _log_int(rng, 1, 32832)
        c["seqs"] = _log_int(rng, 1, max(1, min(64, 270000 // c["rows"])))
        c["new"] = rng.choice([1, _log_int(rng, 1, max(1, min(c["rows"], 4096, MOST_PAIRS // (hq * c["seqs"] * c["rows"]))))])
        c["shared"] = rng.choice([0, 0, rng.randint(0, c["rows"] // c["page"]) * c["page"]])
        return c
    c["dtype"] = rng.choice(["bf16", "bf16", "f32"])
    c["layers"] = _log_int(rng, 1, 14 if c["dtype"] == "f32" else 28)
    if kind == "fork":
        c["seqs"] = _log_int(rng, 1, 4)
        c["rows"] = _log_int(rng, 1, 8302)
        c["forks"] = _log_int(rng, 1, 16)
    else:
        c["seqs"] = _log_int(rng, 2, 12)
        c["rows"] = _log_int(rng, 1, 8302)
        c["ended"] = rng.randint(1, c["seqs"])
    return c


def _deal(case):
    """(rows of each sequence, new tokens among them): every length up to the most, slots without a sequence among them."""
    rng = random.Random(case["deal"])
    got = []
    for i in range(case["seqs"]):
        if case["seqs"] > 1 and i and rng.random() < 0.1:
            got.append((0, 0))
            continue
        rows = case["rows"] if i == 0 else _log_int(rng, max(1, case["rows"] // 16), case["rows"])
        if "new" not in case:
            got.append((rows, 0))
        elif case["kind"] == "extend":  # rows so far, rows to come
            got.append((rows, case["new"] if i == 0 or case["new"] == 1 else rng.randint(1, case["new"])))
        else:
            rows = max(rows, case["shared"] + 1)
            got.append((rows, min(rows, case["new"] if i == 0 or case["new"] == 1 else rng.randint(1, case["new"]))))
    return got


# ---- inputs ---------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 29)


def _randn(gen, shape, dtype=torch.bfloat16):
    return torch.randn(shape, generator=gen, device=DEV, dtype=dtype)


def _pages(rows, page):
    return -(-rows // page)


def _book(lengths, page, entries, pages, seed, shared=0):
    """table, lengths and refs in one int32 buffer, each sequence's pages spread over the pool as after long use."""
    order = list(range(pages))
    random.Random(int(seed) * 31 + 7).shuffle(order)
    first = [order.pop() for _ in range(shared // page)]
    table, refs = [[-1] * entries for _ in lengths], [0] * pages
    for row, n in zip(table, lengths):
        for j in range(_pages(n, page)):
            row[j] = first[j] if j < len(first) else order.pop()
            refs[row[j]] += 1
    flat = [p for row in table for p in row] + list(lengths) + refs
    return torch.tensor(flat, dtype=torch.int32).to(DEV)


def _views(book, seqs, entries):
    """table, lengths and refs of _book's buffer."""
    return book[:seqs * entries].view(seqs, entries), book[seqs * entries:seqs * entries + seqs], book[seqs * entries + seqs:]


def _pool(gen, layers, h, rows, d, dtype):
    """A pool of rows, and keys' few large channels; made a layer at a time."""
    out = torch.empty((layers, 1, h, rows, d), dtype=dtype, device=DEV)
    for layer in out:
        layer.copy_(_randn(gen, (1, h, rows, d), dtype) * torch.where(torch.rand((1, h, 1, d), generator=gen, device=DEV) < 0.06, 4.0, 0.8).to(dtype))
    return out


def prepare(case, seed):
    gen = _gen(seed)
    kind = case["kind"]
    if kind == "logits":
        b, n = case["rows"], case["vocab"]
        s = {"case": case, "logits": (3 * _randn(gen, (b, n), torch.float32)).to(DTYPES[case["dtype"]])}
        # tokens as text has them, few of them often; shorter rows are padded with -1
        for what, most in (("prompt", case["prompt"]), ("generated", case["generated"])):
            t = (n * torch.rand((b, most), generator=gen, device=DEV) ** 3).to(torch.int64).clamp_(max=n - 1)
            keep = (most * (0.5 + 0.5 * torch.rand((b, 1), generator=gen, device=DEV))).ceil()
            s[what] = torch.where(torch.arange(most, device=DEV)[None] < keep, t, -1) if most else None
        row = lambda lo, hi: lo + (hi - lo) * torch.rand((b,), generator=gen, device=DEV)  # noqa: E731
        s["repetition"], s["frequency"], s["presence"] = row(1.0, 1.3), row(0.0, 0.5), row(0.0, 1.0)
        s["bias"] = _randn(gen, (n,), torch.float32) if case["bias"] else None
        s["allowed"] = None
        if case["grammar"]:  # a bit a token; a third of them allowed
            bits = torch.rand((b, _pages(n, 32), 32), generator=gen, device=DEV) < 0.33
            s["allowed"] = (bits.to(torch.int64) << torch.arange(32, device=DEV)).sum(-1).to(torch.uint32).view(torch.int32)
        return s
    page, dealt = case["page"], _deal(case)
    if kind == "attention":
        hq, h, d = HEADS[case["heads"]]
        lengths = [rows for rows, _ in dealt]
        entries = _pages(max(lengths), page)
        pages = sum(_pages(n, page) for n in lengths) + 3
        new = [c for _, c in dealt]
        starts = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32).to(DEV)
        book = _book(lengths, page, entries, pages, seed, case["shared"])
        table, length, refs = _views(book, len(new), entries)
        return {"case": case, "k": _pool(gen, 1, h, pages * page, d, torch.bfloat16), "v": _pool(gen, 1, h, pages * page, d, torch.bfloat16),
                "table": table, "lengths": length, "refs": refs, "starts": starts, "most": max(new),
                # views of token-major rows, as the rotary projection leaves them
                "q": (0.7 * _randn(gen, (1, sum(new), hq, d), torch.float32)).to(torch.bfloat16).transpose(1, 2)}
    if kind == "extend":
        lengths, new = [rows for rows, _ in dealt], [c for _, c in dealt]
        entries = max(_pages(a + b, page) for a, b in dealt) + 2
        pages = sum(_pages(a + b, page) for a, b in dealt) + 5
        saved = _book(lengths, page, entries, pages, seed)
        return {"case": case, "saved": saved, "book": saved.clone(), "entries": entries, "slots": len(new), "tokens": sum(new),
                "counts": torch.tensor(new, dtype=torch.int32).to(DEV), "k": _pool(gen, 1, 1, pages * page, 64, torch.bfloat16)}
    _, h, d = HEADS[case["heads"]]
    lengths, dtype = [rows for rows, _ in dealt], DTYPES[case["dtype"]]
    used = sum(_pages(n, page) for n in lengths)
    s = {"case": case}
    if kind == "fork":
        targets = list(range(len(lengths), len(lengths) + case["forks"]))
        sources = [random.Random(case["deal"] + i).randrange(len(lengths)) for i in range(case["forks"])]
        s["sources"], s["targets"] = (torch.tensor(t, dtype=torch.int32).to(DEV) for t in (sources, targets))
        lengths = lengths + [0] * case["forks"]
        used += case["forks"]
    else:
        ended = random.Random(case["deal"] + 1).sample(range(len(lengths)), case["ended"])
        s["ended"] = torch.tensor(ended, dtype=torch.int32).to(DEV)
    pages, entries = used + 3, _pages(max(lengths), page) + 1
    saved = _book(lengths, page, entries, pages, seed)
    s.update(saved=saved, book=saved.clone(), entries=entries, slots=len(lengths),
             k=_pool(gen, case["layers"], h, pages * page, d, dtype), v=_pool(gen, case["layers"], h, pages * page, d, dtype))
    return s


# ---- the plain forms ------------------------------------------------------------------------


def _attend(state, case):
    """Each sequence's rows gathered, and each of its new tokens' softmax over those up to its own."""
    q, starts = state["q"], state["starts"].tolist()
    hq, h, d = HEADS[case["heads"]]
    out = torch.empty((1, q.shape[2], hq, d), dtype=torch.bfloat16, device=DEV)
    for i, (rows, new) in enumerate(_deal(case)):
        if not new:
            continue
        at = torch.arange(rows, device=DEV)
        at = state["table"][i].long()[at // case["page"]] * case["page"] + at % case["page"]
        hidden = torch.arange(rows, device=DEV)[None, :] > torch.arange(rows - new, rows, device=DEV)[:, None]
        for kv in range(h):
            K, V = (state[t][0, 0, kv, at].float() for t in ("k", "v"))
            heads = slice(kv * (hq // h), (kv + 1) * (hq // h))
            s = torch.matmul(q[0, heads, starts[i]:starts[i + 1]].float(), K.t().contiguous()) / math.sqrt(d)
            s = s.masked_fill_(hidden, -math.inf)
            s = torch.exp(s - s.amax(-1, keepdim=True))
            o = torch.matmul(s, V) / s.sum(-1, keepdim=True)
            out[0, starts[i]:starts[i + 1], heads] = o.transpose(0, 1).to(torch.bfloat16)
    return out


def _free_first(refs):
    """Every page, the free ones first, ascending."""
    return torch.sort((refs != 0).to(torch.int32), stable=True).indices


def _extend(table, lengths, refs, counts, n, page):
    starts = torch.nn.functional.pad(torch.cumsum(counts, 0), (1, 0)).to(torch.int32)
    have, want = (lengths + page - 1) // page, (lengths + counts + page - 1) // page
    need = want - have
    before = torch.cumsum(need, 0) - need
    order = _free_first(refs)
    at = torch.arange(table.shape[1], device=DEV)[None, :]
    rank = (before - have)[:, None] + at
    taken = order[rank.clamp(0, refs.numel() - 1)].to(torch.int32)
    table.copy_(torch.where((at >= have[:, None]) & (at < want[:, None]), taken, table))
    free = refs == 0
    refs.copy_(torch.where(free & (torch.cumsum(free, 0) <= need.sum()), 1, refs))
    token = torch.arange(n, device=DEV)
    s = torch.searchsorted(starts[1:].contiguous(), token.to(torch.int32), right=True)
    positions = lengths.long()[s] + token - starts.long()[s]
    rows = table[s, positions // page].long() * page + positions % page
    lengths += counts
    return positions, rows, starts


def _paged(pool, page):
    return pool.view(pool.shape[0], 1, pool.shape[2], -1, page, pool.shape[4])


def _fork(table, lengths, refs, k, v, sources, targets, page):
    sources, targets = sources.long(), targets.long()
    n = lengths[sources]
    partial = n % page > 0
    taken = _free_first(refs)[(torch.cumsum(partial, 0) - 1).clamp(min=0)]
    last = (n // page).long().clamp(max=table.shape[1] - 1)
    old = table[sources, last].long()
    rows = table[sources]
    whole = torch.arange(table.shape[1], device=DEV)[None, :] < (n // page)[:, None]
    ones = torch.where(whole, 1, 0).to(torch.int32)
    refs.index_add_(0, rows.clamp(min=0).reshape(-1).long(), ones.reshape(-1))
    rows = torch.where(whole, rows, -1)
    rows[torch.arange(len(targets), device=DEV), last] = torch.where(partial, taken.to(torch.int32), rows[torch.arange(len(targets), device=DEV), last])
    table[targets] = rows
    lengths[targets] = n
    src, dst = old[partial], taken[partial]
    refs[dst] = 1
    for pool in (k, v):
        pages = _paged(pool, page)
        pages[:, :, :, dst] = pages[:, :, :, src]


def _free(table, lengths, refs, sequences):
    sequences = sequences.long()
    rows = table[sequences]
    refs.index_add_(0, rows.clamp(min=0).reshape(-1).long(), -(rows >= 0).reshape(-1).to(torch.int32))
    table[sequences] = -1
    lengths[sequences] = 0


def _compact(table, refs, k, v, page):
    used = (refs > 0).sum()
    at = torch.arange(refs.numel(), device=DEV)
    src, dst = at[(refs > 0) & (at >= used)], at[(refs == 0) & (at < used)]
    name = torch.arange(refs.numel(), dtype=torch.int32, device=DEV)
    name[src] = dst.to(torch.int32)
    table.copy_(torch.where(table >= 0, name[table.clamp(min=0).long()], table))
    refs[dst] = refs[src]
    refs[src] = 0
    for pool in (k, v):
        pages = _paged(pool, page)
        pages[:, :, :, dst] = pages[:, :, :, src]
    return used.to(torch.int32).view(1)


def _adjust(state):
    x = state["logits"].float()
    b, n = x.shape
    count, seen = (torch.zeros((b, n + 1), dtype=torch.int32, device=DEV) for _ in range(2))
    for into, what in ((count, "generated"), (seen, "prompt")):
        t = state[what]
        if t is not None:
            t = torch.where((t >= 0) & (t < n), t, n)
            into.scatter_add_(1, t, torch.ones_like(t, dtype=torch.int32))
    count, seen = count[:, :n], seen[:, :n]
    r = state["repetition"][:, None]
    x = torch.where((count > 0) | (seen > 0), torch.where(x > 0, x / r, x * r), x)
    x = x - state["frequency"][:, None] * count
    x = x - torch.where(count > 0, state["presence"][:, None], 0.0)
    if state["bias"] is not None:
        x = x + state["bias"]
    if state["allowed"] is not None:
        at = torch.arange(n, device=DEV)
        x = torch.where((state["allowed"][:, at // 32] >> (at % 32)) & 1 == 1, x, -math.inf)
    return x


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        from chunkkv_amd import ops

        if kind == "logits":
            call = ops.next_tokens if case["token"] else ops.adjust_logits
            got = call(state["logits"], prompt=state["prompt"], generated=state["generated"], repetition=state["repetition"],
                       frequency=state["frequency"], presence=state["presence"], bias=state["bias"], allowed=state["allowed"])
            return {"token" if case["token"] else "logits": got}
        if kind == "attention":
            cache = ops.PagedCache(state["k"], state["v"], state["table"], state["lengths"], state["refs"], case["page"])
            return {"out": ops.attention_paged(state["q"], cache, 0, state["starts"], most=state["most"])}
        state["book"].copy_(state["saved"])
        table, lengths, refs = _views(state["book"], state["slots"], state["entries"])
        book = {"table": table, "lengths": lengths, "refs": refs}
        cache = ops.PagedCache(state["k"], state.get("v", state["k"]), table, lengths, refs, case["page"])
        if kind == "extend":
            got = ops.extend_pages(cache, state["counts"], state["tokens"])
            return dict(book, positions=got.positions, rows=got.rows, starts=got.starts)
        if kind == "fork":
            ops.fork_pages(cache, state["sources"], state["targets"])
            return dict(book, k=state["k"], v=state["v"])
        ops.free_pages(cache, state["ended"])
        return dict(book, used=ops.compact_pages(cache), k=state["k"], v=state["v"])
    if kind == "logits":
        x = _adjust(state)
        return {"token": x.argmax(1)} if case["token"] else {"logits": x}
    if kind == "attention":
        return {"out": _attend(state, case)}
    state["book"].copy_(state["saved"])
    table, lengths, refs = _views(state["book"], state["slots"], state["entries"])
    book = {"table": table, "lengths": lengths, "refs": refs}
    if kind == "extend":
        positions, rows, starts = _extend(table, lengths, refs, state["counts"], state["tokens"], case["page"])
        return dict(book, positions=positions, rows=rows, starts=starts)
    if kind == "fork":
        _fork(table, lengths, refs, state["k"], state["v"], state["sources"], state["targets"], case["page"])
        return dict(book, k=state["k"], v=state["v"])
    _free(table, lengths, refs, state["ended"])
    return dict(book, used=_compact(table, refs, state["k"], state["v"], case["page"]), k=state["k"], v=state["v"])


def work(case):
    kind = case["kind"]
    if kind == "logits":
        b, n = case["rows"], case["vocab"]
        history = 8 * (case["prompt"] + case["generated"])
        return {"bytes": b * (n * DTYPES[case["dtype"]].itemsize + history + (n // 8 if case["grammar"] else 0) + (8 if case["token"] else 4 * n))
                + (4 * n if case["bias"] else 0), "flops": 6 * b * n}
    page, dealt = case["page"], _deal(case)
    if kind == "extend":
        taken = sum(_pages(a + b, page) - _pages(a, page) for a, b in dealt)
        pages = sum(_pages(a + b, page) for a, b in dealt)
        return {"bytes": 4 * pages + 8 * taken + 16 * len(dealt) + 16 * sum(b for _, b in dealt), "flops": pages}
    hq, h, d = HEADS[case["heads"]]
    if kind == "attention":
        pairs = hq * sum(c * n - c * (c - 1) // 2 for n, c in dealt)
        rows = sum(n for n, _ in dealt) - case["shared"] * (sum(n > 0 for n, _ in dealt) - 1)
        return {"bytes": 4 * hq * d * sum(c for _, c in dealt) + 4 * h * rows * d, "flops": 4 * d * pairs}
    one = 4 * case["layers"] * h * page * d * DTYPES[case["dtype"]].itemsize  # a page's K and V, read and written
    if kind == "fork":
        sources = [random.Random(case["deal"] + i).randrange(len(dealt)) for i in range(case["forks"])]
        copies = sum(dealt[s][0] % page > 0 for s in sources)
        return {"bytes": copies * one + 8 * sum(_pages(dealt[s][0], page) for s in sources) + 64, "flops": 0}
    ended = set(random.Random(case["deal"] + 1).sample(range(len(dealt)), case["ended"]))
    left = sum(_pages(n, page) for i, (n, _) in enumerate(dealt) if i not in ended)
    total = sum(_pages(n, page) for n, _ in dealt) + 3
    # pages lie anywhere: of those that stay, the part behind the first `left` moves
    return {"bytes": int(left * (total - left) / total) * one + 4 * total, "flops": 0}


# ---- from the definition, in 64 bits --------------------------------------------------------


def _exact_logits(s):
    x = s["logits"].double()
    b, n = x.shape
    prompt, generated = ([] if s[w] is None else s[w].tolist() for w in ("prompt", "generated"))
    for i in range(b):
        count = {}
        for t in generated[i] if generated else []:
            if 0 <= t < n:
                count[t] = count.get(t, 0) + 1
        known = sorted(set(count) | {t for t in (prompt[i] if prompt else []) if 0 <= t < n})
        if known:
            at = torch.tensor(known, device=DEV)
            times = torch.tensor([count.get(t, 0) for t in known], dtype=torch.float64, device=DEV)
            r, f, p = (s[w][i].double() for w in ("repetition", "frequency", "presence"))
            v = x[i, at]
            x[i, at] = torch.where(v > 0, v / r, v * r) - f * times - p * (times > 0)
    if s["bias"] is not None:
        x += s["bias"].double()
    if s["allowed"] is not None:
        words = s["allowed"].view(torch.uint8).cpu().numpy()
        import numpy

        bits = numpy.unpackbits(words, axis=1, bitorder="little")[:, :n]
        x[torch.from_numpy(bits == 0).to(DEV)] = -math.inf
    return x


def _lists(s, case):
    """table, lengths and refs of a state as lists."""
    return [t.tolist() for t in _views(s["saved"], s["slots"], s["entries"])]


def _back(table, lengths, refs):
    t = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return {"table": t(table), "lengths": t(lengths), "refs": t(refs)}


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "logits":
        x = _exact_logits(s)
        if not case["token"]:
            return {"logits": x}
        best = x.max(1, keepdim=True).values
        return {"token": torch.where(x == best, torch.arange(x.shape[1], device=DEV), x.shape[1]).min(1).values}
    page = case["page"]
    if kind == "attention":
        hq, h, d = HEADS[case["heads"]]
        out = torch.empty((1, s["q"].shape[2], hq, d), dtype=torch.float64, device=DEV)
        table, t0 = s["table"].tolist(), 0
        for names, (rows, new) in zip(table, _deal(case)):
            if not new:
                continue
            at = torch.tensor([names[j // page] * page + j % page for j in range(rows)], device=DEV)
            for i in range(hq):
                K, V = (s[t][0, 0, i // (hq // h)].double()[at] for t in ("k", "v"))
                for a in range(0, new, 2048):
                    b = min(new, a + 2048)
                    x = torch.mm(s["q"][0, i, t0 + a:t0 + b].double(), K.t().contiguous()) * d ** -0.5
                    seen = torch.arange(rows, device=DEV)[None] <= torch.arange(rows - new + a, rows - new + b, device=DEV)[:, None]
                    out[0, t0 + a:t0 + b, i] = torch.mm(torch.softmax(x.masked_fill(~seen, -math.inf), 1), V)
            t0 += new
        return {"out": out}
    table, lengths, refs = _lists(s, case)

    def take():
        p = refs.index(0)
        refs[p] = 1
        return p

    if kind == "extend":
        positions, rows, starts = [], [], [0]
        for i, c in enumerate(s["counts"].tolist()):
            for p in range(lengths[i], lengths[i] + c):
                if p % page == 0:
                    table[i][p // page] = take()
                positions.append(p)
                rows.append(table[i][p // page] * page + p % page)
            lengths[i] += c
            starts.append(len(rows))
        return dict(_back(table, lengths, refs), positions=torch.tensor(positions), rows=torch.tensor(rows), starts=torch.tensor(starts, dtype=torch.int32))
    moves = []
    if kind == "fork":
        for a, b in zip(s["sources"].tolist(), s["targets"].tolist()):
            whole, part = divmod(lengths[a], page)
            lengths[b] = lengths[a]
            for j in range(whole):
                table[b][j] = table[a][j]
                refs[table[a][j]] += 1
            if part:
                table[b][whole] = take()
                moves.append((table[a][whole], table[b][whole]))
        got = _back(table, lengths, refs)
    else:
        for i in s["ended"].tolist():
            for j, p in enumerate(table[i]):
                if p >= 0:
                    refs[p] -= 1
                    table[i][j] = -1
            lengths[i] = 0
        used = sum(r > 0 for r in refs)
        moves = list(zip([p for p in range(used, len(refs)) if refs[p]], [p for p in range(used) if not refs[p]]))
        to = dict(moves)
        table = [[to.get(p, p) for p in row] for row in table]
        for a, b in moves:
            refs[b], refs[a] = refs[a], 0
        got = dict(_back(table, lengths, refs), used=torch.tensor([used], dtype=torch.int32))
    for a, b in moves:
        for pool in (s["k"], s["v"]):
            pool[:, 0, :, b * page:(b + 1) * page] = pool[:, 0, :, a * page:(a + 1) * page]
    return dict(got, k=s["k"], v=s["v"])
