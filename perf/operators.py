"""Calls of the paged cache and its attention over the sizes that they serve: storing new tokens (as they are, in e4m3
or in int8), reading positions back, and attention of new tokens over the pages - single tokens and portions of
prompts, with grouped heads, windows and first tokens that stay visible.

Layouts.  Keys: pages [pages, kv_heads, page, hd]; values: [pages, kv_heads, hd, page]; in 8 bits each (page, head,
position) has an exponent e (int8) and its codes c stand for c 2^e.  A sequence's positions p are in page
table[sequence, p // page].  Rows of all sequences' new tokens follow one another.
"""
import math
import random

import numpy as np
import torch

own = False

# (heads, kv_heads, head size): the OPT sizes 125m, 350m, 1.3b, 6.7b, 13b, 30b and 66b, one of 80, and grouped ones
SHAPES = [(12, 12, 64), (16, 16, 64), (32, 32, 64), (32, 32, 128), (40, 40, 128), (56, 56, 128), (72, 72, 128),
          (32, 32, 80), (32, 8, 128), (16, 4, 256), (16, 2, 192), (8, 1, 64), (20, 4, 96)]
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _case(name, kind, dtype, form, shape, page, seqs, new, behind, window=0, sinks=0):
    return {"name": name, "kind": kind, "dtype": dtype, "format": form, "heads": shape[0], "kv_heads": shape[1],
            "hd": shape[2], "page": page, "seqs": seqs, "new": new, "behind": behind, "window": window, "sinks": sinks}


def listed():
    return [
        # a decode step of the smallest OPT: one token of 16 sequences goes to the cache (launch latency)
        _case("store 125m step e4m3", "store", "fp16", "e4m3", (12, 12, 64), 16, 16, 1, 601),
        # prompts of odd lengths admitted together
        _case("store 6.7b prompts int8", "store", "fp16", "int8", (32, 32, 128), 64, 8, 777, 0),
        # long documents with grouped heads, behind what earlier portions stored
        _case("store grouped e4m3", "store", "bf16", "e4m3", (32, 8, 128), 64, 32, 2500, 1000),
        # sequences handed to another cache: whole, as they are
        _case("read 6.7b fp16", "read", "fp16", "same", (32, 32, 128), 64, 16, 2047, 0),
        # a shared prefix read back from 8 bits
        _case("read grouped int8", "read", "bf16", "int8", (16, 2, 192), 32, 5, 1001, 0),
        # one short conversation (launch latency)
        _case("decode 125m", "attend", "fp16", "same", (12, 12, 64), 16, 1, 1, 57),
        # a decode step's layer: the new token is stored, then attended with its history
        _case("step 6.7b", "step", "fp16", "same", (32, 32, 128), 64, 32, 1, 1281),
        # the largest OPT of one card with its cache in 8 bits
        _case("decode 66b e4m3", "attend", "fp16", "e4m3", (72, 72, 128), 64, 64, 1, 1200),
        # one very long document, grouped heads, int8
        _case("decode long int8", "attend", "bf16", "int8", (32, 8, 128), 128, 1, 1, 131071),
        # portions of prompts behind what is stored already
        _case("portion 6.7b", "attend", "fp16", "same", (32, 32, 128), 64, 4, 513, 1536),
        # a stream that keeps its first tokens and a window: a portion of it ...
        _case("portion window sinks", "attend", "bf16", "same", (32, 8, 128), 64, 2, 4096, 8192, 1024, 4),
        # ... and single tokens of many such streams
        _case("decode window sinks e4m3", "attend", "bf16", "e4m3", (32, 8, 128), 32, 24, 1, 30000, 4096, 16),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(c):
    w = work(c)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(["store", "read", "attend", "attend", "attend", "step"])
        shape = rng.choice(SHAPES)
        c = {"kind": kind, "dtype": rng.choice(["fp16", "bf16"]),
             "format": "same" if kind == "step" else rng.choice(["same", "e4m3", "int8"]),
             "heads": shape[0], "kv_heads": shape[1], "hd": shape[2], "page": rng.choice([16, 32, 64, 128, 256]),
             "seqs": _log(rng, 1, 64), "new": 0, "behind": 0, "window": 0, "sinks": 0}
        if kind in ("store", "read"):
            c["new"] = rng.choice([1, _log(rng, 1, 4096)])
            c["behind"] = rng.choice([0, _log(rng, 1, 4096)])
        else:
            c["new"] = rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 16, 2048)])
            c["behind"] = _log(rng, 1, 131072 if c["new"] == 1 else 8192)
            if rng.random() < 0.4:
                c["window"], c["sinks"] = _log(rng, 16, 4096), rng.choice([0, 1, 4, rng.randint(2, 100)])
        # what the plain form holds: scores, and the sequences' keys and values
        span = c["new"] + c["behind"]
        held = 4 * c["seqs"] * span * max(c["heads"] * c["new"], 2 * c["kv_heads"] * c["hd"])
        if _cost(c) <= most and held <= 12e9:
            return c


def _lengths(c):
    """(new tokens, tokens before them) of every sequence: between about half of the case's and all of it."""
    new = [c["new"] - (i * 7919) % (c["new"] // 2 + 1) for i in range(c["seqs"])]
    behind = [c["behind"] - (i * 104729) % (c["behind"] // 2 + 1) for i in range(c["seqs"])]
    return new, behind


def work(case):
    c = case
    new, behind = _lengths(c)
    n, kvd = sum(new), c["kv_heads"] * c["hd"]
    stored = 2 * (kvd * 2 if c["format"] == "same" else kvd + c["kv_heads"])  # bytes of a position in the cache
    rows = 2 * kvd * 2                                                        # ... of its key and value in 16 bits
    if c["kind"] == "store":    # keys and values in, the cache out, and the values that it holds
        return {"bytes": n * (rows + stored + rows), "flops": 0}
    if c["kind"] == "read":
        return {"bytes": n * (stored + rows), "flops": 0}
    pairs = keys = 0
    for t, b in zip(new, behind):
        p = np.arange(b, b + t, dtype=np.int64)
        if c["window"]:
            first = np.maximum(0, p - c["window"] + 1)
            pairs += int((p - first + 1 + np.minimum(first, c["sinks"])).sum())
            keys += int(p[-1] - first[0] + 1 + min(first[0], c["sinks"]))
        else:
            pairs += int((p + 1).sum())
            keys += b + t
    size = keys * stored + 2 * n * c["heads"] * c["hd"] * 2
    if c["kind"] == "step":     # the new keys and values come in too (and are written among those that are seen)
        size += n * rows
    return {"bytes": size, "flops": 4 * c["hd"] * c["heads"] * pairs}


def prepare(case, seed):
    c, dev = case, "cuda"
    g = torch.Generator(dev).manual_seed(seed)
    new, behind = _lengths(c)
    n, heads, kvh, hd, page = sum(new), c["heads"], c["kv_heads"], c["hd"], c["page"]
    dtype = DTYPES[c["dtype"]]
    randn = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    # rows of a fused projection: queries, keys, values; a few channels are ten times the others, heads differ too
    rows = randn(n, (heads + 2 * kvh) * hd)
    loud = torch.where(torch.rand(2 * kvh * hd, generator=g, device=dev) < 0.02, 10.0, 1.0)
    rows[:, heads * hd:] *= loud * torch.exp2(randn(2 * kvh, 1)).expand(2 * kvh, hd).reshape(-1)
    rows = rows.to(dtype)
    q, k, v = (rows[:, a * hd:b * hd].unflatten(1, (b - a, hd)) for a, b in
               ((0, heads), (heads, heads + kvh), (heads + kvh, heads + 2 * kvh)))
    # pages in an order of their own; entries behind a sequence's end name none
    blocks = [-(-(t + b) // page) for t, b in zip(new, behind)]
    pages = sum(blocks) + 3
    order = torch.randperm(pages, generator=g, device=dev, dtype=torch.int32)
    table = torch.full((c["seqs"], max(blocks)), -1, dtype=torch.int32, device=dev)
    at = 0
    for i, m in enumerate(blocks):
        table[i, :m] = order[at:at + m]
        at += m
    shapes = (pages, kvh, page, hd), (pages, kvh, hd, page)
    exps = [None, None]
    if c["format"] == "same":
        stored = [randn(*s).to(dtype) for s in shapes]
    else:
        top = 448.0 if c["format"] == "e4m3" else 127.0
        held = torch.float8_e4m3fn if c["format"] == "e4m3" else torch.int8
        stored = [(randn(*s) * (top / 3.5)).clamp(-top, top).round().to(held) for s in shapes]
        centre = -8 if c["format"] == "e4m3" else -5
        exps = [torch.randint(centre, centre + 3, (pages, kvh, page), generator=g, device=dev, dtype=torch.int8)
                for _ in range(2)]
    state = {"case": c, "q": q, "k": k, "v": v, "k_pages": stored[0], "v_pages": stored[1], "k_exp": exps[0],
             "v_exp": exps[1], "table": table, "new": new, "behind": behind, "dtype": dtype,
             "new_t": torch.tensor(new, device=dev), "behind_t": torch.tensor(behind, device=dev)}
    if own:  # what a program keeps: the cache, and the plan of its batch
        from metaseq_amd import PagedCache

        state["cache"] = PagedCache(stored[0], stored[1], exps[0], exps[1])
        state["batch"] = state["cache"].batch(new, behind, table)
    return state


# ---- plain forms -----------------------------------------------------------------------------------------------

def _rows_of(s):
    """Per row of the batch: its sequence, its position, its offset among the sequence's new tokens."""
    n = sum(s["new"])
    seq = torch.repeat_interleave(torch.arange(len(s["new"]), device="cuda"), s["new_t"], output_size=n)
    first = torch.cumsum(s["new_t"], 0) - s["new_t"]
    off = torch.arange(n, device="cuda") - first[seq]
    return seq, s["behind_t"][seq] + off, off


def _place(s, seq, pos):
    page = s["case"]["page"]
    return s["table"][seq, pos // page].long(), pos % page


def _power(e):
    """2^e in fp32, from its bits."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _quantise(x, form):
    """(codes, exponents) of rows [n, heads, hd]."""
    top, bits, most = (448.0, 8, 1.75) if form == "e4m3" else (127.0, 6, 1.984375)
    cap = (1.875 if form == "e4m3" else 1.984375) * 2.0 ** (15 if x.dtype == torch.float16 else 127)
    x = x.float().clamp(-cap, cap)
    m, e = torch.frexp(x.abs().amax(-1))
    e = torch.where(m > 0, e - 1 - bits + (2 * m > most).int(), -126).clamp(min=-126)
    y = x * _power(-e).unsqueeze(-1)
    c = y.to(torch.float8_e4m3fn) if form == "e4m3" else y.round().clamp(-top, top).to(torch.int8)
    return c, e.to(torch.int8)


def _bytes(t):
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


def _append(s):
    seq, pos, _ = _rows_of(s)
    page, at = _place(s, seq, pos)
    form = s["case"]["format"]
    for x, pages, exps, transposed in ((s["k"], s["k_pages"], s["k_exp"], False), (s["v"], s["v_pages"], s["v_exp"], True)):
        if form != "same":
            x, e = _quantise(x, form)
            exps[page, :, at] = e
        to = _bytes(pages)
        if transposed:
            to = to.transpose(2, 3)
        to[page, :, at] = _bytes(x)


def _values(codes, exps):
    x = codes.float()
    return x if exps is None else x * _power(exps).unsqueeze(-1)


def _read(s):
    seq, pos, _ = _rows_of(s)
    page, at = _place(s, seq, pos)
    most = torch.finfo(s["dtype"]).max
    got = []
    for pages, exps, transposed in ((s["k_pages"], s["k_exp"], False), (s["v_pages"], s["v_exp"], True)):
        b = _bytes(pages)
        x = (b.transpose(2, 3) if transposed else b)[page, :, at].contiguous()
        x = _values(x.view(pages.dtype), None if exps is None else exps[page, :, at])
        got.append(x.clamp(-most, most).to(s["dtype"]))
    return got


def _attend(s):
    c = s["case"]
    group, kvh, hd, page = c["heads"] // c["kv_heads"], c["kv_heads"], c["hd"], c["page"]
    seqs, longest = len(s["new"]), max(s["new"])
    seq, _, off = _rows_of(s)
    table = s["table"].long().clamp(min=0)
    span = table.shape[1] * page

    def whole(pages, exps, transposed):  # [sequences, kv_heads, positions, hd]
        x = _bytes(pages)[table].view(pages.dtype)
        x = x.transpose(3, 4) if transposed else x
        x = _values(x, None if exps is None else exps[table])
        return x.transpose(1, 2).reshape(seqs, kvh, span, hd)

    q = torch.zeros(seqs, longest, c["heads"], hd, device="cuda")
    q[seq, off] = s["q"].float()
    q = q.view(seqs, longest, kvh, group, hd).permute(0, 2, 3, 1, 4).reshape(seqs, kvh, group * longest, hd)
    scores = torch.matmul(q, whole(s["k_pages"], s["k_exp"], False).transpose(2, 3)) * (1.0 / math.sqrt(hd))
    at = s["behind_t"].view(-1, 1, 1) + torch.arange(longest, device="cuda").view(1, -1, 1)
    key = torch.arange(span, device="cuda").view(1, 1, -1)
    seen = key <= at
    if c["window"]:
        seen = seen & ((key > at - c["window"]) | (key < c["sinks"]))
    scores = scores.view(seqs, kvh, group, longest, span)
    scores.masked_fill_(~seen.view(seqs, 1, 1, longest, span), -math.inf)
    scores -= scores.amax(-1, keepdim=True)
    scores.exp_()
    total = scores.sum(-1, keepdim=True)
    values = whole(s["v_pages"], s["v_exp"], True)
    # positions behind a sequence's last one may hold anything
    end = (s["behind_t"] + s["new_t"]).view(-1, 1, 1, 1)
    values = torch.where(torch.arange(span, device="cuda").view(1, 1, -1, 1) < end, values, 0.0)
    o = torch.matmul(scores.view(seqs, kvh, group * longest, span), values).view(seqs, kvh, group, longest, hd) / total
    return o.permute(0, 3, 1, 2, 4).reshape(seqs, longest, c["heads"], hd)[seq, off].to(s["dtype"])


def run(state):
    s, kind = state, state["case"]["kind"]
    if own:
        cache, batch = s["cache"], s["batch"]
        if kind in ("store", "step"):
            cache.append(batch, s["k"], s["v"])
        if kind in ("store", "read"):
            return cache.read(batch, s["dtype"])
        o = cache.attend(batch, s["q"], window=s["case"]["window"], sinks=s["case"]["sinks"])
    else:
        if kind in ("store", "step"):
            _append(s)
        if kind in ("store", "read"):
            return _read(s)
        o = _attend(s)
    return (o, s["k_pages"], s["v_pages"]) if kind == "step" else o


# ---- from the definitions, in 64 bits --------------------------------------------------------------------------

def _held_exactly(x, form):
    """What a cache holds of rows x [n, heads, hd] in 64 bits: the nearest code times its power of two."""
    big = 2.0 ** (15 if x.dtype == torch.float16 else 127)
    x = x.double()
    if form == "same":
        return x
    top, largest = (448.0, 1.875 * big) if form == "e4m3" else (127.0, 1.984375 * big)
    x = torch.minimum(torch.maximum(x, torch.full_like(x, -largest)), torch.full_like(x, largest))
    most = x.abs().max(dim=-1, keepdim=True).values
    two = lambda e: ((e.long() + 1023) << 52).view(torch.float64)  # noqa: E731
    e = torch.ceil(torch.log2(most / top))
    e = torch.where(two(e) * top < most, e + 1, e)              # the logarithm is rounded, the comparisons are not
    e = torch.where(two(e - 1) * top >= most, e - 1, e).clamp(min=-126)
    y = x / two(e)
    if form == "int8":
        return torch.round(y) * two(e)
    binade = ((y.abs().clamp(min=2.0 ** -6).view(torch.int64) >> 52) - 1023).double()
    step = two(binade - 3)
    return torch.round(y / step) * step * two(e)


def _positions_exactly(s, i, upto, values):
    """Positions 0 .. upto - 1 of sequence i as they stand in the pages, in 64 bits: [upto, kv_heads, hd]."""
    pages, exps = (s["v_pages"], s["v_exp"]) if values else (s["k_pages"], s["k_exp"])
    page = s["case"]["page"]
    which = [int(p) for p in s["table"][i, : -(-upto // page)].tolist()]
    parts = []
    for p in which:
        x = pages[p].double()
        x = x.mT if values else x
        parts.append(x if exps is None else x * ((exps[p].long() + 1023) << 52).view(torch.float64)[..., None])
    return torch.cat(parts, 1)[:, :upto].transpose(0, 1)


def exact(case, seed):
    s, c = prepare(case, seed), case
    n = sum(s["new"])
    if c["kind"] == "store":
        return [_held_exactly(x, c["format"]) for x in (s["k"], s["v"])]
    if c["kind"] == "read":
        return [torch.cat([_positions_exactly(s, i, b + t, values)[b:] for i, (t, b) in enumerate(zip(s["new"], s["behind"]))])
                for values in (False, True)]
    out, row, group = [], 0, c["heads"] // c["kv_heads"]
    stored = [s["k_pages"].double(), s["v_pages"].double()] if c["kind"] == "step" else None
    for i, (t, b) in enumerate(zip(s["new"], s["behind"])):
        keys, values = (_positions_exactly(s, i, b + t, w) for w in (False, True))
        if c["kind"] == "step":
            for j in range(t):
                p, at = int(s["table"][i, (b + j) // c["page"]]), (b + j) % c["page"]
                keys[b + j], values[b + j] = s["k"][row + j].double(), s["v"][row + j].double()
                stored[0][p, :, at], stored[1][p, :, :, at] = keys[b + j], values[b + j]
        for h in range(c["heads"]):
            z = s["q"][row:row + t, h].double() @ keys[:, h // group].T / math.sqrt(c["hd"])
            for_row = torch.arange(b, b + t, device="cuda")[:, None]
            j = torch.arange(b + t, device="cuda")[None]
            hidden = j > for_row
            if c["window"]:
                hidden = hidden | ((j <= for_row - c["window"]) & (j >= c["sinks"]))
            out.append(torch.softmax(z.masked_fill(hidden, -math.inf), -1) @ values[:, h // group])
        row += t
    # [sequence][head][t, hd] -> [n, heads, hd]
    o = torch.cat([torch.stack(out[i * c["heads"]:(i + 1) * c["heads"]], 1) for i in range(c["seqs"])])
    assert o.shape[0] == n
    return (o, stored[0], stored[1]) if c["kind"] == "step" else o
