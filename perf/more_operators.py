"""The operators of decoding over a paged cache, as cases that can be timed.

Four kinds of pass:

  attend   attention of each sequence's newest tokens over its pages: one token
           (a decode step), a few (drafted tokens that are verified) or a chunk
           of a prompt, over bf16 pages or e4m3 pages with a scale a row
  append   new keys and values written into their pages
  advance  a step of the page tables: beams follow their parents, every row gets
           room for its next tokens, shared pages that would be written are copied
  scores   log probabilities of given tokens, the entropy and the best alternatives

Where `own` is false a pass is computed with elementary torch operations,
where it is true with the framework's entry points.
"""
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
E4M3 = torch.float8_e4m3fn
GOLDEN = 0.6180339887498949


def _l2c():
    path = os.path.join(ROOT, "cuda-elastic_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import l2c
    return l2c


# ---------------------------------------------------------------------------
# Cases.

def _attend(sequences, new, context, heads, kv_heads, width, page, cache, window, ragged, name=None):
    c = {"kind": "attend", "sequences": sequences, "new": new, "context": context, "heads": heads,
         "kv_heads": kv_heads, "width": width, "page": page, "cache": cache, "window": window, "ragged": ragged}
    return dict(c, name=name) if name else c


def _append(sequences, new, context, kv_heads, width, page, cache, name=None):
    c = {"kind": "append", "sequences": sequences, "new": new, "context": context, "kv_heads": kv_heads,
         "width": width, "page": page, "cache": cache, "ragged": True}
    return dict(c, name=name) if name else c


def _advance(batch, beams, new, context, page, groups, page_bytes, window, name=None):
    c = {"kind": "advance", "batch": batch, "beams": beams, "new": new, "context": context, "page": page,
         "groups": groups, "page_bytes": page_bytes, "window": window}
    return dict(c, name=name) if name else c


def _scores(rows, vocab, top, name=None):
    c = {"kind": "scores", "rows": rows, "vocab": vocab, "top": top}
    return dict(c, name=name) if name else c


def listed():
    return [
        # One sequence's next token: four query heads share each of eight key heads. Latency.
        _attend(1, 1, 2048, 32, 8, 128, 16, "bf16", 0, False, "attend_1x1_of_2048"),
        # A full decode batch of ragged lengths: the caches streamed once.
        _attend(64, 1, 4096, 32, 8, 128, 16, "bf16", 0, True, "attend_64x1_of_4096"),
        # A few sequences of great length in 8 bits.
        _attend(4, 1, 131072, 32, 8, 128, 64, "e4m3", 0, True, "attend_4x1_of_131072_e4m3"),
        # Five drafted tokens of each sequence, a key head a query head, an odd width, a window.
        _attend(16, 5, 2500, 10, 10, 80, 32, "bf16", 1000, True, "attend_16x5_of_2500"),
        # Chunks of several prompts beside each other.
        _attend(3, 1000, 5000, 32, 8, 128, 16, "bf16", 0, True, "attend_3x1000_of_5000"),
        # The last chunk of a long prompt.
        _attend(1, 4096, 16384, 32, 8, 128, 64, "bf16", 0, False, "attend_1x4096_of_16384"),
        # The keys and values of a decode batch.
        _append(64, 1, 4096, 8, 128, 16, "bf16", "append_64x1"),
        # Those of prompts' chunks, into 8-bit pages.
        _append(4, 2048, 4096, 8, 128, 32, "e4m3", "append_4x2048_e4m3"),
        # The tables of a few requests' beams, keys and values of four layers.
        _advance(8, 4, 1, 500, 16, 8, 8192, 0, "advance_8x4_of_500"),
        # A full batch's.
        _advance(64, 8, 1, 4096, 16, 4, 8192, 0, "advance_64x8_of_4096"),
        # The next token's scores for one row.
        _scores(1, 32000, 5, "scores_1x32000"),
        # A scored prompt of no multiple of four logits.
        _scores(2048, 32003, 20, "scores_2048x32003"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _positions(c):
    """About the positions that all tokens of the case attend to."""
    return c["sequences"] * c["new"] * c["context"]


def draw(rng):
    kind = rng.choice(("attend", "attend", "attend", "append", "advance", "scores"))
    if kind == "attend":
        heads, kv_heads = rng.choice(((32, 8), (32, 32), (8, 1), (10, 10), (12, 4), (64, 8), (40, 8), (6, 2)))
        width, page = rng.choice((64, 80, 128, 128, 256, 96)), rng.choice((16, 32, 64, 128, 48))
        new = rng.choice((1, 1, 1, rng.randint(2, 8), _log_int(rng, 16, 4096), _log_int(rng, 16, 4096)))
        context, sequences = max(new, _log_int(rng, 16, 131072)), _log_int(rng, 1, 128)
        window = 0 if rng.random() < 0.7 else _log_int(rng, 64, 4096)
        c = _attend(sequences, new, context, heads, kv_heads, width, page, rng.choice(("bf16", "bf16", "e4m3")), window,
                    rng.random() < 0.8)
        while (_positions(c) * heads > 4096 * 16384 * 32 or _positions(c) * heads * width > 4096 * 14000 * 32 * 128
               or c["sequences"] * c["context"] * kv_heads * width > 4 * 131072 * 8 * 128):
            if c["sequences"] > 1:
                c["sequences"] //= 2
            else:
                c["context"] = max(16, c["context"] // 2)
                c["new"] = min(c["new"], c["context"])
        return c
    if kind == "append":
        sequences, new = _log_int(rng, 1, 256), rng.choice((1, _log_int(rng, 1, 4096)))
        while sequences * new > 16384:
            sequences = max(1, sequences // 2)
        return _append(sequences, new, new + _log_int(rng, 1, 4096), rng.choice((1, 2, 5, 8, 16)),
                       rng.choice((64, 80, 128, 256)), rng.choice((16, 32, 48, 128)), rng.choice(("bf16", "e4m3")))
    if kind == "advance":
        batch, beams = _log_int(rng, 1, 128), rng.randint(1, 16)
        while batch * beams > 512:
            batch //= 2
        return _advance(batch, beams, rng.choice((1, 1, _log_int(rng, 1, 100))), _log_int(rng, 20, 4096),
                        rng.choice((16, 32, 48, 128)), rng.choice((2, 4, 8)), rng.choice((1024, 4096, 8192)),
                        rng.choice((0, 0, 700)))
    vocab = _log_int(rng, 288, 131072)
    if rng.random() < 0.4:
        vocab = max(256, round(vocab / 256) * 256)
    rows = _log_int(rng, 1, 2048)
    while rows * vocab > 2048 * 32003:
        rows //= 2
    return _scores(rows, vocab, rng.randint(0, 32))


# ---------------------------------------------------------------------------
# Inputs, from the seed alone; how long the sequences are, from the case.

def _lengths(c):
    """(cached positions, the new ones among them) of every sequence."""
    if not c["ragged"]:
        return [c["context"]] * c["sequences"], [c["new"]] * c["sequences"]
    short = [(i * GOLDEN) % 1.0 for i in range(c["sequences"])]
    lengths = [max(1, round(c["context"] * (1.0 - 0.6 * f))) for f in short]
    return lengths, [min(n, max(1, round(c["new"] * (1.0 - 0.4 * f)))) for n, f in zip(lengths, reversed(short))]


def _normal(gen, *shape, dtype=torch.float32):
    return torch.empty(*shape, device="cuda", dtype=dtype).normal_(generator=gen)


def _int(values):
    return torch.tensor(values, device="cuda", dtype=torch.int32)


def _paged(c, gen):
    """Lengths, the new tokens' first rows, and tables of pages in no order."""
    lengths, new = _lengths(c)
    need = [-(-n // c["page"]) for n in lengths]
    most, pages = max(need) + 2, sum(need) + 3
    order = torch.randperm(pages, generator=gen, device="cuda", dtype=torch.int32)
    tables, at = torch.full((c["sequences"], most), -1, device="cuda", dtype=torch.int32), 0
    for s, n in enumerate(need):
        tables[s, :n] = order[at:at + n]
        at += n
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    c.update(lengths=_int(lengths), starts=_int(starts), rows=starts[-1], max_new=max(new), tables=tables, most=most,
             pages=pages)


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    c = dict(case)
    if c["kind"] in ("attend", "append"):
        _paged(c, gen)
        kv, width = c["kv_heads"], c["width"]
        shape = (c["pages"], kv, c["page"], width)
        for which in ("keys", "values"):
            if c["cache"] == "bf16":
                c[which] = _normal(gen, *shape, dtype=torch.bfloat16)
            else:
                c[which] = (110.0 * _normal(gen, *shape)).clamp_(-448, 448).to(E4M3).view(torch.uint8)
            c[which + "_scale"] = None if c["cache"] == "bf16" else torch.empty(
                shape[:3], device="cuda").uniform_(0.005, 0.015, generator=gen)
        # Queries, keys and values as one product leaves them, side by side.
        heads = c.get("heads", kv)
        c["stride"] = (heads + 2 * kv) * width
        fused = _normal(gen, c["rows"], c["stride"], dtype=torch.bfloat16)
        c.update(q=fused[:, :heads * width], k=fused[:, heads * width:(heads + kv) * width],
                 v=fused[:, (heads + kv) * width:])
        if c["kind"] == "attend":
            c["out"] = torch.empty(c["rows"], heads * width, device="cuda", dtype=torch.bfloat16)
            # At most this by the formula that the entry point documents.
            c["workspace"] = torch.empty((width + 2) << 19, device="cuda", dtype=torch.uint8)
    elif c["kind"] == "advance":
        batch, beams, page, rows = c["batch"], c["beams"], c["page"], c["batch"] * c["beams"]
        # The beams of a request share their first pages, and have the last two of their own.
        lengths = [max(1, round(c["context"] * (1.0 - 0.6 * ((b * GOLDEN) % 1.0)))) for b in range(batch)]
        need = [-(-n // page) for n in lengths]
        shared = [max(0, n - 2) for n in need]
        most = max(need) + 2 + c["new"] // page
        used = sum(s + beams * (n - s) for s, n in zip(shared, need))
        pages = used + rows * (2 + c["new"] // page) + 8
        order = torch.randperm(pages, generator=gen, device="cuda", dtype=torch.int32)
        tables, at = torch.full((batch, beams, most), -1, device="cuda", dtype=torch.int32), 0
        for b in range(batch):
            tables[b, :, :shared[b]] = order[at:at + shared[b]]
            at += shared[b]
            last = need[b] - shared[b]
            tables[b, :, shared[b]:need[b]] = order[at:at + beams * last].reshape(beams, last)
            at += beams * last
        parents = torch.randint(beams, (rows,), generator=gen, device="cuda", dtype=torch.int32)
        parents[torch.rand(rows, generator=gen, device="cuda") < 0.02] = -1  # beams without a successor
        held = torch.zeros(pages, device="cuda", dtype=torch.int32)
        held[order[-4:].long()] = 1  # pages that something else keeps
        empty = lambda *s: torch.empty(*s, device="cuda", dtype=torch.int32)  # noqa: E731
        c.update(rows=rows, most=most, pages=pages, tables=tables.reshape(rows, most), parents=parents, held=held,
                 lengths=_int(lengths).repeat_interleave(beams),
                 starts=None if c["new"] == 1 else torch.arange(rows + 1, device="cuda", dtype=torch.int32) * c["new"],
                 tables_out=empty(rows, most), lengths_out=empty(rows), uses=empty(pages), copies=empty(rows, 2),
                 shortage=empty(1),
                 pool=torch.randint(256, (c["groups"], pages, c["page_bytes"]), generator=gen, device="cuda",
                                    dtype=torch.uint8))
    else:
        rows, vocab, top = c["rows"], c["vocab"], c["top"]
        c.update(logits=3.0 * _normal(gen, rows, vocab),
                 tokens=torch.randint(vocab, (rows,), generator=gen, device="cuda", dtype=torch.int32),
                 logprobs=torch.empty(rows, device="cuda"), entropies=torch.empty(rows, device="cuda"),
                 top_tokens=torch.empty(rows, top, device="cuda", dtype=torch.int32),
                 top_logprobs=torch.empty(rows, top, device="cuda"))
        # At most this by the formula that the entry point documents.
        c["workspace"] = torch.empty(rows * -(-vocab // 1024) * (8 * top + 32), device="cuda", dtype=torch.uint8)
    return c


# ---------------------------------------------------------------------------
# The plain forms.

def _new_rows(s):
    """(row, sequence, position) of every new token."""
    starts = s["starts"].long()
    row = torch.arange(s["rows"], device=starts.device)
    sequence = torch.searchsorted(starts, row, right=True) - 1
    return row, sequence, s["lengths"].long()[sequence] - (starts[sequence + 1] - row)


def _of_pages(s, which):
    """A cache's positions after each other, [sequence][head][position][width] in 32 bits."""
    x = s[which]
    x = x.float() if x.dtype is torch.bfloat16 else x.view(E4M3).float() * s[which + "_scale"].unsqueeze(-1)
    x = x[s["tables"].clamp(min=0).long()].transpose(1, 2)
    return x.reshape(s["sequences"], s["kv_heads"], s["most"] * s["page"], s["width"])


def _plain_attend(s):
    n, most, kv, width = s["sequences"], s["max_new"], s["kv_heads"], s["width"]
    group = s["heads"] // kv
    row, sequence, position = _new_rows(s)
    index = row - s["starts"].long()[sequence]
    q = torch.zeros(n, most, kv, group, width, device=row.device)
    q[sequence, index] = s["q"].float().reshape(-1, kv, group, width)
    q = q.transpose(1, 2).reshape(n, kv, most * group, width)
    at = torch.full((n, most), -1, device=row.device)
    at[sequence, index] = position
    at = at.repeat_interleave(group, 1).reshape(n, 1, most * group, 1)
    key = torch.arange(s["most"] * s["page"], device=row.device)
    seen = key <= at
    if s["window"]:
        seen &= key > at - s["window"]
    seen &= (s["tables"] >= 0).repeat_interleave(s["page"], 1).reshape(n, 1, 1, -1)
    score = torch.where(seen, q @ _of_pages(s, "keys").transpose(-1, -2) * width ** -0.5, -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = (score - torch.where(top > -math.inf, top, 0.0)).exp()
    total = weight.sum(-1, keepdim=True)
    there = (key < s["lengths"].reshape(-1, 1)).reshape(n, 1, -1, 1)
    out = (weight @ torch.where(there, _of_pages(s, "values"), 0.0)) / torch.where(total > 0, total, 1.0)
    out = out.reshape(n, kv, most, group, width).transpose(1, 2)[sequence, index]
    return out.reshape(s["rows"], -1).bfloat16()


def _plain_append(s):
    row, sequence, position = _new_rows(s)
    page = s["tables"].long()[sequence, position // s["page"]]
    slot = position % s["page"]
    rows = {which: s[which[0]].reshape(s["rows"], s["kv_heads"], s["width"]) for which in ("keys", "values")}
    if s["cache"] == "bf16":
        s["keys"][page, :, slot] = rows["keys"]
        s["values"][page, :, slot] = rows["values"]
        return {"keys": s["keys"], "values": s["values"]}
    largest = {which: x.float().abs().amax(-1, keepdim=True) for which, x in rows.items()}
    scale = {which: torch.where(m > 0, m / 448.0, 1.0) for which, m in largest.items()}
    code = {which: (x.float() / scale[which]).to(E4M3).view(torch.uint8) for which, x in rows.items()}
    s["keys"][page, :, slot] = code["keys"]
    s["values"][page, :, slot] = code["values"]
    s["keys_scale"][page, :, slot] = scale["keys"].squeeze(-1)
    s["values_scale"][page, :, slot] = scale["values"].squeeze(-1)
    return {"keys": s["keys"].view(E4M3), "values": s["values"].view(E4M3), "key_scales": s["keys_scale"],
            "value_scales": s["values_scale"]}


def _counts(pages, tables):
    """How often each page is named."""
    flat = tables.reshape(-1).long()
    return torch.zeros(pages + 1, device=flat.device, dtype=torch.long).index_add_(
        0, torch.where(flat < 0, pages, flat), torch.ones_like(flat))[:pages]


def _plain_advance(s):
    page, rows, pages, most, new = s["page"], s["rows"], s["pages"], s["most"], s["new"]
    row, column = torch.arange(rows, device="cuda"), torch.arange(most, device="cuda")
    parent = s["parents"].long()
    lives = parent >= 0
    parent = row - row % s["beams"] + parent.clamp(min=0)
    length = torch.where(lives, s["lengths"].long()[parent], 0)
    new = torch.where(lives, new, 0)
    have, want = (length + page - 1) // page, (length + new + page - 1) // page
    tables = torch.where(column < have.unsqueeze(-1), s["tables"][parent], -1)
    if s["window"]:
        tables = torch.where((column + 1) * page <= (length - s["window"] + 1).unsqueeze(-1), -1, tables)
    count = _counts(pages, tables)
    # Rows that write into their last page; one that others name or keep is replaced, but for the
    # first row where all that name it write.
    last = torch.where((length % page > 0) & (new > 0), length // page, most - 1)
    named = tables.gather(1, last.unsqueeze(-1)).squeeze(-1).long()
    writes = (length % page > 0) & (new > 0) & (named >= 0)
    to = torch.where(writes, named, pages)
    writers = torch.zeros(pages + 1, device="cuda", dtype=torch.long).index_add_(0, to, torch.ones_like(to))
    first = torch.full((pages + 1,), rows, device="cuda").scatter_reduce_(0, to, row, "amin")
    free = (count == 0) & (s["held"] == 0)
    at = named.clamp(min=0)
    replaced = writes & ~((count[at] == writers[at]) & (first[at] == row) & (s["held"][at] == 0))
    fresh = (column >= have.unsqueeze(-1)) & (column < want.unsqueeze(-1))
    fresh |= replaced.unsqueeze(-1) & (column == last.unsqueeze(-1))
    rank = fresh.reshape(-1).cumsum(0).reshape(rows, most) - 1
    order = torch.full((pages + rows * most + 1,), -1, device="cuda")
    order[torch.where(free, free.cumsum(0) - 1, pages + rows * most)] = torch.arange(pages, device="cuda")
    order[-1] = -1
    tables = torch.where(fresh, order[rank.clamp(min=0)].int(), tables)
    given = tables.gather(1, last.unsqueeze(-1)).squeeze(-1)
    copied = replaced & (given >= 0)
    s["tables_out"].copy_(tables)
    s["lengths_out"].copy_(length + new)
    s["uses"].copy_(_counts(pages, tables))
    s["copies"].copy_(torch.where(copied.unsqueeze(-1), torch.stack((named, given.long()), -1), -1))
    s["shortage"].copy_((fresh.sum() - free.sum()).clamp(min=0) + (want - most).clamp(min=0).sum())
    s["pool"][:, given[copied].long()] = s["pool"][:, named[copied]]
    return _advanced(s)


def _advanced(s):
    return {"tables": s["tables_out"], "lengths": s["lengths_out"], "uses": s["uses"], "copies": s["copies"],
            "shortage": s["shortage"], "pool": s["pool"]}


def _plain_scores(s):
    """Sums in 64 bits: the scores lie next to each other."""
    x = s["logits"].double()
    away = x - x.amax(-1, keepdim=True)
    weight = away.exp()
    total = weight.sum(-1, keepdim=True)
    score = away - total.log()
    entropy = total.log().squeeze(-1) - (weight * away).sum(-1) / total.squeeze(-1)
    tokens = torch.sort(s["logits"], dim=-1, descending=True, stable=True).indices[:, :s["top"]]
    return {"logprobs": score.gather(1, s["tokens"].long().unsqueeze(-1)).squeeze(-1).float(),
            "entropies": entropy.float(), "top_tokens": tokens.int(), "top_logprobs": score.gather(1, tokens).float()}


def run(s):
    kind = s["kind"]
    if not own:
        return {"attend": _plain_attend, "append": _plain_append, "advance": _plain_advance,
                "scores": _plain_scores}[kind](s)
    l2c = _l2c()
    if kind == "attend":
        l2c.cache_attention(s["out"], s["q"], s["keys"], s["values"], s["tables"], s["lengths"], s["heads"],
                            s["kv_heads"], s["width"], s["page"], s["pages"], s["most"], s["sequences"],
                            s["workspace"], rows=s["rows"], starts=s["starts"] if s["new"] > 1 else None,
                            window=s["window"], key_scales=s["keys_scale"], value_scales=s["values_scale"],
                            q_stride=s["stride"])
        return s["out"]
    if kind == "append":
        l2c.cache_append(s["keys"], s["values"], s["k"], s["v"], s["tables"], s["lengths"], s["kv_heads"], s["width"],
                         s["page"], s["pages"], s["most"], s["sequences"], rows=s["rows"],
                         starts=s["starts"] if s["new"] > 1 else None, key_scales=s["keys_scale"],
                         value_scales=s["values_scale"], k_stride=s["stride"], v_stride=s["stride"])
        if s["cache"] == "bf16":
            return {"keys": s["keys"], "values": s["values"]}
        return {"keys": s["keys"].view(E4M3), "values": s["values"].view(E4M3), "key_scales": s["keys_scale"],
                "value_scales": s["values_scale"]}
    if kind == "advance":
        l2c.cache_advance(s["tables_out"], s["lengths_out"], s["uses"], s["copies"], s["shortage"], s["tables"],
                          s["lengths"], s["rows"], s["most"], s["page"], s["pages"], parents=s["parents"],
                          beams=s["beams"], starts=s["starts"], held=s["held"], window=s["window"])
        l2c.cache_copy(s["pool"], s["copies"], s["rows"], s["pages"], s["page_bytes"], groups=s["groups"])
        return _advanced(s)
    l2c.decoder_logprobs(s["logprobs"], s["entropies"], s["top_tokens"], s["top_logprobs"], s["logits"], s["tokens"],
                         s["vocab"], s["top"], s["rows"], s["workspace"])
    return {"logprobs": s["logprobs"], "entropies": s["entropies"], "top_tokens": s["top_tokens"],
            "top_logprobs": s["top_logprobs"]}


# ---------------------------------------------------------------------------
# What a pass cannot do without.

def work(case):
    c = case
    if c["kind"] == "scores":
        n = c["rows"] * c["vocab"]
        return {"bytes": 4 * n + c["rows"] * (12 + 8 * c["top"]), "flops": 5 * n}
    if c["kind"] == "advance":
        rows, entries, partly = c["batch"] * c["beams"], 0, 0
        for b in range(c["batch"]):
            n = max(1, round(c["context"] * (1.0 - 0.6 * ((b * GOLDEN) % 1.0))))
            entries += c["beams"] * -(-n // c["page"])
            partly += c["beams"] * (n % c["page"] > 0)
        # Beams whose parent has another child, but for the first, by the parents that prepare() draws.
        copied = partly * (1.0 - 1.0 / c["beams"]) ** c["beams"]
        return {"bytes": 8 * entries + 28 * rows + int(2 * copied) * c["groups"] * c["page_bytes"], "flops": 0}
    lengths, new = _lengths(c)
    element = 2 if c["cache"] == "bf16" else 1
    row = c["kv_heads"] * (2 * c["width"] * element + (0 if element == 2 else 8))  # a position's keys and values
    if c["kind"] == "append":
        return {"bytes": sum(new) * (4 * c["kv_heads"] * c["width"] + row), "flops": 0}
    read, pairs = 0, 0
    for length, n in zip(lengths, new):
        span = min(length, c["window"] or length)
        read += min(length, span + n - 1)
        # Position p sees min(p + 1, window) positions.
        first = length - n
        short = max(0, min(length, span) - first)  # tokens that see all before them
        pairs += short * (first + 1 + first + short) // 2 + (n - short) * span
    return {"bytes": read * row + 4 * sum(new) * c["heads"] * c["width"], "flops": 4 * pairs * c["heads"] * c["width"]}


# ---------------------------------------------------------------------------
# The operators in 64 bits, from their definitions.

def exact(case, seed):
    if case["kind"] == "advance" or (case["kind"] == "append" and case["cache"] == "bf16"):
        return None  # whole numbers, copies
    s = prepare(case, seed)

    def attend():
        group, page = s["heads"] // s["kv_heads"], s["page"]
        out = torch.empty(s["rows"], s["heads"], s["width"], device="cuda", dtype=torch.float64)
        starts = s["starts"].tolist()
        for b, length in enumerate(s["lengths"].tolist()):
            used = s["tables"][b, :-(-length // page)].long()
            n = starts[b + 1] - starts[b]
            p = torch.arange(length - n, length, device="cuda").unsqueeze(1)
            j = torch.arange(length, device="cuda").unsqueeze(0)
            hidden = (j > p) | ((j <= p - s["window"]) if s["window"] else False)
            for h in range(s["kv_heads"]):
                def cached(which):
                    x = s[which][used, h]
                    if s["cache"] == "e4m3":
                        x = x.view(E4M3).double() * s[which + "_scale"][used, h].double()[..., None]
                    return x.double().reshape(-1, s["width"])[:length]

                keys, values = cached("keys"), cached("values")
                for g in range(h * group, (h + 1) * group):
                    q = s["q"][starts[b]:starts[b + 1], g * s["width"]:(g + 1) * s["width"]].double()
                    logit = torch.mm(q, keys.t()) / math.sqrt(s["width"])
                    logit.masked_fill_(hidden, -math.inf)
                    out[starts[b]:starts[b + 1], g] = torch.mm(torch.softmax(logit, 1), values)
        return out.reshape(s["rows"], -1)

    def append():
        got = {}
        for which, scales in (("keys", "key_scales"), ("values", "value_scales")):
            x = s[which[0]].double().reshape(s["rows"], s["kv_heads"], s["width"])
            scale = x.abs().amax(-1) / 448.0
            scale = torch.where(scale > 0, scale, torch.ones_like(scale))
            y = x / scale[..., None]
            step = torch.pow(2.0, torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
            y = torch.round(y / step) * step  # halves go to the even one
            cache, scale_of = s[which].view(E4M3).double(), s[which + "_scale"].double()
            r = 0
            for b, (length, n) in enumerate(zip(s["lengths"].tolist(), s["starts"].diff().tolist())):
                p = torch.arange(length - n, length, device="cuda")
                at = s["tables"][b, p // s["page"]].long()
                cache[at, :, p % s["page"]] = y[r:r + n]
                scale_of[at, :, p % s["page"]] = scale[r:r + n]
                r += n
            got[which], got[scales] = cache, scale_of
        return got

    def scores():
        log_p = torch.log_softmax(s["logits"].double(), 1)
        return {"logprobs": log_p[torch.arange(s["rows"], device="cuda"), s["tokens"].long()],
                "entropies": torch.special.entr(log_p.exp()).sum(1), "top_tokens": None,
                "top_logprobs": torch.topk(log_p, s["top"]).values}

    return {"attend": attend, "append": append, "scores": scores}[case["kind"]]()
