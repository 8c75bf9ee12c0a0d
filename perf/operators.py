"""Cases of the paged K/V cache operators: what a serving program calls, with its sizes.

decode   one new token of every sequence attends to its pages
prefill  a ragged batch of new tokens attends to its pages and, causally, to itself
append   the map grows by the new tokens' pages and their K/V rows are written
fork     sequences are forked: full pages shared, the partly filled one copied
compact  finished sequences are freed and the live pages move to the pool's front
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # the first token after a 512-token prompt, one sequence of a 16 / 4 x 256 head model: latency counts
        {"name": "decode_first", "kind": "decode", "batch": 1, "heads": 16, "kv_heads": 4, "dim": 256, "page": 16,
         "dtype": "f16", "q32": True, "order": "heads", "min_len": 513, "max_len": 513, "lens": 1, "window": 0,
         "sinks": 0},
        # one sequence with a long history, fp32 queries as the decode engine has them
        {"name": "decode_long", "kind": "decode", "batch": 1, "heads": 16, "kv_heads": 4, "dim": 256, "page": 16,
         "dtype": "f16", "q32": True, "order": "heads", "min_len": 32768, "max_len": 32768, "lens": 1, "window": 0,
         "sinks": 0},
        # the ragged batch of 64 sequences with histories of 128 to 8192 positions
        {"name": "decode_ragged", "kind": "decode", "batch": 64, "heads": 16, "kv_heads": 4, "dim": 256, "page": 16,
         "dtype": "f16", "q32": False, "order": "heads", "min_len": 128, "max_len": 8192, "lens": 2, "window": 0,
         "sinks": 0},
        # many sequences, some past their window, the first tokens kept; pages laid out by position
        {"name": "decode_window", "kind": "decode", "batch": 100, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "dtype": "bf16", "q32": False, "order": "positions", "min_len": 1, "max_len": 20001, "lens": 3,
         "window": 4096, "sinks": 4},
        # one 64-position chunk of a prompt that is being prefilled: few rows, a long axis
        {"name": "prefill_chunk", "kind": "prefill", "batch": 1, "heads": 16, "kv_heads": 4, "dim": 256, "page": 16,
         "dtype": "f16", "order": "heads", "min_new": 64, "max_new": 64, "min_past": 1984, "max_past": 1984,
         "lens": 4, "window": 0, "sinks": 0},
        # requests that arrive together, each with its own prompt and shared or earlier history
        {"name": "prefill_ragged", "kind": "prefill", "batch": 7, "heads": 32, "kv_heads": 8, "dim": 128, "page": 32,
         "dtype": "bf16", "order": "positions", "min_new": 1, "max_new": 1500, "min_past": 0, "max_past": 2500,
         "lens": 5, "window": 0, "sinks": 0},
        # one long prompt at once
        {"name": "prefill_prompt", "kind": "prefill", "batch": 1, "heads": 16, "kv_heads": 4, "dim": 256, "page": 16,
         "dtype": "f16", "order": "heads", "min_new": 8192, "max_new": 8192, "min_past": 0, "max_past": 0,
         "lens": 6, "window": 0, "sinks": 0},
        # a long prompt under a sliding window with the first tokens kept, seven query heads a group
        {"name": "prefill_window", "kind": "prefill", "batch": 1, "heads": 28, "kv_heads": 4, "dim": 128, "page": 64,
         "dtype": "bf16", "order": "heads", "min_new": 9001, "max_new": 9001, "min_past": 0, "max_past": 0,
         "lens": 7, "window": 1024, "sinks": 16},
        # one token of each of 64 sequences is written: latency counts
        {"name": "append_step", "kind": "append", "batch": 64, "kv_heads": 4, "dim": 256, "page": 16, "dtype": "f16",
         "in32": True, "order": "heads", "min_new": 1, "max_new": 1, "min_past": 128, "max_past": 2048, "lens": 8},
        # a long prompt's rows are written
        {"name": "append_prompt", "kind": "append", "batch": 2, "kv_heads": 8, "dim": 128, "page": 64,
         "dtype": "bf16", "in32": False, "order": "positions", "min_new": 8192, "max_new": 9001, "min_past": 0,
         "max_past": 100, "lens": 9},
        # 64 continuations of eight prompts, over the six attention layers of a hybrid model
        {"name": "fork_samples", "kind": "fork", "parents": 8, "batch": 64, "layers": 6, "kv_heads": 4, "dim": 256,
         "page": 128, "dtype": "f16", "order": "heads", "min_past": 500, "max_past": 4000, "lens": 10},
        # half of 64 sequences have ended: their pages go and the pool closes up
        {"name": "compact_half", "kind": "compact", "batch": 64, "ended": 32, "layers": 6, "kv_heads": 4, "dim": 256,
         "page": 16, "dtype": "f16", "order": "heads", "min_past": 128, "max_past": 4096, "lens": 11},
    ]


HEADS = [(16, 4, 256), (32, 8, 128), (28, 4, 128), (8, 8, 64), (64, 8, 64), (16, 1, 128), (12, 2, 256), (32, 16, 128)]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _one(rng):
    kind = rng.choice(["decode", "decode", "prefill", "prefill", "append", "fork", "compact"])
    heads, kv_heads, dim = rng.choice(HEADS)
    c = {"kind": kind, "kv_heads": kv_heads, "dim": dim, "page": rng.choice([8, 16, 16, 32, 48, 64, 128]),
         "dtype": rng.choice(["f16", "bf16"]), "order": rng.choice(["heads", "positions"]),
         "lens": rng.randrange(1 << 20)}
    if kind in ("decode", "prefill"):
        windowed = rng.random() < 0.5
        c.update(heads=heads, window=_log(rng, 16, 8192) if windowed else 0, sinks=rng.randrange(65) if windowed else 0)
    if kind == "decode":
        top = _log(rng, 1, 32768)
        c.update(batch=_log(rng, 1, 128), q32=c["dtype"] == "f16" and rng.random() < 0.5, max_len=top,
                 min_len=rng.randrange(top + 1))
    elif kind == "prefill":
        new, past = _log(rng, 1, 8192), _log(rng, 1, 8192) - 1
        c.update(batch=_log(rng, 1, 16), max_new=new, min_new=rng.randrange(new + 1), max_past=past,
                 min_past=rng.randrange(past + 1))
    elif kind == "append":
        new, past = _log(rng, 1, 9000), _log(rng, 1, 4096) - 1
        c.update(batch=_log(rng, 1, 128), in32=rng.random() < 0.5, max_new=new, min_new=rng.randrange(new + 1),
                 max_past=past, min_past=rng.randrange(past + 1))
    elif kind == "fork":
        past = _log(rng, 1, 4096)
        c.update(parents=_log(rng, 1, 16), batch=_log(rng, 1, 128), layers=rng.randrange(1, 9), max_past=past,
                 min_past=rng.randrange(1, past + 1))
    else:
        past = _log(rng, 1, 4096)
        c.update(batch=_log(rng, 2, 96), layers=rng.randrange(1, 9), max_past=past, min_past=rng.randrange(past + 1))
        c["ended"] = rng.randrange(1, c["batch"])
    return c


def draw(rng):
    limits = {}
    for c in listed():
        w = work(c)
        for k in w:
            limits[c["kind"], k] = max(limits.get((c["kind"], k), 0), w[k])
    while True:
        c = _one(rng)
        w = work(c)
        seqs, _ = _sizes(c)
        new = c.get("max_new", 1)
        scores = len(seqs) * c.get("heads", 1) * new * max(seqs, default=0)  # what the plain form holds at once
        if (w["bytes"] > 0 and all(w[k] <= limits[c["kind"], k] for k in w) and _positions(c) > 0 and scores <= 2.4e9):
            return c


def _sizes(c):
    """Lengths of the sequences (new tokens included) and their new tokens: the case's, whatever the seed."""
    r = random.Random(c["lens"])
    if c["kind"] == "decode":
        return [r.randint(c["min_len"], c["max_len"]) for _ in range(c["batch"])], [1] * c["batch"]
    if c["kind"] in ("prefill", "append"):
        new = [r.randint(c["min_new"], c["max_new"]) for _ in range(c["batch"])]
        return [r.randint(c["min_past"], c["max_past"]) + n for n in new], new
    n = c["parents"] if c["kind"] == "fork" else c["batch"]
    return [r.randint(c["min_past"], c["max_past"]) for _ in range(n)], [0] * n


def _positions(c):
    seqs, new = _sizes(c)
    return sum(new) if c["kind"] in ("prefill", "append") else sum(seqs)


def _seen(t, window, sinks):
    """How many positions the token at position t sees."""
    if t < 0:
        return 0
    if not window or t < window:
        return t + 1
    return window + min(sinks, t - window + 1)


def work(c):
    seqs, new = _sizes(c)
    row = c["kv_heads"] * c["dim"] * 2  # bytes of one position's K or V
    pages = lambda n: -(-n // c["page"])  # noqa: E731
    if c["kind"] == "decode":
        seen = sum(_seen(n - 1, c["window"], c["sinks"]) for n in seqs)
        wide = 4 if c["q32"] else 2
        q = c["batch"] * c["heads"] * c["dim"] * wide
        return {"bytes": 2 * row * seen + 2 * q + 4 * (sum(map(pages, seqs)) + len(seqs)),
                "flops": 4 * c["heads"] * c["dim"] * seen}
    if c["kind"] == "prefill":
        pairs = read = 0
        for n, m in zip(seqs, new):
            if not m:
                continue
            w, first = c["window"], n - m
            if not w:
                pairs += (n * (n + 1) - first * (first + 1)) // 2
                read += n
            else:
                pairs += sum(_seen(t, w, c["sinks"]) for t in range(first, n))
                low = max(0, first - w + 1)
                read += n - low + min(c["sinks"], low)
        q = sum(new) * c["heads"] * c["dim"] * 2
        return {"bytes": 2 * row * read + 2 * q + 4 * sum(map(pages, seqs)), "flops": 4 * c["heads"] * c["dim"] * pairs}
    if c["kind"] == "append":
        wide = 4 if c["in32"] else 2
        fresh = sum(pages(n) - pages(n - m) for n, m in zip(seqs, new))
        return {"bytes": sum(new) * 2 * (row + row // 2 * wide) + 12 * fresh + 8 * len(seqs), "flops": 0}
    if c["kind"] == "fork":
        full = sum(seqs[i % len(seqs)] // c["page"] for i in range(c["batch"]))
        part = sum(seqs[i % len(seqs)] % c["page"] for i in range(c["batch"]))
        return {"bytes": 4 * row * part * c["layers"] + 16 * full + 12 * c["batch"], "flops": 0}
    # compact: a page at or past the live count moves unless it is free; which ones are free is the seed's, their
    # number follows the share of pages that stay
    total, stay = sum(map(pages, seqs)), sum(map(pages, seqs[c["ended"]:]))
    spare = total // 8 + 1
    moved = stay * (total + spare - stay) // max(1, total + spare)
    return {"bytes": 4 * row * c["page"] * c["layers"] * moved + 8 * total, "flops": 0}


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    seqs, new = _sizes(c)
    page, dt = c["page"], DTYPES[c["dtype"]]
    kind, layers = c["kind"], c.get("layers", 1)
    has = [n - m if kind == "append" else n for n, m in zip(seqs, new)]  # what the map holds before the call
    pages_of = [-(-n // page) for n in has]
    final = [-(-n // page) for n in seqs]
    total = sum(final)
    spare = total // 8 + 1 if kind == "compact" else total // 16 + 1 + (c["batch"] if kind == "fork" else 0)
    pages = total + spare
    slots = len(seqs) + (c["batch"] if kind == "fork" else 0)
    width = max(1, max(final))
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    table = torch.full((slots, width), -1, dtype=torch.int32, device="cuda")
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(pages_of):
        table[s, :n] = order[at:at + n]
        at += n
    refs[order[:at].long()] = 1
    lengths = torch.tensor(has + [0] * (slots - len(has)), dtype=torch.int32, device="cuda")
    shape = (layers, pages, c["kv_heads"], page, c["dim"])
    if c["order"] == "positions":  # [layer][page][position][head][dim] in memory
        shape = (layers, pages, page, c["kv_heads"], c["dim"])
    k, v = torch.empty(shape, dtype=dt, device="cuda"), torch.empty(shape, dtype=dt, device="cuda")
    for t in (k, v):
        for part in t:
            part.normal_(generator=g)
    if c["order"] == "positions":
        k, v = k.transpose(2, 3), v.transpose(2, 3)
    s = {"case": c, "k": k, "v": v, "refs": refs, "table": table, "lengths": lengths}
    starts = [0]
    for m in new:
        starts.append(starts[-1] + m)
    if kind in ("decode", "prefill"):
        s["q"] = torch.randn(starts[-1], c["heads"], c["dim"], device="cuda", generator=g).to(
            torch.float32 if c.get("q32") else dt)
        s["scale"] = c["dim"] ** -0.5
    if kind in ("prefill", "append"):
        s["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
        s["counts"] = torch.tensor(new, dtype=torch.int32, device="cuda")
        s["widest"], s["longest"] = max(1, max(new)), max(1, max(seqs))
    if kind == "decode":
        s["longest"] = max(1, max(_seen(n - 1, c["window"], c["sinks"]) for n in seqs))
    if kind == "append":
        wide = torch.float32 if c["in32"] else dt
        s["new_k"], s["new_v"] = (torch.randn(starts[-1], c["kv_heads"], c["dim"], device="cuda", generator=g).to(wide)
                                  for _ in range(2))
    if kind == "fork":
        s["src"] = (torch.arange(c["batch"], dtype=torch.int32, device="cuda") % c["parents"]).to(torch.int32)
        s["dst"] = torch.arange(c["parents"], c["parents"] + c["batch"], dtype=torch.int32, device="cuda")
    if kind == "compact":
        s["ended"] = torch.arange(c["ended"], dtype=torch.int32, device="cuda")
    if own:  # the handle over those tensors (its workspace), and a second map, so that a pass leaves the first as it was
        at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ray-tracing-attention_b200")
        if at not in sys.path:
            sys.path.insert(0, at)
        from rta_b200.paged import PagedCache, PageMap
        s["cache"] = PagedCache(k, v, PageMap(refs, table, lengths))
        s["map"] = PageMap(torch.empty_like(refs), torch.empty_like(table), torch.empty_like(lengths))
    return s


def run(s):
    c = s["case"]
    return (_own if own else _plain)[c["kind"]](s, c)


# ---------------------------------------------------------------- the framework's calls


def _own_decode(s, c):
    return s["cache"].decode(s["q"], window=c["window"], sinks=c["sinks"], scale=s["scale"])


def _own_prefill(s, c):
    return s["cache"].prefill(s["q"], s["starts"], window=c["window"], sinks=c["sinks"], scale=s["scale"])


def _own_append(s, c):
    m = s["cache"].reserve(s["counts"], out=s["map"])
    s["cache"].append(s["new_k"], s["new_v"], s["starts"], map=m)
    return {"refs": m.refs, "table": m.table, "lengths": m.lengths, "k": s["k"], "v": s["v"]}


def _own_fork(s, c):
    m = s["cache"].fork(s["src"], s["dst"], out=s["map"])
    return {"refs": m.refs, "table": m.table, "lengths": m.lengths, "k": s["k"], "v": s["v"]}


def _own_compact(s, c):
    m = s["cache"].free(s["ended"], out=s["map"])
    s["cache"].compact(map=m)
    return {"refs": m.refs, "table": m.table, "lengths": m.lengths, "k": s["k"], "v": s["v"]}


_own = {"decode": _own_decode, "prefill": _own_prefill, "append": _own_append, "fork": _own_fork,
        "compact": _own_compact}


# ---------------------------------------------------------------- the plain forms


def _rows(pool, table, positions, page):
    """[sequence][position][kv head][dim] in 32 bits of the given positions (any valid number where masked)."""
    which = torch.gather(table, 1, (positions // page).long()).clamp(min=0).long()
    return pool[0].transpose(1, 2)[which, (positions % page).long()].float()


def _attend(q, k, v, visible, scale):
    """q [b][n][heads][dim], k / v [b][l][kv heads][dim], visible [b][n][l] -> [b][n][heads][dim], 32 bits."""
    b, n, heads, dim = q.shape
    kv_heads = k.shape[2]
    group = heads // kv_heads
    q = q.view(b, n, kv_heads, group, dim).permute(0, 2, 3, 1, 4).reshape(b, kv_heads, group * n, dim)
    scores = torch.matmul(q, k.permute(0, 2, 3, 1)).mul_(scale).view(b, kv_heads, group, n, -1)
    scores.masked_fill_(~visible[:, None, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(torch.isinf(top), torch.zeros_like(top), top)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = torch.matmul(scores.view(b, kv_heads, group * n, -1), v.permute(0, 2, 1, 3)).view(b, kv_heads, group, n, dim)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    return out.permute(0, 3, 1, 2, 4).reshape(b, n, heads, dim)


def _plain_decode(s, c):
    page, window, sinks = c["page"], c["window"], c["sinks"]
    n = s["lengths"].long()[:, None]
    u = torch.arange(s["longest"], device="cuda")[None]
    low = (n - window).clamp(min=0) if window else torch.zeros_like(n)
    first = low.clamp(max=sinks)
    p = torch.where(u < first, u, u - first + low)  # the u-th visible position
    visible = p < n
    p = torch.where(visible, p, torch.zeros_like(p))
    k, v = _rows(s["k"], s["table"], p, page), _rows(s["v"], s["table"], p, page)
    return _attend(s["q"].float()[:, None], k, v, visible[:, None], s["scale"])[:, 0].to(s["q"].dtype)


def _plain_prefill(s, c):
    page, window, sinks = c["page"], c["window"], c["sinks"]
    n, m = s["lengths"].long(), s["counts"].long()
    p = torch.arange(s["longest"], device="cuda")[None].expand(len(n), -1)
    k = _rows(s["k"], s["table"], torch.minimum(p, (n - 1).clamp(min=0)[:, None]), page)
    v = _rows(s["v"], s["table"], torch.minimum(p, (n - 1).clamp(min=0)[:, None]), page)
    i = torch.arange(s["widest"], device="cuda")[None]
    mine = i < m[:, None]
    row = torch.where(mine, s["starts"][:-1].long()[:, None] + i, torch.zeros_like(i))
    t = ((n - m)[:, None] + i)[:, :, None]
    p = p[:, None]
    visible = (p <= t) & mine[:, :, None]
    if window:
        visible &= (p > t - window) | (p < sinks)
    return _attend(s["q"].float()[row], k, v, visible, s["scale"])[mine].to(s["q"].dtype)


def _plain_append(s, c):
    page = c["page"]
    n, m, starts = s["lengths"].long(), s["counts"].long(), s["starts"].long()
    have, need = (n + page - 1) // page, (n + m + page - 1) // page
    fresh = need - have
    first = fresh.cumsum(0) - fresh
    free = (s["refs"] == 0).nonzero().flatten()
    j = torch.arange(s["table"].shape[1], device="cuda")[None]
    grown = (j >= have[:, None]) & (j < need[:, None])
    took = free[torch.where(grown, first[:, None] + j - have[:, None], torch.zeros_like(j))]
    table = torch.where(grown, took.to(torch.int32), s["table"])
    refs = s["refs"].clone()
    refs[took[grown]] = 1
    row = torch.arange(s["new_k"].shape[0], device="cuda")
    seq = torch.searchsorted(starts, row, right=True) - 1
    p = n[seq] + row - starts[seq]
    at = table[seq, p // page].long()
    for pool, x in ((s["k"], s["new_k"]), (s["v"], s["new_v"])):
        pool[0].transpose(1, 2)[at, p % page] = x.to(pool.dtype)
    return {"refs": refs, "table": table, "lengths": (n + m).to(torch.int32), "k": s["k"], "v": s["v"]}


def _plain_fork(s, c):
    page, src, dst = c["page"], s["src"].long(), s["dst"].long()
    n = s["lengths"].long()[src]
    full, rest = n // page, n % page
    part = rest > 0
    free = (s["refs"] == 0).nonzero().flatten()
    fresh = free[(part.long().cumsum(0) - 1).clamp(min=0)]
    j = torch.arange(s["table"].shape[1], device="cuda")[None]
    shared = j < full[:, None]
    of = s["table"][src]
    rows = torch.where(shared, of, torch.full_like(of, -1))
    rows = torch.where((j == full[:, None]) & part[:, None], fresh[:, None].to(torch.int32), rows)
    table, refs, lengths = s["table"].clone(), s["refs"].clone(), s["lengths"].clone()
    table[dst] = rows
    refs.index_add_(0, of[shared].long(), torch.ones_like(of[shared]))
    refs[fresh[part]] = 1
    lengths[dst] = n.to(torch.int32)
    a = of[part, full[part]].long()
    b = fresh[part]
    held = (torch.arange(page, device="cuda")[None] < rest[part][:, None])[None, :, None, :, None]
    for pool in (s["k"], s["v"]):
        pool[:, b] = torch.where(held, pool[:, a], pool[:, b])
    return {"refs": refs, "table": table, "lengths": lengths, "k": s["k"], "v": s["v"]}


def _plain_compact(s, c):
    ended = s["ended"].long()
    table, refs, lengths = s["table"].clone(), s["refs"].clone(), s["lengths"].clone()
    gone = table[ended]
    gone = gone[gone >= 0]
    refs.index_add_(0, gone.long(), torch.full_like(gone, -1))
    table[ended] = -1
    lengths[ended] = 0
    live = refs > 0
    at = torch.arange(len(refs), device="cuda")
    count = live.sum()
    holes, movers = at[~live & (at < count)], at[live & (at >= count)]
    to = at.clone()
    to[movers] = holes
    table = torch.where(table >= 0, to[table.clamp(min=0).long()].to(torch.int32), table)
    refs[holes] = refs[movers]
    refs[movers] = 0
    for pool in (s["k"], s["v"]):
        pool[:, holes] = pool[:, movers]
    return {"refs": refs, "table": table, "lengths": lengths, "k": s["k"], "v": s["v"]}


_plain = {"decode": _plain_decode, "prefill": _plain_prefill, "append": _plain_append, "fork": _plain_fork,
          "compact": _plain_compact}


# ---------------------------------------------------------------- 64 bits


def exact(c, seed):
    """Sequence by sequence and head by head in 64 bits.  Forks and compactions only move bits."""
    if c["kind"] in ("fork", "compact"):
        return None
    s = prepare(c, seed)
    seqs, new = _sizes(c)
    page = c["page"]
    if c["kind"] == "append":
        k, v = s["k"].double(), s["v"].double()
        used = s["refs"].tolist()
        free = [i for i, r in enumerate(used) if r == 0]
        table = s["table"].tolist()
        row = 0
        for b, (n, m) in enumerate(zip(seqs, new)):
            for j in range(-(-(n - m) // page), -(-n // page)):
                table[b][j] = free.pop(0)
            p = torch.arange(n - m, n, device="cuda")
            at = torch.tensor(table[b], device="cuda")[p // page]
            k[0, at, :, p % page] = s["new_k"][row:row + m].double()
            v[0, at, :, p % page] = s["new_v"][row:row + m].double()
            row += m
        return {"refs": None, "table": None, "lengths": None, "k": k, "v": v}
    group = c["heads"] // c["kv_heads"]
    out = torch.zeros(sum(new), c["heads"], c["dim"], dtype=torch.float64, device="cuda")
    row = 0
    for b, (n, m) in enumerate(zip(seqs, new)):
        if n and m:
            used = s["table"][b, :-(-n // page)].long()
            t = torch.arange(n - m, n, device="cuda")[:, None]
            p = torch.arange(n, device="cuda")[None]
            hidden = p > t
            if c["window"]:
                hidden |= (p <= t - c["window"]) & (p >= c["sinks"])
            for h in range(c["heads"]):
                if h % group == 0:
                    k = s["k"][0, used, h // group].reshape(-1, c["dim"])[:n].double()
                    v = s["v"][0, used, h // group].reshape(-1, c["dim"])[:n].double()
                score = s["q"][row:row + m, h].double() @ k.T * s["scale"]
                score[hidden] = -math.inf
                out[row:row + m, h] = torch.softmax(score, -1) @ v
        row += m
    return out
