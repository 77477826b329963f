"""The paged-cache operators as they are measured: cases, inputs and plain forms.

Four operators of a serving step, in the order in which a step calls them:

  plan     block tables, slot map and packed offsets from request lengths
  append   new keys and values into the paged cache, through the slot map
  paged    attention of each request's new tokens (a chunk, or one) over its pages
  prompt   causal attention over whole prompts, packed without padding

`run` computes them in elementary torch operations in 32 bits (`own` false) or
by the calls of qwen3-tts_b200/qtb_paged.py (`own` true); `exact` computes them
in 64 bits, request by request.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _ops():
    """The framework's entry points (its package folder is not an importable name)."""
    folder = os.path.join(ROOT, "qwen3-tts_b200")
    if folder not in sys.path:
        sys.path.insert(0, folder)
    import qtb_paged
    return qtb_paged


# ------------------------------------------------------------------- cases --
# Fields. requests, tokens: how many; past: "lo-hi" cached tokens of a request;
# new: "lo-hi" new tokens of a request, long_every: only every n-th request has
# a chunk (the others decode one token); spread "log" or "lin"; lens: the seed
# of the lengths, so that a case's work is its own; heads / kv_heads / dim;
# page: positions in a page; window: keys a token may look back on (0: all).


def listed():
    talker = {"heads": 16, "kv_heads": 8, "dim": 128}
    return [
        # one decode step of 64 requests with contexts of 128 to 2048: every request gets one slot, some a page
        {"name": "plan-decode-64", "op": "plan", "requests": 64, "past": "128-2048", "new": "1-1", "long_every": 1,
         "spread": "lin", "lens": 1, "page": 16},
        # a large mixed step: every 16th of 1024 requests brings a prompt chunk, the others decode
        {"name": "plan-mixed-1024", "op": "plan", "requests": 1024, "past": "0-4096", "new": "128-1024",
         "long_every": 16, "spread": "lin", "lens": 2, "page": 16},
        # one token of 64 requests from an f32 projection into a bf16 cache, one layer
        {"name": "append-decode-64", "op": "append", "tokens": 64, "kv_heads": 8, "dim": 128, "page": 16,
         "source": "f32", "type": "bf16", "padded": 0},
        # the tokens of a large batch of prompts, one layer
        {"name": "append-prompts-32k", "op": "append", "tokens": 32768, "kv_heads": 8, "dim": 128, "page": 64,
         "source": "f16", "type": "f16", "padded": 100},
        # one request, one token: a latency case
        {"name": "paged-decode-1", "op": "paged", "requests": 1, "past": "4095-4095", "new": "1-1", "long_every": 1,
         "spread": "lin", "lens": 3, "page": 16, "type": "bf16", "window": 0, **talker},
        # the decode step of 64 requests with contexts of 256 to 4096
        {"name": "paged-decode-64", "op": "paged", "requests": 64, "past": "255-4095", "new": "1-1", "long_every": 1,
         "spread": "lin", "lens": 4, "page": 16, "type": "bf16", "window": 0, **talker},
        # a large decode batch with long contexts and eight query heads to a key head
        {"name": "paged-decode-128-long", "op": "paged", "requests": 128, "past": "4096-16383", "new": "1-1",
         "long_every": 1, "spread": "lin", "lens": 5, "page": 64, "type": "f16", "window": 0, "heads": 32,
         "kv_heads": 4, "dim": 128},
        # a 64-token chunk of one long prompt over what is cached of it
        {"name": "paged-chunk-64", "op": "paged", "requests": 1, "past": "2048-2048", "new": "64-64", "long_every": 1,
         "spread": "lin", "lens": 6, "page": 16, "type": "bf16", "window": 0, **talker},
        # a mixed step: every fourth request brings a chunk of up to 512 tokens, the others decode
        {"name": "paged-mixed-16", "op": "paged", "requests": 16, "past": "512-7680", "new": "200-512",
         "long_every": 4, "spread": "lin", "lens": 7, "page": 32, "type": "bf16", "window": 0, "heads": 32,
         "kv_heads": 8, "dim": 128},
        # one short prompt: a latency case
        {"name": "prompt-64", "op": "prompt", "requests": 1, "new": "64-64", "spread": "lin", "lens": 8,
         "type": "bf16", "window": 0, **talker},
        # prompts of very different lengths packed together, a key head to each query head
        {"name": "prompt-ragged-24", "op": "prompt", "requests": 24, "new": "1-2048", "spread": "log", "lens": 9,
         "type": "f16", "window": 0, "heads": 16, "kv_heads": 16, "dim": 64},
        # one very long prompt
        {"name": "prompt-16k", "op": "prompt", "requests": 1, "new": "16384-16384", "spread": "lin", "lens": 10,
         "type": "bf16", "window": 0, **talker},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["plan", "append", "paged", "paged", "prompt", "prompt"])
    c = {"op": op, "lens": rng.randrange(1 << 30)}
    if op == "plan":
        lo = _log(rng, 1, 512)
        c |= {"requests": _log(rng, 1, 2048), "past": "0-%d" % _log(rng, 16, 8192), "new": "%d-%d" % (lo, 2 * lo),
              "long_every": rng.choice([1, 8, 32]), "spread": rng.choice(["lin", "log"]),
              "page": rng.choice([16, 32, 64, 128])}
        if c["requests"] * lo * 1.5 / c["long_every"] > 65536:
            c["requests"] = max(1, int(65536 * c["long_every"] / (1.5 * lo)))
        return c
    if op == "append":
        kind = rng.choice(["bf16", "f16"])
        return {"op": op, "tokens": _log(rng, 1, 32768), "kv_heads": rng.choice([1, 2, 4, 8]),
                "dim": rng.choice([64, 128]), "page": rng.choice([16, 32, 64, 128]),
                "source": rng.choice([kind, kind, "f32"]), "type": kind, "padded": rng.choice([0, 3, 17])}
    kv = rng.choice([1, 2, 4, 8])
    c |= {"kv_heads": kv, "heads": kv * rng.choice([1, 2, 4, 5, 7, 8]), "dim": rng.choice([64, 128, 128]),
          "type": rng.choice(["bf16", "f16"]), "spread": rng.choice(["lin", "log"]),
          "window": rng.choice([0, 0, 0, _log(rng, 16, 1024)])}
    while True:
        if op == "paged":
            kind = rng.choice(["decode", "few", "chunk", "mixed"])
            hi = {"decode": 1, "few": _log(rng, 2, 8), "chunk": _log(rng, 16, 512), "mixed": _log(rng, 64, 512)}[kind]
            past = _log(rng, 16, 12000)
            c |= {"requests": _log(rng, 1, 128), "past": "%d-%d" % (rng.choice([0, 1, past // 2]), past),
                  "new": "1-%d" % hi if kind != "chunk" else "%d-%d" % (hi // 2, hi),
                  "long_every": 4 if kind == "mixed" else 1, "page": rng.choice([16, 32, 64, 128])}
            longest = past + hi
        else:
            hi = longest = _log(rng, 16, 8192)
            c |= {"requests": _log(rng, 1, 48), "new": "%d-%d" % (rng.choice([1, max(1, hi // 4), hi]), hi)}
        scores = c["requests"] * c["heads"] * hi * longest   # what the plain form lays out
        if scores < 1.2e9 and c["requests"] * kv * longest * c["dim"] < 6e8:
            return c


# ----------------------------------------------------------------- lengths --
def _span(text):
    lo, hi = text.split("-")
    return int(lo), int(hi)


def _between(rng, span, spread):
    lo, hi = _span(span)
    if spread == "log" and hi > lo:
        return _log(rng, max(1, lo), hi) if lo else _log(rng, 1, hi + 1) - 1
    return rng.randint(lo, hi)


def _new_lengths(case):
    rng = random.Random(case["lens"])
    every = case.get("long_every", 1)
    return [_between(rng, case["new"], case["spread"]) if i % every == 0 else 1 for i in range(case["requests"])]


def _past_lengths(case, seed):
    rng = random.Random("%d past %d" % (case["lens"], seed))
    return [_between(rng, case["past"], case["spread"]) for _ in range(case["requests"])]


def _visible(past, new, window):
    """(query, key) pairs of one request, and the keys that any of its tokens sees."""
    pairs = sum(min(past + i + 1, window) if window else past + i + 1 for i in range(new))
    first = max(0, past + 1 - window) if window else 0
    return pairs, past + new - first


def work(case):
    op = case["op"]
    if op == "plan":
        r, t = case["requests"], sum(_new_lengths(case))
        pages = t // case["page"]
        # lengths in, offsets and lengths out; slot, position and request of a token; new pages from the list to the table
        return {"bytes": 16 * r + 4 + 16 * t + 8 * pages, "flops": 0}
    if op == "append":
        vals = 2 * case["tokens"] * case["kv_heads"] * case["dim"]
        return {"bytes": vals * ((4 if case["source"] == "f32" else 2) + 2) + 8 * case["tokens"], "flops": 0}
    new = _new_lengths(case)
    past = _past_lengths(case, 0) if op == "paged" else [0] * len(new)
    pairs = keys = 0
    for p, n in zip(past, new):
        a, b = _visible(p, n, case["window"])
        pairs, keys = pairs + a, keys + b
    t, h, d = sum(new), case["heads"], case["dim"]
    size = t * h * (2 * d * 2 + 4) + keys * case["kv_heads"] * d * 2 * 2
    if op == "paged":
        size += 4 * (keys // case["page"] + 2 * len(new))
    return {"bytes": size, "flops": 4 * d * h * pairs}


# ------------------------------------------------------------------ inputs --
def _int(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _normal(gen, shape, kind):
    return torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32 if kind == "f32" else TYPES[kind])


def _table(gen, lens, page, width, n_pages, spare=0):
    """A block table whose first ceil(len / page) entries of each row are pages of their own, and the pages left."""
    counts = _int([-(-n // page) for n in lens])
    perm = torch.randperm(n_pages, generator=gen, device=DEV).to(torch.int32)
    ends = counts.cumsum(0)
    cols = torch.arange(width, device=DEV)
    at = (ends - counts)[:, None] + cols
    used = sum(-(-n // page) for n in lens)
    return torch.where(cols < counts[:, None], perm[at.clamp(max=n_pages - 1)], -1).to(torch.int32), perm[used:].clone()


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed * 7919 + 17)
    op, s = case["op"], {"case": case}
    if op == "plan":
        new, past, page = _new_lengths(case), _past_lengths(case, seed), case["page"]
        longest = _span(case["past"])[1] + max(new)
        need = sum(-(-(p + n) // page) for p, n in zip(past, new))
        table, free = _table(gen, past, page, -(-longest // page) + 2, need + 8)
        # a program that serves such steps keeps room for a rounded-up count of tokens
        return s | {"past": _int(past), "new": _int(new), "table": table, "free": free, "page": page,
                    "room": -(-sum(new) // 64) * 64, "head": _int([0])}
    if op == "append":
        t, kv, d, page = case["tokens"], case["kv_heads"], case["dim"], case["page"]
        pages = -(-t // page) + 4
        slot = torch.randperm(pages * page, generator=gen, device=DEV)[:t].clone()
        if case["padded"]:
            slot[case["padded"] - 1::case["padded"]] = -1
        # keys and values as parts of one fused projection row
        both = _normal(gen, (t, 2 * kv, d), case["source"])
        return s | {"k": both[:, :kv], "v": both[:, kv:], "slot": slot,
                    "kpool": _normal(gen, (pages, kv, page, d), case["type"]),
                    "vpool": _normal(gen, (pages, kv, page, d), case["type"])}
    new = _new_lengths(case)
    h, kv, d, kind, t = case["heads"], case["kv_heads"], case["dim"], case["type"], sum(new)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    s |= {"cu": _int(cu), "max_new": max(new), "scale": 1 / math.sqrt(d), "window": case["window"]}
    if op == "prompt":
        qkv = _normal(gen, (t, h + 2 * kv, d), kind)   # the rows of a fused projection
        return s | {"q": qkv[:, :h], "k": qkv[:, h:h + kv], "v": qkv[:, h + kv:]}
    past, page = _past_lengths(case, 0), case["page"]
    total = [p + n for p, n in zip(past, new)]
    pages = sum(-(-n // page) for n in total) + 4
    table, _ = _table(gen, total, page, -(-max(total) // page), pages)
    return s | {"q": _normal(gen, (t, h, d), kind), "table": table, "kv_len": _int(total), "max_kv": max(total),
                "kpool": _normal(gen, (pages, kv, page, d), kind), "vpool": _normal(gen, (pages, kv, page, d), kind)}


# ------------------------------------------------------------- plain forms --
def _plain_plan(past, new, table, free, page, room, head):
    ends = new.cumsum(0)
    cu = torch.cat([ends.new_zeros(1), ends]).to(torch.int32)
    have, want = (past + page - 1) // page, (past + new + page - 1) // page
    taken = (want - have).cumsum(0)
    first = head + taken - (want - have)                       # where each request's new pages start in the list
    cols = torch.arange(table.shape[1], device=DEV)
    fresh = (cols >= have[:, None]) & (cols < want[:, None])
    at = (first[:, None] + cols - have[:, None]).clamp(0, free.shape[0] - 1)
    table.copy_(torch.where(fresh, free[at], table))
    tok = torch.arange(room, device=DEV)
    req = torch.searchsorted(ends, tok, right=True)
    real = req < new.shape[0]
    row = req.clamp(max=new.shape[0] - 1)
    pos = past[row] + tok - cu[row]
    slot = table[row, (pos // page).clamp(max=table.shape[1] - 1)].long() * page + pos % page
    return {"table": table, "cu": cu, "kv_len": past + new, "slot": torch.where(real, slot, -1),
            "pos": torch.where(real, pos, -1).to(torch.int32), "req": torch.where(real, req, -1).to(torch.int32),
            "head": (head + taken[-1:]).to(torch.int32)}


def _plain_append(k, v, kpool, vpool, slot):
    page = kpool.shape[2]
    real = slot >= 0
    at = slot[real]
    kpool[at // page, :, at % page] = k[real].to(kpool.dtype)
    vpool[at // page, :, at % page] = v[real].to(vpool.dtype)
    return {"kpool": kpool, "vpool": vpool}


def _plain_attend(q, k, v, cu, kv_len, max_new, scale, window):
    """q packed [T, H, D]; k, v padded [R, KV, L, D] in 32 bits; a request's queries are its last tokens."""
    r, kv, l, d = k.shape
    t, h = q.shape[:2]
    new = cu[1:] - cu[:-1]
    i = torch.arange(max_new, device=DEV)
    at = (cu[:-1, None] + i).clamp(max=t - 1).long()                    # [R, N]
    qp = q[at].float().reshape(r, max_new, kv, h // kv, d).permute(0, 2, 3, 1, 4)
    scores = (qp.reshape(r, kv, -1, d) @ k.transpose(2, 3)).reshape(r, kv, h // kv, max_new, l) * scale
    last = (kv_len - new)[:, None] + i                                  # the last key that a token sees
    key = torch.arange(l, device=DEV)
    seen = key <= last[..., None]
    if window:
        seen &= key > last[..., None] - window
    scores = scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.reshape(r, kv, -1, l) @ v).reshape(r, kv, h // kv, max_new, d) / total
    lse = (top + total.log())[..., 0]
    tok = torch.arange(t, device=DEV)
    row = torch.searchsorted(cu, tok, right=True) - 1
    col = tok - cu[row]
    o = o.permute(0, 3, 1, 2, 4)[row, col].reshape(t, h, d)
    return {"out": o.to(q.dtype), "lse": lse.permute(0, 3, 1, 2)[row, col].reshape(t, h)}


def _plain_paged(s):
    page = s["kpool"].shape[2]
    table = s["table"][:, :-(-s["max_kv"] // page)].clamp(min=0).long()

    def rows(pool):
        g = pool[table]                                                 # [R, pages, KV, page, D]
        return g.permute(0, 2, 1, 3, 4).reshape(table.shape[0], pool.shape[1], -1, pool.shape[3]).float()

    return _plain_attend(s["q"], rows(s["kpool"]), rows(s["vpool"]), s["cu"], s["kv_len"], s["max_new"], s["scale"],
                         s["window"])


def _plain_prompt(s):
    cu = s["cu"]
    at = (cu[:-1, None] + torch.arange(s["max_new"], device=DEV)).clamp(max=s["k"].shape[0] - 1).long()
    k, v = (x[at].permute(0, 2, 1, 3).float() for x in (s["k"], s["v"]))
    return _plain_attend(s["q"], k, v, cu, cu[1:] - cu[:-1], s["max_new"], s["scale"], s["window"])


def run(s):
    op = s["case"]["op"]
    if own:
        p = _ops()
        if op == "plan":
            got = p.plan(s["past"], s["new"], s["table"], s["free"], s["page"], s["room"], free_head=s["head"])
            return {"table": s["table"], "cu": got.cu_new, "kv_len": got.kv_len, "slot": got.slot, "pos": got.pos,
                    "req": got.req, "head": got.free_head}
        if op == "append":
            p.append(s["k"], s["v"], s["kpool"], s["vpool"], s["slot"])
            return {"kpool": s["kpool"], "vpool": s["vpool"]}
        if op == "paged":
            out, lse = p.paged_attention(s["q"], s["kpool"], s["vpool"], s["table"], s["cu"], s["kv_len"],
                                         s["max_new"], s["max_kv"], scale=s["scale"], window=s["window"])
        else:
            out, lse = p.prompt_attention(s["q"], s["k"], s["v"], s["cu"], s["max_new"], scale=s["scale"],
                                          window=s["window"])
        return {"out": out, "lse": lse}
    if op == "plan":
        return _plain_plan(s["past"], s["new"], s["table"], s["free"], s["page"], s["room"], s["head"])
    if op == "append":
        return _plain_append(s["k"], s["v"], s["kpool"], s["vpool"], s["slot"])
    return _plain_paged(s) if op == "paged" else _plain_prompt(s)


# ------------------------------------------------------------------- exact --
def _exact_request(q, k, v, scale, window):
    """One request in 64 bits, head by head: q [n, H, D] are the last tokens of k, v [l, KV, D]."""
    n, h, _ = q.shape
    l, kv = k.shape[:2]
    key = torch.arange(l, device=DEV)
    last = torch.arange(l - n, l, device=DEV)[:, None]
    hidden = key > last
    if window:
        hidden |= key <= last - window
    outs, lses = [], []
    for head in range(h):
        x = (q[:, head].double() @ k[:, head * kv // h].double().T) * scale
        x.masked_fill_(hidden, -math.inf)
        lse = torch.logsumexp(x, 1)
        outs.append(torch.exp(x - lse[:, None]) @ v[:, head * kv // h].double())
        lses.append(lse)
    return torch.stack(outs, 1), torch.stack(lses, 1)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "plan":
        page, head = s["page"], int(s["head"])
        past, new, free = s["past"].tolist(), s["new"].tolist(), s["free"].tolist()
        table = s["table"].cpu().numpy().astype(np.int64)
        room = s["room"]
        slot, pos, req = (np.full(room, -1, np.int64) for _ in range(3))
        cu = [0]
        for i, (a, n) in enumerate(zip(past, new)):
            for j in range(-(-a // page), -(-(a + n) // page)):
                table[i, j] = free[head]
                head += 1
            for x in range(n):
                at = cu[-1] + x
                pos[at], req[at] = a + x, i
                slot[at] = table[i, (a + x) // page] * page + (a + x) % page
            cu.append(cu[-1] + n)
        return {"table": table, "cu": np.array(cu), "kv_len": np.array(past) + np.array(new), "slot": slot, "pos": pos,
                "req": req, "head": np.array([head])}
    if op == "append":
        page, slot = s["kpool"].shape[2], s["slot"].cpu().numpy()
        real = torch.from_numpy(np.flatnonzero(slot >= 0)).to(DEV)
        pages, places = (torch.from_numpy(x[slot >= 0]).to(DEV) for x in (slot // page, slot % page))
        for pool, x in ((s["kpool"], s["k"]), (s["vpool"], s["v"])):
            flat = pool.transpose(1, 2).double()      # [page, position, head, dim]
            flat.index_put_((pages, places), x.double().index_select(0, real).to(pool.dtype).double())
            pool.copy_(flat.transpose(1, 2))
        return {"kpool": s["kpool"], "vpool": s["vpool"]}
    cu = s["cu"].tolist()
    outs, lses = [], []
    for i, (a, b) in enumerate(zip(cu, cu[1:])):
        if op == "prompt":
            k, v = s["k"][a:b], s["v"][a:b]
        else:
            n = int(s["kv_len"][i])
            pages = s["table"][i, :-(-n // case["page"])].long()
            k, v = (p[pages].transpose(1, 2).flatten(0, 1)[:n] for p in (s["kpool"], s["vpool"]))
        o, lse = _exact_request(s["q"][a:b], k, v, s["scale"], s["window"])
        outs.append(o)
        lses.append(lse)
    return {"out": torch.cat(outs), "lse": torch.cat(lses)}
