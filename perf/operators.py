"""What the speed of the paged cache's operators is measured on.

`append` takes the fresh query, key and value rows of a call (a ragged batch: each sequence has its own number of new
tokens), norms queries and keys per head where the model does, rotates them to their positions and places keys and values
in the cache's pages. `attend` is the attention of those rows over the pages: a decode step's single tokens, a prompt, or a
chunk of new tokens behind what is cached. A case is one call; `listed()` are the fixed cases, `draw(rng)` gives others of
the same ranges.
"""
import math
import random

import torch

own = False
DEV = "cuda"
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}
BYTES = {"float32": 4, "bfloat16": 2}


def listed():
    return [
        # the smallest call of a serving loop: one token of one sequence of a 768-wide model
        {"name": "append_one", "op": "append", "batch": 1, "new_lo": 1, "new_hi": 1, "past_lo": 200, "past_hi": 200, "heads": 12, "kv": 12,
         "hd": 64, "rows": "float32", "cache": "float32", "page": 16, "norm": False, "mix": 1},
        # a decode step of the 2048-wide serving model at its batch, keys and values kept in bfloat16
        {"name": "append_step", "op": "append", "batch": 32, "new_lo": 1, "new_hi": 1, "past_lo": 1215, "past_hi": 1278, "heads": 16, "kv": 16,
         "hd": 128, "rows": "float32", "cache": "bfloat16", "page": 64, "norm": False, "mix": 2},
        # ragged prompts of a model with grouped heads and per-head norms
        {"name": "append_prompts", "op": "append", "batch": 16, "new_lo": 33, "new_hi": 1024, "past_lo": 0, "past_hi": 0, "heads": 32, "kv": 8,
         "hd": 128, "rows": "bfloat16", "cache": "bfloat16", "page": 64, "norm": True, "mix": 3},
        # the attention of the smallest call
        {"name": "one_token", "op": "attend", "batch": 1, "new_lo": 1, "new_hi": 1, "past_lo": 200, "past_hi": 200, "heads": 12, "kv": 12,
         "hd": 64, "rows": "float32", "cache": "float32", "page": 16, "window": 0, "softcap": 0.0, "mix": 4},
        # the decode step of the serving model on float32 pages, sequences of their own lengths
        {"name": "step_f32", "op": "attend", "batch": 32, "new_lo": 1, "new_hi": 1, "past_lo": 1215, "past_hi": 1278, "heads": 16, "kv": 16,
         "hd": 128, "rows": "float32", "cache": "float32", "page": 64, "window": 0, "softcap": 0.0, "mix": 5},
        # a decode step of a larger batch with grouped heads, lengths far apart, small pages
        {"name": "step_grouped", "op": "attend", "batch": 64, "new_lo": 1, "new_hi": 1, "past_lo": 90, "past_hi": 8191, "heads": 32, "kv": 8,
         "hd": 128, "rows": "bfloat16", "cache": "bfloat16", "page": 16, "window": 0, "softcap": 0.0, "mix": 6},
        # one sequence with a very long past: few rows, a long axis
        {"name": "step_long", "op": "attend", "batch": 1, "new_lo": 1, "new_hi": 1, "past_lo": 131000, "past_hi": 131000, "heads": 32, "kv": 8,
         "hd": 128, "rows": "bfloat16", "cache": "bfloat16", "page": 64, "window": 0, "softcap": 0.0, "mix": 7},
        # the serving model's prompts: float32 rows over bfloat16 pages, nothing cached before
        {"name": "prompt_mixed", "op": "attend", "batch": 4, "new_lo": 1024, "new_hi": 1024, "past_lo": 0, "past_hi": 0, "heads": 16, "kv": 16,
         "hd": 128, "rows": "float32", "cache": "bfloat16", "page": 64, "window": 0, "softcap": 0.0, "mix": 8},
        # the same prompts on float32 pages
        {"name": "prompt_f32", "op": "attend", "batch": 4, "new_lo": 1024, "new_hi": 1024, "past_lo": 0, "past_hi": 0, "heads": 16, "kv": 16,
         "hd": 128, "rows": "float32", "cache": "float32", "page": 64, "window": 0, "softcap": 0.0, "mix": 9},
        # a chunk of a long prompt behind what is cached of it: the largest call
        {"name": "chunk", "op": "attend", "batch": 1, "new_lo": 2048, "new_hi": 2048, "past_lo": 14336, "past_hi": 14336, "heads": 32, "kv": 8,
         "hd": 128, "rows": "bfloat16", "cache": "bfloat16", "page": 64, "window": 0, "softcap": 0.0, "mix": 10},
        # a mixed step of a serving loop: chunks and single tokens together, a sliding window and capped scores
        {"name": "chunk_ragged", "op": "attend", "batch": 12, "new_lo": 1, "new_hi": 509, "past_lo": 0, "past_hi": 4000, "heads": 28, "kv": 4,
         "hd": 128, "rows": "bfloat16", "cache": "bfloat16", "page": 32, "window": 1024, "softcap": 50.0, "mix": 11},
    ]


def _span(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(c):
    w = work(c)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    most, room = max(_cost(c) for c in listed()), 4.5e9
    while True:
        op = rng.choice(["append", "attend", "attend", "attend"])
        heads, kv, hd = rng.choice([(12, 12, 64), (16, 16, 128), (32, 8, 128), (28, 4, 128), (8, 1, 128), (16, 4, 64), (20, 20, 80), (24, 8, 96)])
        rows = rng.choice(["float32", "bfloat16", "bfloat16"])
        c = {"op": op, "heads": heads, "kv": kv, "hd": hd, "rows": rows, "cache": "bfloat16" if rows == "bfloat16" else rng.choice(["float32", "bfloat16"]),
             "page": rng.choice([16, 32, 64, 128, 256]), "mix": rng.randrange(1 << 20)}
        if rng.random() < 0.5:  # a decode step, now and then of a few tokens a sequence
            new = 1 if rng.random() < 0.7 else rng.randint(2, 5)
            c |= {"batch": _span(rng, 1, 96), "new_lo": new, "new_hi": new, "past_lo": 0, "past_hi": _span(rng, 16, 131000 if op == "attend" else 8000)}
            c["past_lo"] = rng.choice([c["past_hi"], c["past_hi"] // 2, c["past_hi"] // 16])
        else:  # prompts and chunks
            c |= {"batch": _span(rng, 1, 16), "new_hi": _span(rng, 6, 2048)}
            c["new_lo"] = rng.choice([c["new_hi"], 1 + c["new_hi"] // 8])
            c["past_hi"] = rng.choice([0, _span(rng, 16, 14336)])
            c["past_lo"] = rng.choice([0, c["past_hi"]])
        if op == "append":
            c["norm"] = rng.random() < 0.5
        else:
            c["window"] = rng.choice([0, 0, 0, _span(rng, 64, 4096)])
            c["softcap"] = rng.choice([0.0, 0.0, 0.0, 30.0])
        length = c["past_hi"] + c["new_hi"]
        if _cost(c) <= most and 4 * c["batch"] * length * max(2 * kv * hd, heads * c["new_hi"]) <= room:
            return c


# ---- inputs --------------------------------------------------------------------------------------------------------

def _sizes(c):
    """New tokens and tokens cached before, sequence by sequence: of the case alone."""
    r = random.Random(c["mix"])
    return ([r.randint(c["new_lo"], c["new_hi"]) for _ in range(c["batch"])], [r.randint(c["past_lo"], c["past_hi"]) for _ in range(c["batch"])])


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    new, past = _sizes(c)
    rows, cache, page, hd = TYPES[c["rows"]], TYPES[c["cache"]], c["page"], c["hd"]
    total, lengths = sum(new), [n + p for n, p in zip(new, past)]
    used = [-(-n // page) for n in lengths]
    s = {"case": c, "cu": _ints([sum(new[:i]) for i in range(len(new) + 1)]), "lengths": _ints(lengths), "max_new": max(new), "max_length": max(lengths)}

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).mul_(scale).to(dtype)

    # a pool somewhat larger than what is used, its pages handed out in no order; what a page holds past its sequence is stale
    pages = sum(used) + 8
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(new), max(used)), -1, dtype=torch.int32, device=DEV)
    first = 0
    for i, n in enumerate(used):
        table[i, :n] = order[first:first + n]
        first += n
    s["table"] = table
    s["k_cache"] = normal(pages, c["kv"], page, hd, dtype=cache)
    s["v_cache"] = normal(pages, c["kv"], page, hd, dtype=cache)
    if c["op"] == "attend":
        sharp = torch.linspace(0.5, 3.0, c["heads"], device=DEV)[None, :, None]  # heads attend more or less narrowly
        s["q"] = (normal(total, c["heads"], hd) * sharp).to(rows)
        return s
    fused = normal(total, (c["heads"] + 2 * c["kv"]) * hd, dtype=rows)  # the rows of the fused q|k|v product
    wq, wk = c["heads"] * hd, c["kv"] * hd
    s["q"], s["k"], s["v"] = (t.unflatten(1, (-1, hd)) for t in (fused[:, :wq], fused[:, wq:wq + wk], fused[:, wq + wk:]))
    angle = torch.arange(s["max_length"], device=DEV, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(hd // 2, device=DEV, dtype=torch.float64) / (hd // 2))
    s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    s["q_norm"], s["k_norm"] = (1 + normal(hd, scale=0.1), 1 + normal(hd, scale=0.1)) if c["norm"] else (None, None)
    return s


# ---- one pass ------------------------------------------------------------------------------------------------------

def run(s):
    c = s["case"]
    if own:
        from mojolearn_b200 import paged
        if c["op"] == "append":
            q = paged.append(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["cu"], s["lengths"], s["cos"], s["sin"],
                             q_norm=s["q_norm"], k_norm=s["k_norm"], eps=1e-6)
            return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
        return paged.attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["cu"], s["lengths"], max_new=s["max_new"], max_length=s["max_length"],
                               window=c["window"], softcap=c["softcap"])
    return _append(s) if c["op"] == "append" else _attend(s, c["window"], c["softcap"])


def _rows(s):
    """The sequence of each new row and its place in it."""
    t = torch.arange(s["q"].shape[0], device=DEV)
    seq = (t[:, None] >= s["cu"][None, 1:]).sum(dim=1)
    return seq, t - s["cu"][seq]


def _normed(x, w):
    return x if w is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w


def _turned(x, cos, sin):
    a, b = x.chunk(2, dim=-1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def _append(s):
    k_cache, v_cache, page = s["k_cache"], s["v_cache"], s["k_cache"].shape[2]
    seq, i = _rows(s)
    at = (s["lengths"] - s["cu"][1:] + s["cu"][:-1])[seq] + i
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    q, k = _turned(_normed(s["q"].float(), s["q_norm"]), cos, sin), _turned(_normed(s["k"].float(), s["k_norm"]), cos, sin)
    where = s["table"][seq, at // page].long()
    k_cache[where, :, at % page] = k.to(k_cache.dtype)
    v_cache[where, :, at % page] = s["v"].to(v_cache.dtype)
    return {"q": q.to(s["q"].dtype), "k_cache": k_cache, "v_cache": v_cache}


def _gathered(cache, table, inside):
    """A cache's pages in the order of the sequences' positions, [B, KV, positions, hd] in 32 bits, zero where there is none."""
    x = cache[table.clamp(min=0).long()].float().transpose(1, 2).flatten(2, 3)
    return torch.where(inside[:, None, :, None], x, 0.0)


def _attend(s, window, softcap):
    q, cu, lengths, table = s["q"], s["cu"], s["lengths"], s["table"]
    total, heads, hd = q.shape
    kv, page = s["k_cache"].shape[1:3]
    batch, group = lengths.shape[0], heads // kv
    j = torch.arange(table.shape[1] * page, device=DEV)
    inside = j < lengths[:, None]
    k, v = _gathered(s["k_cache"], table, inside), _gathered(s["v_cache"], table, inside)
    i = torch.arange(s["max_new"], device=DEV)
    rows = q[(cu[:-1, None] + i).clamp(max=total - 1)].float()  # [B, new, H, hd]; rows past a sequence's are not read back
    rows = rows.unflatten(2, (kv, group)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    score = (rows @ k.transpose(-1, -2)) * (1.0 / math.sqrt(hd))
    if softcap:
        score = torch.tanh(score / softcap) * softcap
    at = (lengths - cu[1:] + cu[:-1])[:, None] + i
    seen = (j <= at[..., None]) & inside[:, None]
    if window:
        seen &= j > at[..., None] - window
    score = score.unflatten(2, (group, -1)).masked_fill_(~seen[:, None, None], float("-inf"))
    e = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-3e38))
    out = e.flatten(2, 3) @ v / e.sum(-1).flatten(2, 3)[..., None].clamp(min=1e-30)
    out = out.unflatten(2, (group, -1)).permute(0, 3, 1, 2, 4).flatten(2, 3)
    seq, n = _rows(s)
    return out[seq, n].to(q.dtype)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------

def work(c):
    new, past = _sizes(c)
    total, hd, heads, kv = sum(new), c["hd"], c["heads"], c["kv"]
    rb, cb = BYTES[c["rows"]], BYTES[c["cache"]]
    if c["op"] == "append":
        tables = 4 * hd * max(n + p for n, p in zip(new, past)) if c["past_hi"] == 0 else 4 * hd * total
        return {"bytes": total * hd * ((2 * heads + 2 * kv) * rb + 2 * kv * cb) + min(tables, 4 * hd * total), "flops": total * (heads + kv) * hd * (6 if c["norm"] else 3)}
    w = c["window"] or 1 << 60
    keys = sum(min(n + p, n + w - 1) for n, p in zip(new, past))
    pairs = sum(sum(min(w, p + i + 1) for i in range(n)) for n, p in zip(new, past))
    return {"bytes": 2 * total * heads * hd * rb + 2 * keys * kv * hd * cb, "flops": 4 * pairs * heads * hd}


# ---- the same in 64 bits -------------------------------------------------------------------------------------------

def exact(c, seed):
    s = prepare(c, seed)
    new, past = _sizes(c)
    page, hd, first, outs = c["page"], c["hd"], 0, []
    if c["op"] == "append":
        caches = [s["k_cache"].double(), s["v_cache"].double()]
        fresh = {n: s[n].double() for n in "qkv"}
        for n in "qk":
            if c["norm"]:
                fresh[n] = fresh[n] / (fresh[n].pow(2).sum(-1, keepdim=True) / hd + 1e-6).sqrt() * s[n + "_norm"].double()
        half = hd // 2
        for b, (n, p) in enumerate(zip(new, past)):
            cos, sin = s["cos"][p:p + n, None].double(), s["sin"][p:p + n, None].double()
            for name in "qk":
                x = fresh[name][first:first + n]
                turned = torch.empty_like(x)
                turned[..., :half] = x[..., :half] * cos - x[..., half:] * sin
                turned[..., half:] = x[..., half:] * cos + x[..., :half] * sin
                fresh[name][first:first + n] = turned
            pages = s["table"][b].tolist()
            for i in range(p // page, -(-(p + n) // page)):
                lo, hi = max(p, i * page), min(p + n, (i + 1) * page)
                for cache, name in zip(caches, "kv"):
                    cache[pages[i], :, lo % page:lo % page + hi - lo] = fresh[name][first + lo - p:first + hi - p].transpose(0, 1)
            first += n
        return {"q": fresh["q"], "k_cache": caches[0], "v_cache": caches[1]}
    group, window = c["heads"] // c["kv"], c["window"]
    for b, (n, p) in enumerate(zip(new, past)):
        ids = s["table"][b, :-(-(n + p) // page)].long()
        keys, values = (s[name][ids].double().transpose(0, 1).reshape(c["kv"], -1, hd)[:, :n + p] for name in ("k_cache", "v_cache"))
        q = s["q"][first:first + n].double().transpose(0, 1)
        hidden = torch.arange(n + p, device=DEV)[None] > p + torch.arange(n, device=DEV)[:, None]
        if window:
            hidden = hidden | (torch.arange(n + p, device=DEV)[None] <= p + torch.arange(n, device=DEV)[:, None] - window)
        o = torch.empty_like(q)
        for h in range(c["heads"]):
            z = q[h] @ keys[h // group].T / math.sqrt(hd)
            z = c["softcap"] * torch.tanh(z / c["softcap"]) if c["softcap"] else z
            o[h] = torch.softmax(z.masked_fill(hidden, float("-inf")), -1) @ values[h // group]
        outs.append(o.transpose(0, 1))
        first += n
    return torch.cat(outs)
