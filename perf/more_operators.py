"""What the speed of the paged cache in 4 bits is measured on.

Keys and values are held as groups of 32 columns of a head: a whole number from -8 to 7 a column, 4 bits, and a bfloat16 scale of
five significant bits a group, the smallest (from 2^-100 on) of which 7 reach the group's largest magnitude. `append` norms, rotates and
places the fresh rows of a call in that form, and `read` gives rows of it back; a write is measured with the reading of what it
wrote, so that its outputs are values. `read` alone gathers whole sequences. `attend` is the attention of a call's rows over such a
cache: single tokens, a few drafted ones, prompts and chunks. A case is one call (a write: two); `listed()` are the fixed cases,
`draw(rng)` gives others of the same ranges.
"""
import math
import random

import torch

own = False
DEV = "cuda"
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}
BYTES = {"float32": 4, "bfloat16": 2}
GROUP = 32


def listed():
    return [
        # the smallest call of a serving loop: one token of one sequence of a 768-wide model
        {"name": "append_one", "op": "append", "batch": 1, "new_lo": 1, "new_hi": 1, "past_lo": 200, "past_hi": 200, "heads": 12, "kv": 12,
         "hd": 64, "rows": "float32", "page": 16, "norm": False, "mix": 1},
        # a decode step of the 2048-wide serving model at its batch
        {"name": "append_step", "op": "append", "batch": 32, "new_lo": 1, "new_hi": 1, "past_lo": 1215, "past_hi": 1278, "heads": 16, "kv": 16,
         "hd": 128, "rows": "float32", "page": 64, "norm": False, "mix": 2},
        # ragged prompts of a model with grouped heads and per-head norms
        {"name": "append_prompts", "op": "append", "batch": 16, "new_lo": 33, "new_hi": 1024, "past_lo": 0, "past_hi": 0, "heads": 32, "kv": 8,
         "hd": 128, "rows": "bfloat16", "page": 64, "norm": True, "mix": 3},
        # one sequence of the 768-wide model taken out of its pages
        {"name": "read_one", "op": "read", "batch": 1, "past_lo": 201, "past_hi": 201, "heads": 12, "kv": 12, "hd": 64, "rows": "float32", "page": 16, "mix": 4},
        # a batch of long sequences taken out, grouped heads
        {"name": "read_batch", "op": "read", "batch": 16, "past_lo": 90, "past_hi": 4000, "heads": 32, "kv": 8, "hd": 128, "rows": "bfloat16", "page": 64, "mix": 5},
        # the attention of the smallest call
        {"name": "one_token", "op": "attend", "batch": 1, "new_lo": 1, "new_hi": 1, "past_lo": 200, "past_hi": 200, "heads": 12, "kv": 12,
         "hd": 64, "rows": "float32", "page": 16, "window": 0, "softcap": 0.0, "mix": 6},
        # the decode step of the serving model, sequences of their own lengths
        {"name": "step_f32", "op": "attend", "batch": 32, "new_lo": 1, "new_hi": 1, "past_lo": 1215, "past_hi": 1278, "heads": 16, "kv": 16,
         "hd": 128, "rows": "float32", "page": 64, "window": 0, "softcap": 0.0, "mix": 7},
        # a decode step of a larger batch with grouped heads, lengths far apart, small pages
        {"name": "step_grouped", "op": "attend", "batch": 64, "new_lo": 1, "new_hi": 1, "past_lo": 90, "past_hi": 8191, "heads": 32, "kv": 8,
         "hd": 128, "rows": "bfloat16", "page": 16, "window": 0, "softcap": 0.0, "mix": 8},
        # one sequence with a very long past: few rows, a long axis
        {"name": "step_long", "op": "attend", "batch": 1, "new_lo": 1, "new_hi": 1, "past_lo": 131000, "past_hi": 131000, "heads": 32, "kv": 8,
         "hd": 128, "rows": "bfloat16", "page": 64, "window": 0, "softcap": 0.0, "mix": 9},
        # drafted tokens checked at once: a few rows a sequence, seven heads a key head, a sliding window and capped scores
        {"name": "step_drafts", "op": "attend", "batch": 24, "new_lo": 5, "new_hi": 5, "past_lo": 90, "past_hi": 8191, "heads": 28, "kv": 4,
         "hd": 128, "rows": "bfloat16", "page": 32, "window": 4096, "softcap": 50.0, "mix": 10},
        # a mixed step of the serving model: chunks of prompts and single tokens together
        {"name": "chunk_ragged", "op": "attend", "batch": 12, "new_lo": 1, "new_hi": 509, "past_lo": 0, "past_hi": 4000, "heads": 16, "kv": 16,
         "hd": 128, "rows": "float32", "page": 64, "window": 0, "softcap": 0.0, "mix": 11},
        # a chunk of a long prompt behind what is cached of it: the largest call
        {"name": "chunk", "op": "attend", "batch": 1, "new_lo": 2048, "new_hi": 2048, "past_lo": 14336, "past_hi": 14336, "heads": 32, "kv": 8,
         "hd": 128, "rows": "bfloat16", "page": 64, "window": 0, "softcap": 0.0, "mix": 12},
    ]


def _span(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(c):
    w = work(c)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    most, room = max(_cost(c) for c in listed()), 4.5e9
    while True:
        op = rng.choice(["append", "attend", "attend", "attend", "read"])
        heads, kv, hd = rng.choice([(12, 12, 64), (16, 16, 128), (32, 8, 128), (28, 4, 128), (8, 1, 128), (16, 4, 64), (20, 20, 80), (24, 8, 96)])
        c = {"op": op, "heads": heads, "kv": kv, "hd": hd, "rows": rng.choice(["float32", "bfloat16"]), "page": rng.choice([16, 32, 64, 128, 256]), "mix": rng.randrange(1 << 20)}
        if op == "read":
            c |= {"batch": _span(rng, 1, 32), "past_hi": _span(rng, 16, 16000)}
            c["past_lo"] = rng.choice([c["past_hi"], 1 + c["past_hi"] // 2, 1 + c["past_hi"] // 16])
        elif rng.random() < 0.6:  # a decode step, now and then of a few tokens a sequence
            new = 1 if rng.random() < 0.6 else rng.randint(2, 8)
            c |= {"batch": _span(rng, 1, 96), "new_lo": new, "new_hi": new, "past_hi": _span(rng, 16, 131000 if op == "attend" else 8000)}
            c["past_lo"] = rng.choice([c["past_hi"], c["past_hi"] // 2, c["past_hi"] // 16])
        else:  # prompts and chunks
            c |= {"batch": _span(rng, 1, 16), "new_hi": _span(rng, 6, 2048)}
            c["new_lo"] = rng.choice([c["new_hi"], 1 + c["new_hi"] // 8])
            c["past_hi"] = rng.choice([0, _span(rng, 16, 14336)])
            c["past_lo"] = rng.choice([0, c["past_hi"]])
        if op == "append":
            c["norm"] = rng.random() < 0.5
        elif op == "attend":
            c["window"] = rng.choice([0, 0, 0, _span(rng, 64, 4096)])
            c["softcap"] = rng.choice([0.0, 0.0, 0.0, 30.0])
        new, past = _sizes(c)
        length = max(n + p for n, p in zip(new, past))
        if _cost(c) <= most and 4 * c["batch"] * length * max(2 * kv * hd, heads * max(new) if op == "attend" else 0) <= room:
            return c


# ---- inputs --------------------------------------------------------------------------------------------------------

def _sizes(c):
    """The rows of a call and the tokens cached before them, sequence by sequence: of the case alone. A read's rows are all that is cached."""
    r = random.Random(c["mix"])
    if c["op"] == "read":
        return [r.randint(c["past_lo"], c["past_hi"]) for _ in range(c["batch"])], [0] * c["batch"]
    return ([r.randint(c["new_lo"], c["new_hi"]) for _ in range(c["batch"])], [r.randint(c["past_lo"], c["past_hi"]) for _ in range(c["batch"])])


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _padded(hd):
    return -(-hd // GROUP) * GROUP


def _quantised(x):
    """x [..., head_dim] as whole numbers and scales of its groups of 32 columns, a last one filled up with zeros: [..., groups, 32], [..., groups, 1]."""
    x = torch.nn.functional.pad(x, (0, _padded(x.shape[-1]) - x.shape[-1])).unflatten(-1, (-1, GROUP))
    part, power = torch.frexp((x.abs().amax(-1, keepdim=True) / 7).clamp(min=2.0 ** -100))
    scale = torch.ldexp(torch.ceil(part * 32) / 32, power)
    return (x / scale).round().clamp(-7, 7), scale


#: eight columns are a 32-bit word: column 2i in its i-th four bits, column 2i + 1 in the (i + 4)-th
_SHIFT = [4 * (i // 2) + 16 * (i % 2) for i in range(8)]


def _packed(codes, scale):
    """Whole numbers and scales of [pages, kv, page, ...] as the bytes of the pages: a page's codes, then its scales."""
    word = sum(((codes.unflatten(-1, (4, 8))[..., i] + 8).to(torch.int64) << _SHIFT[i]) for i in range(8)).to(torch.int32)
    return torch.cat([word.view(torch.uint8).flatten(2), scale.to(torch.bfloat16).view(torch.uint8).flatten(2)], dim=-1)


def _fresh_cache(shape, g):
    """A pool of quantised normal words, a part of it at a time."""
    pages, kv, page, hd = shape
    cache = torch.empty(pages, kv, page, _padded(hd) * 18 // GROUP, dtype=torch.uint8, device=DEV)
    step = max(1, (1 << 25) // (kv * page * hd))
    for i in range(0, pages, step):
        x = torch.randn(min(step, pages - i), kv, page, hd, generator=g, device=DEV)
        cache[i:i + step] = _packed(*_quantised(x)).view(-1, *cache.shape[1:])
    return cache


def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    new, past = _sizes(c)
    rows, page, hd, kv = TYPES[c["rows"]], c["page"], c["hd"], c["kv"]
    total, lengths = sum(new), [n + p for n, p in zip(new, past)]
    used = [-(-n // page) for n in lengths]
    s = {"case": c, "cu": _ints([sum(new[:i]) for i in range(len(new) + 1)]), "lengths": _ints(lengths), "total": total, "max_new": max(new), "max_length": max(lengths)}

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
    s["k_cache"], s["v_cache"] = _fresh_cache((pages, kv, page, hd), g), _fresh_cache((pages, kv, page, hd), g)
    if c["op"] == "attend":
        sharp = torch.linspace(0.5, 3.0, c["heads"], device=DEV)[None, :, None]  # heads attend more or less narrowly
        s["q"] = (normal(total, c["heads"], hd) * sharp).to(rows)
    if c["op"] != "append":
        return s
    fused = normal(total, (c["heads"] + 2 * kv) * hd, dtype=rows)  # the rows of the fused q|k|v product
    wq, wk = c["heads"] * hd, kv * hd
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
        tables = s["table"], s["cu"], s["lengths"]
        if c["op"] == "append":
            q = paged.append(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], *tables, s["cos"], s["sin"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=1e-6)
            k, v = paged.read(s["k_cache"], s["v_cache"], *tables, rows=s["total"], head_dim=c["hd"], dtype=torch.bfloat16)
            return {"q": q, "k": k, "v": v}
        if c["op"] == "read":
            k, v = paged.read(s["k_cache"], s["v_cache"], *tables, rows=s["total"], head_dim=c["hd"], dtype=TYPES[c["rows"]])
            return {"k": k, "v": v}
        return paged.attention(s["q"], s["k_cache"], s["v_cache"], *tables, max_new=s["max_new"], max_length=s["max_length"], window=c["window"], softcap=c["softcap"])
    return {"append": _append, "read": _read, "attend": _attend}[c["op"]](s)


def _rows(s):
    """The sequence of each row and its position in it."""
    t = torch.arange(s["total"], device=DEV)
    seq = (t[:, None] >= s["cu"][None, 1:]).sum(dim=1)
    return seq, t - s["cu"][seq] + (s["lengths"] - s["cu"][1:] + s["cu"][:-1])[seq]


def _normed(x, w):
    return x if w is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w


def _turned(x, cos, sin):
    a, b = x.chunk(2, dim=-1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def _put(cache, where, at, x):
    """Rows x [rows, kv, head_dim] into their places of a cache; the values that they are held as."""
    codes, scale = _quantised(x)
    pages, kv, page, _ = cache.shape
    groups = codes.shape[-2]
    flat = cache.view(pages, kv, -1)
    code_bytes, scale_bytes = flat[..., :16 * groups * page].unflatten(-1, (page, -1)), flat[..., 16 * groups * page:].unflatten(-1, (page, -1))
    packed = _packed(codes, scale)
    code_bytes[where, :, at % page] = packed[..., :16 * groups]
    scale_bytes[where, :, at % page] = packed[..., 16 * groups:]
    return (codes * scale).flatten(-2)[..., :x.shape[-1]].to(torch.bfloat16)


def _append(s):
    # keys in 64 bits: a code is one or the next by less than 32 bits hold where a key is near the middle of two
    page = s["k_cache"].shape[2]
    seq, at = _rows(s)
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    q, k = _turned(_normed(s["q"].float(), s["q_norm"]), cos, sin), _turned(_normed(s["k"].double(), s["k_norm"]), cos.double(), sin.double())
    where = s["table"][seq, at // page].long()
    return {"q": q.to(s["q"].dtype), "k": _put(s["k_cache"], where, at, k), "v": _put(s["v_cache"], where, at, s["v"].double())}


def _unpacked(x, hd):
    """The 32-bit values of pages [..., page, bytes of a row]: [..., page, hd]."""
    page, groups = x.shape[-2], x.shape[-1] // 18
    flat = x.flatten(-2)
    word = flat[..., :16 * groups * page].contiguous().view(torch.int32).unflatten(-1, (page, groups, 4))
    scale = flat[..., 16 * groups * page:].contiguous().view(torch.bfloat16).float().unflatten(-1, (page, groups, 1, 1))
    shift = torch.tensor(_SHIFT, dtype=torch.int32, device=x.device)
    return ((((word[..., None] >> shift) & 15) - 8) * scale).flatten(-3)[..., :hd]


def _read(s):
    hd, dtype, page = s["case"]["hd"], TYPES[s["case"]["rows"]], s["k_cache"].shape[2]
    seq, at = _rows(s)
    place = (s["table"].clamp(min=0).long() * page).repeat_interleave(page, 1)[seq, at] + at % page
    k, v = (_unpacked(s[name], hd).transpose(1, 2).flatten(0, 1)[place] for name in ("k_cache", "v_cache"))
    return {"k": k.to(dtype), "v": v.to(dtype)}


def _gathered(cache, table, inside, hd):
    """A cache's pages in the order of the sequences' positions, [B, KV, positions, hd] in 32 bits, zero where there is none."""
    x = _unpacked(cache[table.clamp(min=0).long()], hd).transpose(1, 2).flatten(2, 3)
    return torch.where(inside[:, None, :, None], x, 0.0)


def _attend(s):
    q, cu, lengths, table, window, softcap = s["q"], s["cu"], s["lengths"], s["table"], s["case"]["window"], s["case"]["softcap"]
    total, heads, hd = q.shape
    kv, page = s["k_cache"].shape[1:3]
    group = heads // kv
    j = torch.arange(table.shape[1] * page, device=DEV)
    inside = j < lengths[:, None]
    k, v = _gathered(s["k_cache"], table, inside, hd), _gathered(s["v_cache"], table, inside, hd)
    i = torch.arange(s["max_new"], device=DEV)
    rows = q[(cu[:-1, None] + i).clamp(max=total - 1)].float()  # [B, new, H, hd]; rows past a sequence's are not read back
    rows = rows.unflatten(2, (kv, group)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    score = (rows @ k.transpose(-1, -2)) * (1.0 / math.sqrt(hd))
    if softcap:
        score = torch.tanh(score / softcap) * softcap
    before = lengths - cu[1:] + cu[:-1]
    at = before[:, None] + i
    seen = (j <= at[..., None]) & inside[:, None]
    if window:
        seen &= j > at[..., None] - window
    score = score.unflatten(2, (group, -1)).masked_fill_(~seen[:, None, None], float("-inf"))
    e = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-3e38))
    out = e.flatten(2, 3) @ v / e.sum(-1).flatten(2, 3)[..., None].clamp(min=1e-30)
    out = out.unflatten(2, (group, -1)).permute(0, 3, 1, 2, 4).flatten(2, 3)
    seq, n = _rows(s)
    return out[seq, n - before[seq]].to(q.dtype)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------

def work(c):
    new, past = _sizes(c)
    total, hd, heads, kv, rb = sum(new), c["hd"], c["heads"], c["kv"], BYTES[c["rows"]]
    held = hd / 2 + 2 * -(-hd // GROUP)  # bytes of a row of a head in the cache
    if c["op"] == "append":  # rows in, queries out, rows into the cache, and their values out
        turns = 4 * hd * min(total, max(n + p for n, p in zip(new, past)))
        return {"bytes": total * ((2 * heads + 2 * kv) * hd * rb + 2 * kv * (held + 2 * hd)) + turns, "flops": total * (heads + kv) * hd * (6 if c["norm"] else 3)}
    if c["op"] == "read":
        return {"bytes": 2 * total * kv * (held + hd * rb), "flops": 2 * total * kv * hd}
    w = c["window"] or 1 << 60
    keys = sum(min(n + p, n + w - 1) for n, p in zip(new, past))
    pairs = sum(sum(min(w, p + i + 1) for i in range(n)) for n, p in zip(new, past))
    return {"bytes": 2 * total * heads * hd * rb + 2 * keys * kv * held, "flops": 4 * pairs * heads * hd}


# ---- the same in 64 bits -------------------------------------------------------------------------------------------

def _nearest(x):
    """x [..., hd] in 64 bits as the values of its 4-bit form: the scale by its bits, rounded up to four behind the first."""
    out = torch.empty_like(x)
    for lo in range(0, x.shape[-1], GROUP):
        part = x[..., lo:lo + GROUP]
        bits = torch.clamp(part.abs().max(dim=-1, keepdim=True).values / 7, min=2.0 ** -100).view(torch.int64)
        scale = ((bits + ((1 << 48) - 1)) & ~((1 << 48) - 1)).view(torch.float64)
        out[..., lo:lo + GROUP] = torch.clamp(torch.round(part / scale), -7, 7) * scale
    return out


def _held(cache, ids, kv, hd):
    """The values of some pages in their order, [kv, positions, hd] in 64 bits, from the bytes' halves."""
    page, groups = cache.shape[2], cache.shape[3] // 18
    flat = cache[ids].reshape(len(ids), kv, -1)
    byte = flat[..., :16 * groups * page].reshape(len(ids), kv, page, groups, 4, 4).to(torch.int64)
    scale = flat[..., 16 * groups * page:].contiguous().view(torch.bfloat16).reshape(len(ids), kv, page, groups, 1).double()
    x = torch.empty(len(ids), kv, page, groups, 4, 8, dtype=torch.float64, device=cache.device)
    for i, (b, high) in enumerate([(0, 0), (2, 0), (0, 1), (2, 1), (1, 0), (3, 0), (1, 1), (3, 1)]):
        x[..., i] = (byte[..., b] // 16 if high else byte[..., b] % 16).double() - 8
    x = x.flatten(-2) * scale
    return x.transpose(0, 1).reshape(kv, len(ids) * page, groups * GROUP)[..., :hd]


def exact(c, seed):
    s = prepare(c, seed)
    new, past = _sizes(c)
    page, hd, kv, first, outs = c["page"], c["hd"], c["kv"], 0, []
    if c["op"] == "append":
        fresh = {n: s[n].double() for n in "qkv"}
        for n in "qk":
            if c["norm"]:
                fresh[n] = fresh[n] / (fresh[n].pow(2).sum(-1, keepdim=True) / hd + 1e-6).sqrt() * s[n + "_norm"].double()
        half = hd // 2
        for n, p in zip(new, past):
            cos, sin = s["cos"][p:p + n, None].double(), s["sin"][p:p + n, None].double()
            for name in "qk":
                x = fresh[name][first:first + n]
                turned = torch.empty_like(x)
                turned[..., :half] = x[..., :half] * cos - x[..., half:] * sin
                turned[..., half:] = x[..., half:] * cos + x[..., :half] * sin
                fresh[name][first:first + n] = turned
            first += n
        return {"q": fresh["q"], "k": _nearest(fresh["k"]), "v": _nearest(fresh["v"])}
    if c["op"] == "read":
        for name in ("k_cache", "v_cache"):
            outs.append(torch.cat([_held(s[name], s["table"][b, :-(-n // page)].long(), kv, hd)[:, :n].transpose(0, 1) for b, n in enumerate(new)]))
        return {"k": outs[0], "v": outs[1]}
    group, window = c["heads"] // kv, c["window"]
    for b, (n, p) in enumerate(zip(new, past)):
        ids = s["table"][b, :-(-(n + p) // page)].long()
        keys, values = (_held(s[name], ids, kv, hd)[:, :n + p] for name in ("k_cache", "v_cache"))
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
