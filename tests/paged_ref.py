"""The paged cache's operators in 64 bits, sequence by sequence, and the making of their inputs."""
import math

import torch

F32, BF16 = torch.float32, torch.bfloat16
TYPES = [(F32, F32), (F32, BF16), (BF16, BF16)]


class Case(object):
    """new[b] rows of sequence b behind past[b] cached positions, pages in no order; `lengths` may say less than that."""

    def __init__(self, new, past, heads, kv, hd, page, rows, cache, seed=0, spare=3, sharp=1.0, lengths=None, pad=0, device="cuda"):
        g = torch.Generator(device=device).manual_seed(seed)
        self.new, self.heads, self.kv, self.hd, self.page, self.rows, self.cache = list(new), heads, kv, hd, page, rows, cache
        self.length = [n + p for n, p in zip(new, past)] if lengths is None else list(lengths)
        self.first = [sum(self.new[:i]) for i in range(len(self.new) + 1)]
        self.total = self.first[-1] + pad
        used = [-(-n // page) for n in self.length]
        self.pages = sum(used) + spare
        order = torch.randperm(self.pages, generator=g, device=device).to(torch.int32)
        self.table = torch.full((len(self.new), max(1, max(used))), -1, dtype=torch.int32, device=device)
        at = 0
        for i, n in enumerate(used):
            self.table[i, :n] = order[at:at + n]
            at += n

        def normal(*shape):
            return torch.randn(shape, generator=g, device=device)

        self.k_cache, self.v_cache = normal(self.pages, kv, page, hd).to(cache), normal(self.pages, kv, page, hd).to(cache)
        self.fused = (normal(max(self.total, 1), (heads + 2 * kv) * hd) * sharp).to(rows)[:self.total]
        w = heads * hd
        self.q, self.k, self.v = (t.unflatten(1, (-1, hd)) for t in (self.fused[:, :w], self.fused[:, w:w + kv * hd], self.fused[:, w + kv * hd:]))
        self.cu = torch.tensor(self.first, dtype=torch.int32, device=device)
        self.lengths = torch.tensor(self.length, dtype=torch.int32, device=device)

    def args(self):
        return self.table, self.cu, self.lengths

    def gathered(self, cache, b):
        """Sequence b's positions [kv, length, hd] in 64 bits."""
        n = self.length[b]
        ids = self.table[b, :-(-n // self.page)].long()
        return cache[ids].double().transpose(0, 1).reshape(self.kv, -1, self.hd)[:, :n]

    def attention(self, window=0, softcap=0.0, scale=None, q=None):
        """[total, heads, hd] in 64 bits; a masked key is left out, not multiplied by zero."""
        q = (self.q if q is None else q).double()
        out = torch.zeros(self.total, self.heads, self.hd, dtype=torch.float64, device=q.device)
        scale = 1 / math.sqrt(self.hd) if scale is None else scale
        for b, n in enumerate(self.new):
            if not n or not self.length[b]:
                continue
            keys, values = self.gathered(self.k_cache, b), self.gathered(self.v_cache, b)
            keys, values = (x.repeat_interleave(self.heads // self.kv, dim=0) for x in (keys, values))
            z = torch.einsum("nhd,hjd->hnj", q[self.first[b]:self.first[b] + n], keys) * scale
            if softcap:
                z = softcap * torch.tanh(z / softcap)
            pos = self.length[b] - n + torch.arange(n, device=q.device)[:, None]
            j = torch.arange(self.length[b], device=q.device)[None]
            seen = (j <= pos) & (j > pos - window) if window else j <= pos
            z = z.masked_fill(~seen, float("-inf"))
            p = torch.exp(z - z.amax(-1, keepdim=True).clamp(min=-1e300))
            p = torch.nan_to_num(p / p.sum(-1, keepdim=True), nan=0.0) if not bool(seen.any(-1).all()) else p / p.sum(-1, keepdim=True)
            dirty = ~torch.isfinite(values).all(-1).all(0)  # positions whose values are not finite: added by hand where they are seen
            o = torch.einsum("hnj,hjd->nhd", p, torch.where(dirty[None, :, None], 0.0, values))
            for at in torch.nonzero(dirty).flatten().tolist():
                o = torch.where(seen[:, at, None, None], o + p[:, :, at].T[..., None] * values[None, :, at], o)
            out[self.first[b]:self.first[b] + n] = o
        return out

    def most(self):
        """The largest magnitude of a value that is in a sequence."""
        return max([float(self.gathered(self.v_cache, b).abs().max()) for b in range(len(self.new)) if self.length[b]] or [1.0])


def bounds(rows):
    """(of one element in units of the largest value, of the 2-norm): how far an output of attention may be off.

    bfloat16: a weight and the output are each rounded once to 8 bits (2^-8 relative each at most); both are random over an
    output's terms, uniform in +-2^-9 .. 2^-8, so the norm is off by about sqrt(2) of 1.7e-3. float32: a weight's two pieces of 8 bits
    leave 2^-16 of it at most and 7e-7 on average; a score of 128 products is off by about 1e-6 of its size."""
    return (2.0 ** -7, 3e-3) if rows == BF16 else (3e-5, 2e-6)


def check(got, want, rows, most):
    each, norm = bounds(rows)
    assert got.dtype == rows and got.shape == want.shape
    assert bool(torch.isfinite(got).all())
    off = (got.double() - want).abs()
    assert float(off.max()) <= each * most, (float(off.max()), each * most)
    size = float(want.norm())
    if size:
        assert float(off.norm()) / size <= norm, float(off.norm()) / size


def rotated(x, pos, cos, sin, weight=None, eps=1e-6, shift=0.0):
    """x [rows, heads, hd] normed per head and rotated to positions pos, in 64 bits."""
    x = x.double()
    if weight is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * (weight.double() + shift)
    if cos is None:
        return x
    half = cos.shape[1]
    c, s = cos[pos].double()[:, None], sin[pos].double()[:, None]
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * half:]], dim=-1)
