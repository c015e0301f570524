"""The paged cache in 4 bits in 64 bits: its quantisation, the order of its bytes, and cases whose caches are held so."""
import torch

from paged_ref import BF16, Case

SHIFTS = [4 * (i // 2) + 16 * (i % 2) for i in range(8)]  # of a 32-bit word's eight columns


def quantised(x):
    """x [..., head_dim] as codes [..., groups, 32] and 64-bit scales [..., groups]: the definition, word for word."""
    x = x.double()
    x = torch.nn.functional.pad(x, (0, -x.shape[-1] % 32)).unflatten(-1, (-1, 32))
    most = x.abs().amax(-1)
    broken = ~torch.isfinite(x).all(-1)
    part, power = torch.frexp(torch.where(broken, 1.0, most).div(7).clamp(min=2.0 ** -100))
    scale = torch.ldexp(torch.ceil(part * 32) / 32, power).clamp(max=2.0 ** 90)
    codes = torch.where(broken[..., None], 0.0, x / scale[..., None]).round().clamp(-7, 7) + 8
    return codes.to(torch.int64), torch.where(broken, float("nan"), scale)


def packed(codes, scale):
    """Codes [pages, kv, page, groups, 32] and scales as the bytes of a cache."""
    pages, kv, page, groups, _ = codes.shape
    word = sum(codes.unflatten(-1, (4, 8))[..., i] << SHIFTS[i] for i in range(8))
    word = torch.where(word >= 1 << 31, word - (1 << 32), word).to(torch.int32).contiguous()
    scale = torch.where(torch.isnan(scale), 0x7FFF, scale.to(BF16).view(torch.int16)).to(torch.int16).contiguous()
    return torch.cat([word.view(torch.uint8).reshape(pages, kv, -1), scale.view(torch.uint8).reshape(pages, kv, -1)], -1).view(pages, kv, page, 18 * groups)


def parts(cache):
    """The codes [pages, kv, page, groups, 32] and the 64-bit scales [pages, kv, page, groups] of a cache's bytes."""
    pages, kv, page, width = cache.shape
    groups = width // 18
    flat = cache.reshape(pages, kv, page * width)
    byte = flat[..., :16 * groups * page].reshape(pages, kv, page, groups, 4, 4).to(torch.int64)
    word = sum(byte[..., i] << (8 * i) for i in range(4))
    codes = torch.stack([(word >> s) & 15 for s in SHIFTS], -1).flatten(-2)
    scale = flat[..., 16 * groups * page:].contiguous().view(BF16).reshape(pages, kv, page, groups).double()
    return codes, scale


def values(cache, hd):
    """What a cache holds, [pages, kv, page, hd] in 64 bits."""
    codes, scale = parts(cache)
    return ((codes - 8) * scale[..., None]).flatten(-2)[..., :hd]


class Case4(Case):
    """A Case whose caches are what quantising its words gives."""

    def __init__(self, new, past, heads, kv, hd, page, rows, **kw):
        super().__init__(new, past, heads, kv, hd, page, rows, torch.float32, **kw)
        self.hold(self.k_cache, self.v_cache)

    def hold(self, k, v):
        self.k_cache, self.v_cache = packed(*quantised(k)), packed(*quantised(v))

    def gathered(self, cache, b):
        n = self.length[b]
        ids = self.table[b, :-(-n // self.page)].long()
        return values(cache[ids], self.hd).transpose(0, 1).reshape(self.kv, len(ids) * self.page, self.hd)[:, :n]
