"""A paged key-value cache: what writes it, what reads it, and who owns its pages.

`append` takes the fresh query, key and value rows of a call, norms queries and keys per head where the model does,
rotates them to their positions and places keys and values in the cache's pages; `attention` is the attention of the
rotated queries over the pages: a prompt, a chunk of new tokens behind what is cached, or a decode step's single tokens;
`read` gives rows of the cache back. `PagedCache` keeps the pool of pages and hands them to sequences.

The reference keeps one contiguous cache per batch (`TransformerState`, `_transformer_impl.py:194-236`) and has none of
this. It is not part of the identical-mode contract either: sums run in 32 bits in an order that the kernels choose (the
same words for the same call), and the tensor cores take part.

Layout. A cache is `[pages, n_kv_heads, page, head_dim]`, keys and values apart, `page` a power of two from 16 to 256 and
`head_dim` a multiple of 8 up to 128. `page_table` `[batch, max_pages]` int32 names each sequence's pages in the order of its
positions. The rows of all sequences stand one after another: sequence b's are `cu[b]:cu[b + 1]`, and `lengths[b]` counts
what its cache holds with them, so that its last row is at position `lengths[b] - 1`. `cu`, `lengths` and `page_table` are
device tensors and are read by the kernels only, so a call can be captured in a CUDA graph and replayed after they have
changed. Rows and cache are float32 and float32, float32 and bfloat16, or bfloat16 and bfloat16, and either with a cache in 4 bits.

A cache in 4 bits is uint8 `[pages, n_kv_heads, page, row_bytes(head_dim)]`. A head's columns go by groups of 32 (a last one filled up with zeros): a
column is a whole number from -7 to 7 and a group has a bfloat16 scale of five significant bits, the smallest (from 2^-100 to 2^90) of which 7 reach its
largest magnitude; a key or value x is held as the whole number nearest to x / scale, ties to even, of the 64-bit value of x. The product of the two is
a bfloat16 word, so what is held is rounded once and by nothing that reads it. A group with a word that is not finite is held as NaN; words beyond
8.6e27 are cut to that. `include/b200i.h` gives the order of the bytes.

Calls are asynchronous on the current stream. A page number outside the pool is treated as a page of zeros and not written; a
sequence with more positions than its row of the page table has room for, or with offsets that are not the call's, is left
out. Both are reported by `torch_ops.check_status`.
"""
import functools
import math

import torch

from . import _native
from .torch_ops import _bind_host_call, _host_call, _on, _stream, _vp

_TYPES = {torch.float32: 0, torch.bfloat16: 1}
_CACHES = {torch.float32: 0, torch.bfloat16: 1, torch.uint8: 2}
_NORMS = {"rmsnorm": 0, "rmsnorm_offset": 2}


def _bind(name):
    def first(*args):
        if not _bind_host_call():
            return None
        globals()["_plain_" + name] = getattr(_host_call, "paged_" + name)
        return globals()["_plain_" + name](*args)
    return first if _host_call is not None else None


#: the calls on plain device tensors in native code, or None where a call is anything else: those go through the checks below
_plain_append, _plain_attention, _plain_read = _bind("append"), _bind("attention"), _bind("read")


def row_bytes(head_dim):
    """Bytes that a position of a head takes in a cache of 4 bits: 18 for each group of 32 columns."""
    return -(-int(head_dim) // 32) * 18


def _rows(t, name, heads, head_dim, dtype, device, total):
    """The row pitch of `t` [rows, heads, head_dim], whose heads stand side by side."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError("%s must be a CUDA tensor" % name)
    if t.dtype != dtype:
        raise TypeError("%s must be %s, got %s (operands are never cast)" % (name, dtype, t.dtype))
    if t.device != device:
        raise ValueError("operands live on different devices")
    if t.dim() != 3 or (total is not None and t.shape[0] != total) or t.shape[1] != heads or t.shape[2] != head_dim:
        raise ValueError("%s must be (%s, %d, %d), got %s" % (name, "rows" if total is None else total, heads, head_dim, tuple(t.shape)))
    if t.stride(2) != 1 or (heads > 1 and t.stride(1) != head_dim):
        raise ValueError("the heads of %s must stand side by side in each row" % name)
    return t.stride(0) if t.shape[0] > 1 else heads * head_dim


def _cache(k_cache, v_cache, page_table, cu, lengths, row_dtype, device, head_dim):
    for t, name in ((k_cache, "k_cache"), (v_cache, "v_cache"), (page_table, "page_table"), (cu, "cu"), (lengths, "lengths")):
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise TypeError("%s must be a CUDA tensor" % name)
        if t.device != device:
            raise ValueError("operands live on different devices")
        if not t.is_contiguous():
            raise ValueError("%s must be contiguous" % name)
    if k_cache.dtype not in _CACHES or v_cache.dtype != k_cache.dtype or (row_dtype == torch.bfloat16 and k_cache.dtype == torch.float32):
        raise TypeError("rows and caches must be float32 and float32, float32 and bfloat16, bfloat16 and bfloat16, or either and uint8 (4 bits): got %s, %s and %s" %
                        (row_dtype, k_cache.dtype, v_cache.dtype))
    if k_cache.dim() != 4 or v_cache.shape != k_cache.shape:
        raise ValueError("the caches must both be (pages, n_kv_heads, page, head_dim)")
    if k_cache.dtype == torch.uint8 and k_cache.shape[3] != row_bytes(head_dim):
        raise ValueError("a cache in 4 bits must be (pages, n_kv_heads, page, %d) for a head_dim of %d, got %s" % (row_bytes(head_dim), head_dim, tuple(k_cache.shape)))
    for t, name in ((page_table, "page_table"), (cu, "cu"), (lengths, "lengths")):
        if t.dtype != torch.int32:
            raise TypeError("%s must be int32, got %s" % (name, t.dtype))
    if page_table.dim() != 2 or cu.dim() != 1 or lengths.dim() != 1 or lengths.shape[0] != page_table.shape[0] or cu.shape[0] != lengths.shape[0] + 1:
        raise ValueError("page_table must be (batch, max_pages), cu (batch + 1,) and lengths (batch,)")


def _vector(t, name, n, device):
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype != torch.float32:
        raise TypeError("%s must be a float32 CUDA tensor" % name)
    if tuple(t.shape) != (n,) or not t.is_contiguous() or t.device != device:
        raise ValueError("%s must be (%d,), contiguous and on the rows' device" % (name, n))
    return t


@functools.lru_cache(maxsize=None)
def _scale(head_dim):
    return 1.0 / math.sqrt(max(head_dim, 1))


def _head_dim(q, k_cache):
    """The columns of a head: what a cache of words has, or the rows of one in 4 bits."""
    if not isinstance(q, torch.Tensor) or not q.is_cuda or q.dtype not in _TYPES:
        raise TypeError("q must be a float32 or bfloat16 CUDA tensor")
    four = isinstance(k_cache, torch.Tensor) and k_cache.dtype == torch.uint8
    return (q if four else k_cache).shape[-1] if isinstance(k_cache, torch.Tensor) and q.dim() and k_cache.dim() else 0


def _out(out, q):
    if out is None:
        return torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if not isinstance(out, torch.Tensor) or out.dtype != q.dtype or out.device != q.device:
        raise TypeError("out must be a CUDA tensor of the rows' type")
    if out.shape != q.shape or not out.is_contiguous():
        raise ValueError("out must be %s and contiguous" % (tuple(q.shape),))
    return out


def append(q, k, v, k_cache, v_cache, page_table, cu, lengths, cos=None, sin=None, *, q_norm=None, k_norm=None, eps=1e-6, norm="rmsnorm", out=None):
    """Rows q [rows, n_heads, head_dim], k and v [rows, n_kv_heads, head_dim] (column blocks of a fused q|k|v product may be
    given as they are): the rotated queries [rows, n_heads, head_dim], keys and values put in their pages.

    `cos`, `sin` float32 [positions, rope_dim / 2] hold the rotation of every position (None: no rotation); columns from rope_dim on
    pass through, and a row whose position they do not hold is not written and reported by `torch_ops.check_status`. `q_norm`, `k_norm` float32 [head_dim]: an RMSNorm over each head's vector before the rotation, of weight w
    ("rmsnorm") or 1 + w ("rmsnorm_offset"). Rows past cu[-1] belong to no sequence: their part of the answer is not written."""
    if out is None and norm in _NORMS and _plain_append is not None:
        done = _plain_append(q, k, v, k_cache, v_cache, page_table, cu, lengths, cos, sin, q_norm, k_norm, eps, _NORMS[norm])
        if done is not None:
            return done
    hd = _head_dim(q, k_cache)
    _cache(k_cache, v_cache, page_table, cu, lengths, q.dtype, q.device, hd)
    pages, n_kv, page, _ = k_cache.shape
    rows, n_heads = q.shape[0], q.shape[1] if q.dim() == 3 else 0
    ldq = _rows(q, "q", n_heads, hd, q.dtype, q.device, rows)
    ldk, ldv = _rows(k, "k", n_kv, hd, q.dtype, q.device, rows), _rows(v, "v", n_kv, hd, q.dtype, q.device, rows)
    q_norm, k_norm = _vector(q_norm, "q_norm", hd, q.device), _vector(k_norm, "k_norm", hd, q.device)
    if norm not in _NORMS:
        raise ValueError("norm must be one of %s, got %r" % (", ".join(_NORMS), norm))
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    half = positions = 0
    if cos is not None:
        for t, name in ((cos, "cos"), (sin, "sin")):
            if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype != torch.float32:
                raise TypeError("%s must be a float32 CUDA tensor" % name)
            if t.dim() != 2 or not t.is_contiguous() or t.device != q.device or t.shape != cos.shape:
                raise ValueError("cos and sin must both be (positions, rope_dim / 2), contiguous and on the rows' device")
        positions, half = cos.shape
        if half < 1 or 2 * half > hd:
            raise ValueError("a rotation of %d columns does not fit head_dim %d" % (2 * half, hd))
    out = _out(out, q)
    if rows == 0:
        return out
    with _on(q.device):
        _native.call("b200i_paged_append", q.device.index, _stream(q.device), _vp(out), _vp(k_cache), _vp(v_cache), _vp(q), _vp(k), _vp(v), ldq, ldk, ldv,
                     _TYPES[q.dtype], _CACHES[k_cache.dtype], _vp(cos), _vp(sin), 2 * half, positions, _vp(q_norm), _vp(k_norm), float(eps), _NORMS[norm],
                     _vp(page_table), _vp(cu), _vp(lengths), rows, lengths.shape[0], n_heads, n_kv, hd, pages, page, page_table.shape[1])
    return out


def attention(q, k_cache, v_cache, page_table, cu, lengths, *, max_new=None, max_length=None, scale=None, window=0, softcap=0.0, out=None):
    """softmax(scale q.k) v of the rows q [rows, n_heads, head_dim] over the cached positions that each sees: those up to its own
    and, with `window`, the last `window` of them. `softcap` caps every score as cap * tanh(score / cap). A row that sees nothing
    is zero (one whose scores are all -infinity has no softmax: NaN); what stands in places that a row does not see, or past a sequence's length, never reaches it.

    `max_new` and `max_length` are what the caller knows of the most new tokens of a sequence and of the longest cache (by default
    all rows and the whole table): the call is cut by them, and a sequence with more than `max_new` rows is reported by
    `torch_ops.check_status`. `scale` is 1 / sqrt(head_dim) by default. Rows past cu[-1] are not written.

    Scores, statistics and sums are of 32 bits. Weights keep 16 bits or more (float32 rows, and bfloat16 rows of sequences with up to 16 of them
    for a key head, 24 on a cache in 4 bits), so that bfloat16 outputs are off by their own rounding (1.7e-3 of the norm); of more bfloat16 rows a
    weight is one bfloat16 word (2.2e-3 to 2.4e-3 in all).

    More than 512 bfloat16 rows of a sequence and key head over a cache in 4 bits take scratch for its words, of all positions that the page table has
    room for, where that is at most 256 MB; a wider table's codes are read as they are, which is slower."""
    if out is None and max_new is not None and max_length is not None and _plain_attention is not None and isinstance(q, torch.Tensor):
        done = _plain_attention(q, k_cache, v_cache, page_table, cu, lengths, max_new, max_length, _scale(q.shape[-1] if q.dim() else 1) if scale is None else scale, window, softcap)
        if done is not None:
            return done
    hd = _head_dim(q, k_cache)
    _cache(k_cache, v_cache, page_table, cu, lengths, q.dtype, q.device, hd)
    pages, n_kv, page, _ = k_cache.shape
    rows, n_heads, batch, max_pages = q.shape[0], q.shape[1] if q.dim() == 3 else 0, lengths.shape[0], page_table.shape[1]
    ldq = _rows(q, "q", n_heads, hd, q.dtype, q.device, rows)
    max_new = max(rows, 1) if max_new is None else int(max_new)
    max_length = max_pages * page if max_length is None else int(max_length)
    out = _out(out, q)
    if rows == 0:
        return out
    with _on(q.device):
        types = _TYPES[q.dtype], _CACHES[k_cache.dtype]
        need = int(_native.lib().b200i_paged_attention_table_workspace_bytes(q.device.index, *types, rows, batch, n_heads, n_kv, hd, max_new, max_length, int(window),
                                                                               max_pages * page))
        ws = torch.empty((need,), dtype=torch.uint8, device=q.device) if need else None
        _native.call("b200i_paged_attention", q.device.index, _stream(q.device), _vp(out), _vp(q), ldq, _vp(k_cache), _vp(v_cache), *types, _vp(page_table), _vp(cu),
                     _vp(lengths), rows, batch, n_heads, n_kv, hd, pages, page, max_pages, max_new, max_length, _scale(hd) if scale is None else float(scale),
                     int(window), float(softcap), _vp(ws), need)
    return out


def read(k_cache, v_cache, page_table, cu, lengths, *, rows, head_dim=None, dtype=None):
    """What the caches hold at the positions of `rows` rows: keys and values [rows, n_kv_heads, head_dim]. Sequence b's rows are cu[b]:cu[b + 1], the last
    of its lengths[b] positions as in a call that wrote them; with `cu` the running sums of `lengths` they are all of each sequence.

    `head_dim` is the caches' own unless they are in 4 bits. `dtype` is float32 or, of caches in bfloat16 and 4 bits, bfloat16, which holds what they
    hold exactly and is the default there. A row at a position before the first, or in a page outside the pool, is zeros; rows past cu[-1] are not written."""
    if not isinstance(k_cache, torch.Tensor) or not k_cache.is_cuda or k_cache.dtype not in _CACHES:
        raise TypeError("k_cache must be a float32, bfloat16 or uint8 CUDA tensor")
    four = k_cache.dtype == torch.uint8
    if head_dim is None:
        if four:
            raise ValueError("a cache in 4 bits does not say what its head_dim is")
        head_dim = k_cache.shape[-1]
    if dtype is None:
        dtype = torch.bfloat16 if four else k_cache.dtype
    if dtype not in _TYPES:
        raise TypeError("rows are read as float32 or bfloat16, got %s" % (dtype,))
    if _plain_read is not None:
        done = _plain_read(k_cache, v_cache, page_table, cu, lengths, rows, head_dim, _TYPES[dtype])
        if done is not None:
            return done
    rows, head_dim, device = int(rows), int(head_dim), k_cache.device
    _cache(k_cache, v_cache, page_table, cu, lengths, dtype, device, head_dim)
    pages, n_kv, page, width = k_cache.shape
    if not four and width != head_dim:
        raise ValueError("the caches have a head_dim of %d, not %d" % (width, head_dim))
    if rows < 0:
        raise ValueError("rows must not be negative, got %d" % rows)
    k, v = (torch.empty((rows, n_kv, head_dim), dtype=dtype, device=device) for _ in range(2))
    if rows == 0:
        return k, v
    with _on(device):
        _native.call("b200i_paged_read", device.index, _stream(device), _vp(k), _vp(v), _vp(k_cache), _vp(v_cache), _TYPES[dtype], _CACHES[k_cache.dtype],
                     _vp(page_table), _vp(cu), _vp(lengths), rows, lengths.shape[0], n_kv, head_dim, pages, page, page_table.shape[1])
    return k, v


class PagedCache(object):
    """A pool of pages for the layers of one model, and the sequences that hold them.

    `open()` begins a sequence, `extend(sequences, counts)` takes the pages that so many further tokens of each need and gives the
    (page_table, cu, lengths) of a call over them, `close(sequence)` gives its pages back. All layers share the page numbers; `k[i]`
    and `v[i]` are layer i's caches, of words of `dtype` or, with dtype "int4", in 4 bits. Sequences and free pages are kept on the host, so nothing here waits for the device."""

    def __init__(self, n_pages, n_kv_heads, head_dim, *, page=64, layers=1, dtype=torch.bfloat16, device=None):
        if dtype not in _TYPES and dtype != "int4":
            raise TypeError("a cache is float32, bfloat16 or \"int4\", got %s" % (dtype,))
        if n_pages < 1 or layers < 1 or n_kv_heads < 1:
            raise ValueError("a cache has at least one page, one key head and one layer")
        if page < 16 or page > 256 or page & (page - 1):
            raise ValueError("a page holds a power of two from 16 to 256 positions, got %r" % (page,))
        if head_dim < 8 or head_dim > 128 or head_dim % 8:
            raise ValueError("head_dim must be a multiple of 8 up to 128, got %r" % (head_dim,))
        _native.require_device()
        self.device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        self.page, self.pages, self.dtype = int(page), int(n_pages), dtype
        self.head_dim, four = int(head_dim), dtype == "int4"
        shape = (self.pages, int(n_kv_heads), self.page, row_bytes(head_dim) if four else self.head_dim)
        self.k = [torch.zeros(shape, dtype=torch.uint8 if four else dtype, device=self.device) for _ in range(layers)]
        self.v = [torch.zeros(shape, dtype=torch.uint8 if four else dtype, device=self.device) for _ in range(layers)]
        self.free = list(range(self.pages - 1, -1, -1))
        self.held, self.length, self._next = {}, {}, 0

    def open(self):
        name, self._next = self._next, self._next + 1
        self.held[name], self.length[name] = [], 0
        return name

    def close(self, sequence):
        self.free.extend(reversed(self.held.pop(sequence)))
        del self.length[sequence]

    def pages_for(self, sequence, count):
        """How many further pages `count` more tokens of a sequence take."""
        return max(0, -(-(self.length[sequence] + count) // self.page) - len(self.held[sequence]))

    def retract(self, sequences, counts):
        """Take back an `extend` whose tokens were not written: the lengths and pages are as before it. What was queued on the device for
        them may still run; pages go to later calls on the same stream."""
        for s, n in reversed(list(zip(sequences, counts))):
            if not 0 <= n <= self.length[s]:
                raise ValueError("sequence %r has %d tokens, not %d to take back" % (s, self.length[s], n))
            self.length[s] -= n
            keep = -(-self.length[s] // self.page)
            self.free.extend(reversed(self.held[s][keep:]))
            del self.held[s][keep:]

    def extend(self, sequences, counts):
        """Room for counts[i] more tokens of sequences[i]: (page_table, cu, lengths) on the device. Refused as a whole, with no
        page taken, where the pool has too few left."""
        sequences, counts = list(sequences), [int(n) for n in counts]
        if len(sequences) != len(counts) or not counts or any(n < 0 for n in counts) or len(set(sequences)) != len(sequences):
            raise ValueError("extend takes different sequences and a count that is not negative for each")
        need = [self.pages_for(s, n) for s, n in zip(sequences, counts)]
        if sum(need) > len(self.free):
            raise ValueError("paged cache: %d pages are wanted and %d are free REFUSED" % (sum(need), len(self.free)))
        at, held = len(self.free), []
        for s, m in zip(sequences, need):
            held.append(self.held[s] + self.free[at - m:at][::-1])
            at -= m
        lengths, width = [self.length[s] + n for s, n in zip(sequences, counts)], max(1, max(len(h) for h in held))
        cu = [0]
        for n in counts:
            cu.append(cu[-1] + n)
        # one copy to the device for all three, and nothing is taken before it is on its way
        flat = cu + lengths
        for h in held:
            flat.extend(h)
            flat.extend([-1] * (width - len(h)))
        t = torch.tensor(flat, dtype=torch.int32, pin_memory=True).to(self.device, non_blocking=True)
        b = len(sequences)
        tables = t[2 * b + 1:].view(b, width), t[:b + 1], t[b + 1:2 * b + 1]
        for s, h, n in zip(sequences, held, lengths):
            self.held[s], self.length[s] = h, n
        del self.free[at:]
        return tables
