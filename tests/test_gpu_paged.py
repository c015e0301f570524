"""The paged cache on the device against 64-bit arithmetic: placements, rotations, norms and attention at the sizes, masks and
layouts where they can go wrong (bounds: tests/paged_ref.py)."""
import pytest
import torch

from paged_ref import BF16, F32, TYPES, Case, check, rotated

pytestmark = pytest.mark.gpu
if torch.cuda.is_available():
    from mojolearn_b200 import _native, paged, torch_ops

HEADS = [(12, 12, 64), (16, 2, 128), (28, 4, 128), (8, 1, 80), (6, 6, 96), (4, 4, 8), (40, 8, 128), (20, 4, 64), (33, 1, 64)]


def attend(c, **kw):
    if "max_new" not in kw:
        kw["max_new"] = max(1, max(c.new))
    return paged.attention(c.q, c.k_cache, c.v_cache, *c.args(), **kw)


def held_to_64_bits(c, window=0, softcap=0.0, scale=None, **kw):
    got = attend(c, window=window, softcap=softcap, scale=scale, **kw)
    check(got, c.attention(window, softcap, scale), c.rows, c.most())
    torch_ops.check_status()
    return got


# ---- attention ----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows,cache", TYPES)
@pytest.mark.parametrize("heads,kv,hd", HEADS)
def test_single_tokens(rows, cache, heads, kv, hd):
    held_to_64_bits(Case([1] * 7, [0, 1, 14, 15, 16, 200, 777], heads, kv, hd, 16, rows, cache, seed=heads))


@pytest.mark.parametrize("rows,cache", TYPES)
@pytest.mark.parametrize("heads,kv,hd", HEADS)
def test_chunks(rows, cache, heads, kv, hd):
    held_to_64_bits(Case([130, 1, 17, 64, 255], [0, 300, 77, 512, 1], heads, kv, hd, 32, rows, cache, seed=heads))


@pytest.mark.parametrize("rows,cache", TYPES)
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("new", [1, 3, 150])
def test_pages(rows, cache, page, new):
    """Lengths at, before and past the ends of pages and tiles."""
    past = [0, page - 1, page, page + 1, 127, 128, 129, 300]
    held_to_64_bits(Case([new] * len(past), past, 8, 2, 64, page, rows, cache, seed=page))


@pytest.mark.parametrize("rows,cache", TYPES)
@pytest.mark.parametrize("new", [1, 2, 5, 9, 40, 300])
@pytest.mark.parametrize("window", [1, 2, 33, 64, 200, 5000])
def test_windows(rows, cache, new, window):
    held_to_64_bits(Case([new, new, 1], [0, 500, 129], 8, 2, 64, 16, rows, cache, seed=window), window=window)


@pytest.mark.parametrize("rows,cache", TYPES)
@pytest.mark.parametrize("new", [1, 3, 90])
def test_capped_scores_and_scales(rows, cache, new):
    c = Case([new] * 3, [0, 65, 400], 8, 2, 128, 64, rows, cache, sharp=4.0)
    held_to_64_bits(c, softcap=5.0)
    held_to_64_bits(c, softcap=50.0, window=70)
    held_to_64_bits(c, scale=0.03)
    held_to_64_bits(c, scale=0.0)


@pytest.mark.parametrize("rows,cache", TYPES)
@pytest.mark.parametrize("new", [[1, 0, 1, 0], [0, 0, 40, 1], [0, 1, 0, 200]])
def test_sequences_without_rows_and_empty_caches(rows, cache, new):
    """A sequence may have no new token; one whose lengths say less than its rows has rows that see nothing: zero."""
    held_to_64_bits(Case(new, [50, 0, 16, 3], 8, 2, 64, 16, rows, cache))
    short = [0 if n == 1 else max(0, n - 7) for n in new]
    c = Case(new, [0] * 4, 8, 2, 64, 16, rows, cache, lengths=short)
    got = held_to_64_bits(c)
    for b, n in enumerate(new):
        assert not bool(got[c.first[b]:c.first[b] + n - short[b]].any())


@pytest.mark.parametrize("rows,cache", TYPES)
@pytest.mark.parametrize("new", [1, 4, 70])
def test_what_is_not_seen_has_no_influence(rows, cache, new):
    """NaN and infinities past the lengths, in pages of nobody and before a window; page numbers there mean nothing."""
    c = Case([new] * 4, [0, 30, 100, 333], 8, 2, 64, 32, rows, cache, seed=new)
    clean = attend(c, window=50)
    for bad in (float("nan"), float("inf"), torch.finfo(cache).min):
        held = torch.zeros(c.pages, c.page, dtype=torch.bool, device="cuda")
        for b, n in enumerate(c.length):
            for pos in range(max(0, n - new - 50 + 1), n):
                held[int(c.table[b, pos // c.page]), pos % c.page] = True
        for x in (c.k_cache, c.v_cache):
            x.copy_(torch.where(held[:, None, :, None], x, torch.full_like(x, bad)))
        got = attend(c, window=50)
        assert torch.equal(got, clean)


@pytest.mark.parametrize("rows,cache", TYPES)
@pytest.mark.parametrize("new", [1, 2, 6, 60, 300])
def test_a_value_that_is_not_finite_reaches_only_rows_that_see_it(rows, cache, new):
    c = Case([new, new], [40, 500], 8, 2, 64, 16, rows, cache, seed=new)
    for b in (0, 1):
        for pos in (c.length[b] - 1, c.length[b] - new // 2 - 1):
            c.v_cache[int(c.table[b, pos // 16]), :, pos % 16, 5] = float("nan")
    want, got = c.attention(), attend(c)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and bool(torch.isnan(got).any())
    clean = ~torch.isnan(want)
    check(torch.where(clean, got, torch.zeros_like(got)), torch.where(clean, want, 0.0), rows, 6.0)


@pytest.mark.parametrize("rows,cache", TYPES)
@pytest.mark.parametrize("new", [1, 3, 90])
@pytest.mark.parametrize("size", [2.0 ** -66, 2.0 ** -20, 2.0 ** 20, 2.0 ** 50])
def test_capped_scores_of_any_size(rows, cache, new, size):
    """Keys of any magnitude whose scale brings the scores back to ordinary ones."""
    c = Case([new] * 3, [0, 65, 400], 8, 2, 64, 32, rows, cache)
    c.k_cache.mul_(size)
    held_to_64_bits(c, softcap=3.0, scale=0.25 / size)


@pytest.mark.parametrize("rows,cache", TYPES)
@pytest.mark.parametrize("new", [1, 3, 150])
def test_scores_of_minus_infinity(rows, cache, new):
    """Infinite keys: a capped score is the cap; uncapped, a row whose scores are all -infinity has no softmax: NaN. A row without keys is zero."""
    c = Case([new, new], [0, 300], 4, 2, 64, 32, rows, cache, lengths=[new, 0])
    c.q[:, :, 3] = 1.0
    c.k_cache[int(c.table[0, 0]), :, 0, 3] = float("-inf")
    capped = attend(c, softcap=30.0)
    check(capped, c.attention(softcap=30.0), rows, c.most())
    got = attend(c)
    assert bool(torch.isnan(got[0]).all()) and not bool(got[new:].any())
    if new > 1:
        check(got[1:new], c.attention()[1:new], rows, c.most())


@pytest.mark.parametrize("rows,cache", TYPES)
@pytest.mark.parametrize("new", [1, 200])
def test_scores_far_apart(rows, cache, new):
    """Scores of hundreds, rising and falling along the keys: the running maximum moves, and most weights are zero."""
    c = Case([new] * 2, [900, 0], 4, 2, 64, 64, rows, cache, seed=3)
    c.k_cache[:] = (c.k_cache * 40).to(cache)
    each, most = (2.0 ** -7, 3e-5)[rows == F32], c.most()
    # a score of 200 is off by about 2e-5 in 32 bits, and a weight by as much
    off = (attend(c).double() - c.attention()).abs().max()
    assert float(off) <= (each + 4e-4) * most


@pytest.mark.parametrize("rows,cache", TYPES)
def test_row_pitch_padding_and_given_output(rows, cache):
    """Queries as a column block of a wider matrix, rows past the last sequence, an output given by the caller."""
    c = Case([1, 9, 33], [5, 100, 0], 8, 2, 64, 32, rows, cache, pad=5)
    out = torch.full((c.total, 8, 64), 7.0, dtype=rows, device="cuda")
    got = attend(c, out=out)
    assert got is out and bool((out[c.first[-1]:] == 7.0).all())
    assert torch.equal(out[:c.first[-1]], paged.attention(c.q.contiguous(), c.k_cache, c.v_cache, *c.args(), max_new=33)[:c.first[-1]])
    check(out[:c.first[-1]], c.attention()[:c.first[-1]], rows, c.most())
    assert attend(Case([0], [5], 8, 2, 64, 32, rows, cache)).shape == (0, 8, 64)


@pytest.mark.parametrize("rows,cache", TYPES)
@pytest.mark.parametrize("new,past", [(1, 40000), (2, 9000), (17, 9000), (1, 3)])
def test_one_sequence(rows, cache, new, past):
    """One sequence alone: its past is cut over many blocks, or is too short for that."""
    c = Case([new], [past], 8, 2, 128, 64, rows, cache)
    a = held_to_64_bits(c)
    assert torch.equal(a, attend(c)), "the same call gives the same words"
    held_to_64_bits(c, window=4100)


@pytest.mark.parametrize("rows,cache", TYPES)
def test_many_sequences(rows, cache):
    """More sequences than a block has threads, most of them short."""
    new = [(7 * i) % 3 for i in range(700)]
    past = [(13 * i) % 90 if i % 50 else 3000 for i in range(700)]
    held_to_64_bits(Case(new, past, 4, 2, 64, 16, rows, cache))


@pytest.mark.parametrize("rows,cache", TYPES)
def test_bounds_only_cut_the_work(rows, cache):
    """max_length smaller or larger than the lengths changes no answer beyond rounding."""
    c = Case([1, 1, 1], [4000, 10, 700], 8, 2, 128, 64, rows, cache)
    for most in (1, 64, 4001, 1 << 20):
        held_to_64_bits(c, max_length=most)
    c = Case([100, 1, 3], [4000, 10, 700], 8, 2, 128, 64, rows, cache)
    for kw in ({"max_length": 1}, {"max_length": 1 << 20}, {"max_new": 5000}, {"max_new": None}):
        held_to_64_bits(c, **kw)


def test_a_long_pool():
    """Places past 2^31 elements of the pool, for the append as for what reads it."""
    c = Case([1, 70], [300, 0], 8, 2, 128, 64, BF16, BF16)
    pages = (1 << 31) // (2 * 64 * 128) + c.pages + 1
    big = [torch.empty((pages, 2, 64, 128), dtype=BF16, device="cuda") for _ in range(2)]
    for x, small in zip(big, (c.k_cache, c.v_cache)):
        x[pages - c.pages:] = small
    small_table = c.table
    c.table = torch.where(c.table >= 0, c.table + (pages - c.pages), c.table).to(torch.int32)
    paged.append(c.q, c.k, c.v, big[0], big[1], *c.args())
    got = paged.attention(c.q, big[0], big[1], *c.args(), max_new=70)
    c.table = small_table
    paged.append(c.q, c.k, c.v, c.k_cache, c.v_cache, *c.args())
    assert torch.equal(got, attend(c)) and torch.equal(big[0][pages - c.pages:], c.k_cache)
    check(got, c.attention(), BF16, c.most())


@pytest.mark.parametrize("new", [1, 100])
def test_a_page_outside_the_pool_is_reported(new):
    c = Case([new], [200], 8, 2, 64, 16, BF16, BF16)
    page = int(c.table[0, 2])
    c.k_cache[page], c.v_cache[page] = 0, 0
    want = attend(c)
    torch_ops.check_status()
    for wrong in (c.pages, -1, 1 << 30):
        c.table[0, 2] = wrong
        got = attend(c)
        with pytest.raises(_native.NativeError, match="outside the pool"):
            torch_ops.check_status()
        assert torch.equal(got, want)


def test_more_rows_than_the_bound_are_reported():
    c = Case([3, 1], [20, 20], 8, 2, 64, 16, BF16, BF16)
    out = torch.full((4, 8, 64), 7.0, dtype=BF16, device="cuda")
    attend(c, max_new=2, out=out)
    with pytest.raises(_native.NativeError, match="max_new"):
        torch_ops.check_status()
    want = attend(c)
    assert torch.equal(out[3], want[3]) and torch.equal(out[:2], want[:2]) and bool((out[2] == 7.0).all())


# ---- append -------------------------------------------------------------------------------------------------------------

def tables(positions, half, device="cuda"):
    a = torch.arange(positions, device=device, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(half, device=device, dtype=torch.float64) / half)
    return a.cos().float(), a.sin().float()


def near(got, want, scale):
    """A rounding to 8 bits where the type is bfloat16, and 32-bit arithmetic of a norm and a rotation: the root, the quotient,
    two products and a sum, at most 8 roundings of 2^-24 of the larger of the two columns that meet."""
    tol = want.abs() * (2.0 ** -8 if got.dtype == BF16 else 0.0) + scale * 8 * 2.0 ** -24 + 1e-30
    assert bool(((got.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("rows,cache", TYPES)
@pytest.mark.parametrize("heads,kv,hd", HEADS)
@pytest.mark.parametrize("norm", [None, "rmsnorm", "rmsnorm_offset"])
@pytest.mark.parametrize("rope_dim", [None, 0, 4, 32])
def test_append(rows, cache, heads, kv, hd, norm, rope_dim):
    rope_dim = hd if rope_dim is None else min(rope_dim, hd)
    c = Case([1, 0, 37, 5], [0, 20, 100, 15], heads, kv, hd, 16, rows, cache, pad=2, seed=hd)
    cos, sin = tables(140, rope_dim // 2) if rope_dim else (None, None)
    wq, wk = ((torch.rand(hd, device="cuda") + 0.5, torch.rand(hd, device="cuda") + 0.5) if norm else (None, None))
    kb, vb = c.k_cache.clone(), c.v_cache.clone()
    out = torch.full((c.total, heads, hd), 7.0, dtype=rows, device="cuda")
    got = paged.append(c.q, c.k, c.v, c.k_cache, c.v_cache, *c.args(), cos, sin, q_norm=wq, k_norm=wk, norm=norm or "rmsnorm", out=out)
    torch_ops.check_status()
    assert got is out and bool((out[c.first[-1]:] == 7.0).all())
    shift = 1.0 if norm == "rmsnorm_offset" else 0.0
    for b, n in enumerate(c.new):
        at, pos = c.first[b], torch.arange(c.length[b] - n, c.length[b], device="cuda")
        wantq, wantk = rotated(c.q[at:at + n], pos, cos, sin, wq, 1e-6, shift), rotated(c.k[at:at + n], pos, cos, sin, wk, 1e-6, shift)
        near(got[at:at + n], wantq, wantq.abs().amax(-1, keepdim=True) if n else 0.0)
        for i, p in enumerate(pos.tolist()):
            page, slot = int(c.table[b, p // 16]), p % 16
            near(c.k_cache[page, :, slot], wantk[i], wantk[i].abs().amax(-1, keepdim=True))
            assert torch.equal(c.v_cache[page, :, slot], c.v[at + i].to(cache))
            kb[page, :, slot], vb[page, :, slot] = c.k_cache[page, :, slot], c.v_cache[page, :, slot]
    assert torch.equal(kb, c.k_cache) and torch.equal(vb, c.v_cache), "something else was written"


def test_append_refuses_what_lies_outside():
    """A page outside the pool and a position before the sequence: nothing written, the first reported."""
    c = Case([4], [30], 4, 2, 64, 16, BF16, BF16)
    kb, vb = c.k_cache.clone(), c.v_cache.clone()
    keep = c.table.clone()
    c.table[:] = c.pages
    paged.append(c.q, c.k, c.v, c.k_cache, c.v_cache, *c.args())
    with pytest.raises(_native.NativeError, match="outside the pool"):
        torch_ops.check_status()
    c.table = keep
    paged.append(c.q, c.k, c.v, c.k_cache, c.v_cache, c.table, c.cu, torch.zeros_like(c.lengths))
    torch_ops.check_status()
    assert torch.equal(kb, c.k_cache) and torch.equal(vb, c.v_cache)


def test_infinite_and_passed_columns():
    """Columns that are not rotated pass as they are, infinities too; a rotation of none copies."""
    c = Case([3], [5], 4, 2, 64, 16, F32, F32)
    c.q[0, 0, 40] = float("inf")
    c.k[1, 1, 50] = float("-inf")
    cos, sin = tables(8, 16)
    got = paged.append(c.q, c.k, c.v, c.k_cache, c.v_cache, *c.args(), cos, sin)
    assert torch.equal(got[..., 32:], c.q[..., 32:])
    assert torch.equal(paged.append(c.q, c.k, c.v, c.k_cache, c.v_cache, *c.args()), c.q)


# ---- both, as they are used ---------------------------------------------------------------------------------------------

def test_on_another_stream_and_in_a_graph():
    """A step captured once and replayed with other lengths, on a stream of its own."""
    c = Case([1] * 5, [0, 10, 63, 64, 200], 8, 2, 128, 64, F32, BF16, spare=8)
    cos, sin = tables(400, 64)
    table = torch.cat([c.table, torch.full((5, 1), -1, dtype=torch.int32, device="cuda")], dim=1)
    free = sorted(set(range(c.pages)) - set(c.table.flatten().tolist()))
    for b in range(5):
        table[b, -(-c.length[b] // 64)] = free[b]

    def step(q, k, v, lengths):
        r = paged.append(q, k, v, c.k_cache, c.v_cache, table, c.cu, lengths, cos, sin)
        return paged.attention(r, c.k_cache, c.v_cache, table, c.cu, lengths, max_new=1, max_length=300)

    side = torch.cuda.Stream()
    q, k, v, lengths = c.q.clone(), c.k.clone(), c.v.clone(), c.lengths.clone()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(q, k, v, lengths)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step(q, k, v, lengths)
        g = torch.Generator(device="cuda").manual_seed(5)
        for i in range(4):
            for t in (q, k, v):
                t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
            lengths.copy_(c.lengths + i)
            graph.replay()
            got, kc, vc = out.clone(), c.k_cache.clone(), c.v_cache.clone()
            assert torch.equal(step(q, k, v, lengths), got) and torch.equal(kc, c.k_cache) and torch.equal(vc, c.v_cache)
    side.synchronize()


def test_pool():
    cache = paged.PagedCache(8, 2, 64, page=16, layers=2, dtype=F32)
    a, b = cache.open(), cache.open()
    table, cu, lengths = cache.extend([a, b], [17, 3])
    assert cu.tolist() == [0, 17, 20] and lengths.tolist() == [17, 3] and table.shape == (2, 2) and int(table[1, 1]) == -1
    assert cache.pages_for(b, 13) == 0 and cache.pages_for(b, 14) == 1
    with pytest.raises(ValueError, match="REFUSED"):
        cache.extend([a, b], [97, 3])
    assert cache.length == {a: 17, b: 3} and len(cache.free) == 5
    table, cu, lengths = cache.extend([b], [1])
    assert lengths.tolist() == [4] and table.shape == (1, 1)
    cache.close(a)
    assert len(cache.free) == 7
    with pytest.raises(ValueError):
        cache.extend([b, b], [1, 1])


def test_refusals():
    c = Case([2], [5], 4, 2, 64, 16, F32, BF16)
    ok = lambda **kw: paged.attention(kw.pop("q", c.q), kw.pop("k", c.k_cache), kw.pop("v", c.v_cache), kw.pop("table", c.table), kw.pop("cu", c.cu),  # noqa: E731
                                      kw.pop("lengths", c.lengths), **kw)
    ok()
    for kw in ({"q": c.q.half()}, {"q": c.q.cpu()}, {"k": c.k_cache.float()}, {"table": c.table.long()}, {"cu": c.cu.float()}, {"q": c.q.to(BF16), "k": c.k_cache.float(), "v": c.v_cache.float()},
               {"out": torch.empty_like(c.q, dtype=BF16)}):
        with pytest.raises(TypeError):
            ok(**kw)
    for kw in ({"q": c.q[:, :, :32]}, {"q": c.q[0]}, {"q": c.q.transpose(1, 2).contiguous().transpose(1, 2)}, {"cu": c.cu[:1]}, {"lengths": c.lengths.repeat(2)}, {"table": c.table[0]},
               {"k": c.k_cache[:1]}, {"out": torch.empty(1, 4, 64, device="cuda")}, {"k": c.k_cache.transpose(1, 2)}):
        with pytest.raises(ValueError):
            ok(**kw)
    for kw in ({"window": -1}, {"softcap": -1.0}, {"softcap": float("nan")}, {"scale": float("inf")}, {"max_new": 0}, {"max_length": 0}, {"q": c.q[:, :3]}):
        with pytest.raises((_native.NativeError, ValueError)):
            ok(**kw)
    odd = torch.zeros(2, 4 * 64 + 1, device="cuda")[:, :256].unflatten(1, (4, 64))
    with pytest.raises(_native.NativeError, match="16-byte"):
        ok(q=odd)
    for pages, page, hd in ((2, 24, 64), (2, 8, 64), (2, 512, 64), (2, 16, 136), (2, 16, 12)):
        k = torch.zeros(pages, 2, page, hd, dtype=BF16, device="cuda")
        with pytest.raises(_native.NativeError):
            paged.attention(torch.zeros(2, 4, hd, device="cuda"), k, k, c.table, c.cu, c.lengths)
    put = lambda **kw: paged.append(kw.pop("q", c.q), kw.pop("k", c.k), kw.pop("v", c.v), c.k_cache, c.v_cache, c.table, c.cu, c.lengths, **kw)  # noqa: E731
    put()
    t = torch.zeros(10, 16, device="cuda")
    for kw, error in (({"k": c.k[:1]}, ValueError), ({"v": c.v.to(BF16)}, TypeError), ({"cos": t}, ValueError), ({"cos": t, "sin": t[:5]}, ValueError),
                      ({"cos": torch.zeros(10, 33, device="cuda"), "sin": torch.zeros(10, 33, device="cuda")}, ValueError), ({"cos": t.double(), "sin": t.double()}, TypeError),
                      ({"q_norm": torch.zeros(32, device="cuda")}, ValueError), ({"k_norm": torch.zeros(64)}, TypeError), ({"norm": "layernorm"}, ValueError)):
        with pytest.raises(error):
            put(**kw)
