"""The paged cache in 4 bits on the device: what is written byte for byte, what is read back word for word, and attention against 64-bit arithmetic
at the sizes, masks and layouts where it can go wrong (bounds: tests/paged_ref.py, since what is cached is exactly a bfloat16 word)."""
import pytest
import torch

from paged_int4_ref import Case4, packed, parts, quantised, values
from paged_ref import BF16, F32, Case, check, rotated

pytestmark = pytest.mark.gpu
if torch.cuda.is_available():
    from mojolearn_b200 import _native, paged, torch_ops

ROWS = [F32, BF16]
HEADS = [(12, 12, 64), (16, 2, 128), (28, 4, 128), (8, 1, 80), (6, 6, 96), (4, 4, 8), (40, 8, 128), (20, 4, 64), (33, 1, 64), (6, 2, 40), (4, 2, 104)]


def attend(c, **kw):
    if "max_new" not in kw:
        kw["max_new"] = max(1, max(c.new))
    return paged.attention(c.q, c.k_cache, c.v_cache, *c.args(), **kw)


def held_to_64_bits(c, window=0, softcap=0.0, scale=None, **kw):
    got = attend(c, window=window, softcap=softcap, scale=scale, **kw)
    check(got, c.attention(window, softcap, scale), c.rows, c.most())
    torch_ops.check_status()
    return got


# ---- read ---------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kv,hd", [(12, 64), (2, 128), (1, 80), (6, 96), (3, 8), (2, 40), (5, 104)])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_whole_sequences_are_read_back(kv, hd, page):
    c = Case4([1, 0, page, 3 * page + 5, 200], [0] * 5, kv, kv, hd, page, BF16, seed=hd)
    for dtype in (BF16, F32):
        k, v = paged.read(c.k_cache, c.v_cache, *c.args(), rows=c.total, head_dim=hd, dtype=dtype)
        assert k.dtype == v.dtype == dtype and k.shape == v.shape == (c.total, kv, hd)
        for got, cache in ((k, c.k_cache), (v, c.v_cache)):
            assert torch.equal(got.double(), torch.cat([c.gathered(cache, b).transpose(0, 1) for b in range(5)]))
    torch_ops.check_status()


@pytest.mark.parametrize("rows,cache", [(F32, F32), (F32, BF16), (BF16, BF16)])
def test_caches_of_words_are_read_back(rows, cache):
    c = Case([20, 0, 7, 300], [5, 9, 0, 0], 6, 2, 72, 32, rows, cache)
    k, v = paged.read(c.k_cache, c.v_cache, *c.args(), rows=c.total, dtype=rows)
    for got, x in ((k, c.k_cache), (v, c.v_cache)):
        assert torch.equal(got.double(), torch.cat([c.gathered(x, b).transpose(0, 1)[c.length[b] - n:] for b, n in enumerate(c.new)]))
    assert paged.read(c.k_cache, c.v_cache, *c.args(), rows=c.total)[0].dtype == cache


def test_rows_that_are_not_there_are_zeros_or_left():
    """Positions before the first are zeros, pages outside the pool too and reported; rows past the last sequence are not written."""
    c = Case4([9, 40], [0, 0], 2, 2, 64, 16, BF16, lengths=[4, 40])
    clean = paged.read(c.k_cache, c.v_cache, *c.args(), rows=49, head_dim=64)
    assert not bool(clean[0][:5].any()) and not bool(clean[1][:5].any()) and bool(clean[0][5:].any(-1).all())
    torch_ops.check_status()
    c.table[1, 1] = c.pages
    k, v = paged.read(c.k_cache, c.v_cache, *c.args(), rows=60, head_dim=64)
    with pytest.raises(_native.NativeError, match="outside the pool"):
        torch_ops.check_status()
    assert not bool(k[9 + 16:9 + 32].any()) and torch.equal(k[9 + 32:49], clean[0][9 + 32:]) and torch.equal(v[:25], clean[1][:25])
    k, v = paged.read(c.k_cache, c.v_cache, *c.args(), rows=0, head_dim=64)
    assert k.shape == v.shape == (0, 2, 64)


# ---- append -------------------------------------------------------------------------------------------------------------

def tables(positions, half, device="cuda"):
    a = torch.arange(positions, device=device, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(half, device=device, dtype=torch.float64) / half)
    return a.cos().float(), a.sin().float()


def written(c, wantk, wantv, before):
    """The caches as they are to be: `before` with the quantised keys and values in their places, byte for byte."""
    out = []
    for cache, want in zip(before, (wantk, wantv)):
        codes, scale = parts(cache)
        new, s = quantised(want)
        for b, n in enumerate(c.new):
            for i in range(n):
                p = c.length[b] - n + i
                if p < 0:
                    continue
                at = int(c.table[b, p // c.page]), slice(None), p % c.page
                codes[at], scale[at] = new[c.first[b] + i], s[c.first[b] + i]
        out.append(packed(codes, scale))
    return out


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("heads,kv,hd", HEADS)
@pytest.mark.parametrize("norm", [None, "rmsnorm", "rmsnorm_offset"])
@pytest.mark.parametrize("rope_dim", [None, 0, 6, 32])
def test_append(rows, heads, kv, hd, norm, rope_dim):
    rope_dim = hd if rope_dim is None else min(rope_dim, hd)
    c = Case4([1, 0, 137, 5], [0, 20, 100, 15], heads, kv, hd, 16, rows, pad=2, seed=hd)
    cos, sin = tables(240, rope_dim // 2) if rope_dim else (None, None)
    wq, wk = ((torch.rand(hd, device="cuda") + 0.5, torch.rand(hd, device="cuda") + 0.5) if norm else (None, None))
    before = c.k_cache.clone(), c.v_cache.clone()
    out = torch.full((c.total, heads, hd), 7.0, dtype=rows, device="cuda")
    got = paged.append(c.q, c.k, c.v, c.k_cache, c.v_cache, *c.args(), cos, sin, q_norm=wq, k_norm=wk, norm=norm or "rmsnorm", out=out)
    torch_ops.check_status()
    assert got is out and bool((out[c.first[-1]:] == 7.0).all())
    shift = 1.0 if norm == "rmsnorm_offset" else 0.0
    pos = torch.cat([torch.arange(n - m, n, device="cuda") for n, m in zip(c.length, c.new)])
    turn = lambda x, w: rotated(x[:c.first[-1]], pos, cos, sin, w, 1e-6, shift)  # noqa: E731
    wantq = turn(c.q, wq)
    tol = wantq.abs() * (2.0 ** -8 if rows == BF16 else 0.0) + wantq.abs().amax(-1, keepdim=True) * 8 * 2.0 ** -24 + 1e-30  # as of the caches of words
    assert bool(((got[:c.first[-1]].double() - wantq).abs() <= tol).all())
    for have, want in zip((c.k_cache, c.v_cache), written(c, turn(c.k, wk), c.v[:c.first[-1]], before)):
        assert torch.equal(have, want)


@pytest.mark.parametrize("rows", ROWS)
def test_codes_near_a_border_are_those_of_64_bits(rows):
    """Half a million normed and rotated words, of which 32-bit arithmetic gives another code to some: none differs."""
    c = Case4([1000, 900], [0, 100], 8, 2, 128, 64, rows, seed=11)
    cos, sin = tables(1000, 64)
    w = torch.rand(128, device="cuda") + 0.5
    before = c.k_cache.clone(), c.v_cache.clone()
    paged.append(c.q, c.k, c.v, c.k_cache, c.v_cache, *c.args(), cos, sin, q_norm=w, k_norm=w)
    pos = torch.cat([torch.arange(1000), torch.arange(100, 1000)]).cuda()
    for have, want in zip((c.k_cache, c.v_cache), written(c, rotated(c.k, pos, cos, sin, w), c.v, before)):
        assert torch.equal(have, want)


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("hd,half", [(64, 32), (128, 64), (72, 3), (40, 0)])
def test_words_of_any_kind(rows, hd, half):
    """Ties, zeros, the smallest and the largest words, infinities and NaN: as the definition says, with and without a rotation that leaves them as they are."""
    c = Case4([64], [3], 2, 2, hd, 16, rows, seed=hd)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randint(-28, 29, (64, 2, hd), generator=g, device="cuda").float() / 4  # many are halfway between two codes
    x[0] = 0.0
    x[1] *= 2.0 ** -110
    x[2] *= 2.0 ** -99
    x[3] *= 2.0 ** 100
    x[4, :, 5] = float("inf")
    x[5, :, hd - 1] = float("-inf")
    x[6, :, 0] = float("nan")
    x[7] = 3e38
    x[8] *= 2.0 ** -126
    x[9, 0, 1:] = 0.0
    x = x.to(rows)
    q = torch.zeros_like(x)
    cos, sin = (torch.ones(80, half, device="cuda"), torch.zeros(80, half, device="cuda")) if half else (None, None)
    before = c.k_cache.clone(), c.v_cache.clone()
    paged.append(q, x, x, c.k_cache, c.v_cache, *c.args(), cos, sin)
    finite = x.double()
    if half:  # a rotation by nothing multiplies the partner by zero: an infinity makes both of NaN
        y = finite.clone()
        for lo, hi in ((0, half), (half, 0)):
            y[..., lo:lo + half] += 0.0 * finite[..., hi:hi + half]
        finite = y
    wantk, wantv = written(c, finite, x, before)
    assert torch.equal(c.v_cache, wantv) and torch.equal(c.k_cache, wantk)


def test_append_leaves_what_lies_outside():
    """A page outside the pool and a position before the sequence: nothing written, the first reported."""
    c = Case4([4], [30], 4, 2, 64, 16, BF16)
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


# ---- attention ----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("heads,kv,hd", HEADS)
def test_single_tokens(rows, heads, kv, hd):
    held_to_64_bits(Case4([1] * 7, [0, 1, 14, 15, 16, 200, 777], heads, kv, hd, 16, rows, seed=heads))


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("heads,kv,hd", HEADS)
def test_chunks(rows, heads, kv, hd):
    held_to_64_bits(Case4([130, 1, 17, 64, 255], [0, 300, 77, 512, 1], heads, kv, hd, 32, rows, seed=heads))


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("heads,kv", [(1, 1), (2, 1), (3, 1), (4, 2), (5, 1), (8, 1), (16, 1)])
@pytest.mark.parametrize("new", [1, 2, 3, 4, 5, 8, 16, 24, 33, 40, 41])
def test_a_few_rows(rows, heads, kv, new):
    """Every number of rows of a key head that has a layout of its own, and those next to it."""
    held_to_64_bits(Case4([new, 1, new], [1500, 130, 0], heads, kv, 128, 32, rows, seed=new))


@pytest.mark.parametrize("new,heads,kv", [(3, 7, 1), (5, 28, 4), (20, 2, 1), (40, 2, 2)])
@pytest.mark.parametrize("hd", [8, 64, 80, 96, 128])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_rows_of_drafted_tokens(new, heads, kv, hd, page):
    """17 to 40 rows: the columns of the values shared by two warps where a head is wide, parts of long sequences and whole short ones, a window, caps."""
    c = Case4([new, 1, new, 2], [3000, 200, 0, 700], heads, kv, hd, page, BF16, seed=hd)
    held_to_64_bits(c)
    held_to_64_bits(c, window=300, softcap=20.0)
    held_to_64_bits(Case4([new] * 2, [90, 33], heads, kv, hd, page, BF16, seed=hd), max_length=200)


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("new", [1, 3, 6, 150])
def test_pages(rows, page, new):
    """Lengths at, before and past the ends of pages and tiles."""
    past = [0, page - 1, page, page + 1, 127, 128, 129, 300]
    held_to_64_bits(Case4([new] * len(past), past, 8, 2, 64, page, rows, seed=page))


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("new", [1, 2, 5, 9, 40, 300])
@pytest.mark.parametrize("window", [1, 2, 33, 64, 200, 5000])
def test_windows(rows, new, window):
    held_to_64_bits(Case4([new, new, 1], [0, 500, 129], 8, 2, 64, 16, rows, seed=window), window=window)


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("new", [1, 3, 4, 90])
def test_capped_scores_and_scales(rows, new):
    c = Case4([new] * 3, [0, 65, 400], 8, 2, 128, 64, rows, sharp=4.0)
    held_to_64_bits(c, softcap=5.0)
    held_to_64_bits(c, softcap=50.0, window=70)
    held_to_64_bits(c, scale=0.03)
    held_to_64_bits(c, scale=0.0)
    held_to_64_bits(c, scale=-0.05)


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("new", [[1, 0, 1, 0], [0, 0, 40, 1], [0, 1, 0, 200]])
def test_sequences_without_rows_and_empty_caches(rows, new):
    held_to_64_bits(Case4(new, [50, 0, 16, 3], 8, 2, 64, 16, rows))
    short = [0 if n == 1 else max(0, n - 7) for n in new]
    c = Case4(new, [0] * 4, 8, 2, 64, 16, rows, lengths=short)
    got = held_to_64_bits(c)
    for b, n in enumerate(new):
        assert not bool(got[c.first[b]:c.first[b] + n - short[b]].any())


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("new", [1, 4, 9, 70])
@pytest.mark.parametrize("hd", [64, 128])
def test_what_is_not_seen_has_no_influence(rows, new, hd):
    """Bytes whose scales are NaN or the largest number past the lengths, in pages of nobody and before a window; page numbers there mean nothing."""
    c = Case4([new] * 4, [0, 30, 100, 333], 8, 2, hd, 32, rows, seed=new)
    clean = attend(c, window=50)
    held = torch.zeros(c.pages, c.page, dtype=torch.bool, device="cuda")
    for b, n in enumerate(c.length):
        for pos in range(max(0, n - new - 50 + 1), n):
            held[int(c.table[b, pos // c.page]), pos % c.page] = True
    for bad in (float("nan"), float("inf"), 3.3e38):
        for name in ("k_cache", "v_cache"):
            codes, scale = parts(getattr(c, name))
            codes, scale = torch.where(held[:, None, :, None, None], codes, 15), torch.where(held[:, None, :, None], scale, bad)
            setattr(c, name, packed(codes, scale))
        assert torch.equal(attend(c, window=50), clean)


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("new", [1, 2, 4, 6, 9, 60, 300])
def test_a_group_that_is_not_finite_reaches_only_rows_that_see_it(rows, new):
    c = Case4([new, new], [40, 500], 8, 2, 64, 16, rows, seed=new)
    codes, scale = parts(c.v_cache)
    for b in (0, 1):
        for pos in (c.length[b] - 1, c.length[b] - new // 2 - 1):
            scale[int(c.table[b, pos // 16]), :, pos % 16, 1] = float("nan")
    c.v_cache = packed(codes, scale)
    want, got = c.attention(), attend(c)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and bool(torch.isnan(got).any())
    clean = ~torch.isnan(want)
    check(torch.where(clean, got, torch.zeros_like(got)), torch.where(clean, want, 0.0), rows, 6.0)


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("new,past", [(1, 131000), (5, 30000), (300, 9000)])
@pytest.mark.parametrize("what", ["value", "key", "masked value"])
def test_what_is_not_finite_in_a_long_past(rows, new, past, what):
    c = Case4([new, 1], [past, 700], 8, 2, 128, 64, rows, seed=new)
    pos = c.length[0] - 1 if what == "masked value" else 3
    name = "k_cache" if what == "key" else "v_cache"
    codes, scale = parts(getattr(c, name))
    scale[int(c.table[0, pos // 64]), :, pos % 64, 2] = float("nan")
    setattr(c, name, packed(codes, scale))
    got = attend(c)
    torch_ops.check_status()
    want = c.attention()
    seen = torch.isnan(want)
    assert torch.equal(torch.isnan(got), seen) and int(seen.any(-1).sum()) == (8 if what == "masked value" else 8 * new)
    check(torch.where(seen, torch.zeros_like(got), got), torch.where(seen, 0.0, want), rows, 6.0)


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("new", [1, 3, 90])
def test_scores_far_apart(rows, new):
    """Scores of hundreds, rising and falling along the keys: the largest moves, and most weights are zero."""
    c = Case4([new] * 2, [900, 0], 4, 2, 64, 64, rows, seed=3)
    c.hold(40 * values(c.k_cache, 64), values(c.v_cache, 64))
    each, most = (2.0 ** -7, 3e-5)[rows == F32], c.most()
    # a score of 200 is off by about 2e-5 in 32 bits, and a weight by as much
    off = (attend(c).double() - c.attention()).abs().max()
    assert float(off) <= (each + 4e-4) * most


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("size", [2.0 ** -80, 2.0 ** 60])
@pytest.mark.parametrize("new", [1, 6, 40])
def test_keys_and_values_of_any_size(rows, size, new):
    c = Case4([new] * 2, [300, 0], 4, 2, 64, 64, rows, seed=3)
    plain = c.attention()
    c.hold(size * values(c.k_cache, 64), size * values(c.v_cache, 64))
    check(attend(c, scale=0.125 / size), size * plain, rows, c.most())


@pytest.mark.parametrize("rows", ROWS)
def test_row_pitch_padding_and_given_output(rows):
    c = Case4([1, 9, 33], [5, 100, 0], 8, 2, 64, 32, rows, pad=5)
    out = torch.full((c.total, 8, 64), 7.0, dtype=rows, device="cuda")
    got = attend(c, out=out)
    assert got is out and bool((out[c.first[-1]:] == 7.0).all())
    assert torch.equal(out[:c.first[-1]], paged.attention(c.q.contiguous(), c.k_cache, c.v_cache, *c.args(), max_new=33)[:c.first[-1]])
    check(out[:c.first[-1]], c.attention()[:c.first[-1]], rows, c.most())
    assert attend(Case4([0], [5], 8, 2, 64, 32, rows)).shape == (0, 8, 64)


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("new,past", [(1, 40000), (2, 9000), (4, 20000), (17, 9000), (1, 3)])
def test_one_sequence(rows, new, past):
    """One sequence alone: its past is cut over many blocks, or is too short for that."""
    c = Case4([new], [past], 8, 2, 128, 64, rows)
    a = held_to_64_bits(c)
    assert torch.equal(a, attend(c)), "the same call gives the same words"
    held_to_64_bits(c, window=4100)


@pytest.mark.parametrize("rows", ROWS)
def test_many_sequences(rows):
    """More sequences than a block has threads, most of them short."""
    new = [(7 * i) % 3 for i in range(700)]
    past = [(13 * i) % 90 if i % 50 else 3000 for i in range(700)]
    held_to_64_bits(Case4(new, past, 4, 2, 64, 16, rows))


@pytest.mark.parametrize("rows", ROWS)
def test_bounds_only_cut_the_work(rows):
    c = Case4([1, 1, 1], [4000, 10, 700], 8, 2, 128, 64, rows)
    for most in (1, 64, 4001, 1 << 20):
        held_to_64_bits(c, max_length=most)
    c = Case4([100, 1, 3], [4000, 10, 700], 8, 2, 128, 64, rows)
    for kw in ({"max_length": 1}, {"max_length": 1 << 20}, {"max_new": 5000}, {"max_new": None}):
        held_to_64_bits(c, **kw)


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("new", [1, 4, 100])
@pytest.mark.parametrize("page", [16, 256])
def test_a_page_outside_the_pool_is_reported(rows, new, page):
    """It counts as a page of zeros, as one of scale zero does."""
    c = Case4([new], [800], 8, 2, 64, page, rows)
    codes, scale = parts(c.k_cache)
    scale[int(c.table[0, 2])] = 0.0
    c.k_cache = packed(codes, scale)
    codes, scale = parts(c.v_cache)
    scale[int(c.table[0, 2])] = 0.0
    c.v_cache = packed(codes, scale)
    want = attend(c)
    torch_ops.check_status()
    for wrong in (c.pages, -1, 1 << 30):
        c.table[0, 2] = wrong
        got = attend(c)
        with pytest.raises(_native.NativeError, match="outside the pool"):
            torch_ops.check_status()
        assert torch.equal(got, want)


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("new", [1, 4, 70, 300])
@pytest.mark.parametrize("nobody", [-1, 1 << 30])
def test_pages_below_the_window_need_no_number(page, new, nobody):
    c = Case4([new] * 3, [0, 100, 700], 4, 2, 64, page, BF16, seed=new)
    call = lambda: attend(c, window=50)  # noqa: E731
    want = call()
    for b, n in enumerate(c.length):
        c.table[b, :max(0, n - new + 1 - 50) // page] = nobody
    assert torch.equal(call(), want)
    torch_ops.check_status()


def test_more_rows_than_the_bound_are_reported():
    c = Case4([3, 1], [20, 20], 8, 2, 64, 16, BF16)
    out = torch.full((4, 8, 64), 7.0, dtype=BF16, device="cuda")
    attend(c, max_new=2, out=out)
    with pytest.raises(_native.NativeError, match="max_new"):
        torch_ops.check_status()
    want = attend(c)
    check(out[3:], want[3:].double(), BF16, c.most())
    check(out[:2], want[:2].double(), BF16, c.most())
    assert bool((out[2] == 7.0).all())


@pytest.mark.parametrize("rows", ROWS)
def test_a_sequence_that_its_tables_do_not_hold_is_left_out(rows):
    for new in (1, 3, 90):
        c = Case4([new] * 3, [10, 64 * 3 - new, 40], 4, 2, 64, 64, rows, seed=new)
        c.table = c.table[:, :3].contiguous()
        lengths, before = c.lengths.clone(), (c.k_cache.clone(), c.v_cache.clone())
        lengths[1] = 64 * 3 + 1
        q, out = (torch.full((c.total, 4, 64), 7.0, dtype=rows, device="cuda") for _ in range(2))
        for call in (lambda: paged.append(c.q, c.k, c.v, c.k_cache, c.v_cache, c.table, c.cu, lengths, out=q),
                     lambda: paged.attention(c.q, c.k_cache, c.v_cache, c.table, c.cu, lengths, max_new=new, out=out),
                     lambda: paged.read(c.k_cache, c.v_cache, c.table, c.cu, lengths, rows=c.total, head_dim=64)):
            call()
            with pytest.raises(_native.NativeError, match="more positions than its page table"):
                torch_ops.check_status()
        assert bool((q[new:2 * new] == 7.0).all()) and bool((out[new:2 * new] == 7.0).all()) and torch.equal(q[:new], c.q[:new])
        pages = [int(p) for p in c.table[1] if p >= 0]
        assert torch.equal(before[0][pages], c.k_cache[pages]) and torch.equal(before[1][pages], c.v_cache[pages])
        want = c.attention()
        for at in (slice(0, new), slice(2 * new, 3 * new)):
            check(out[at], want[at], rows, c.most())


def test_a_long_pool():
    """Places past 2^32 bytes of the pool, for what writes and what reads it."""
    c = Case4([1, 70], [300, 0], 8, 2, 128, 64, BF16)
    small = c.k_cache, c.v_cache
    pages = (1 << 32) // (2 * 64 * 72) + c.pages + 1
    big = [torch.empty((pages, 2, 64, 72), dtype=torch.uint8, device="cuda") for _ in range(2)]
    for x, s in zip(big, small):
        x[pages - c.pages:] = s
    far = torch.where(c.table >= 0, c.table + (pages - c.pages), c.table).to(torch.int32)
    paged.append(c.q, c.k, c.v, *big, far, c.cu, c.lengths)
    paged.append(c.q, c.k, c.v, *small, *c.args())
    assert torch.equal(big[0][pages - c.pages:], small[0]) and torch.equal(big[1][pages - c.pages:], small[1])
    for got, want in zip(paged.read(*big, far, c.cu, c.lengths, rows=71, head_dim=128), paged.read(*small, *c.args(), rows=71, head_dim=128)):
        assert torch.equal(got, want)
    for new in (1, 70):
        one = Case4([new], [371 - new], 8, 2, 128, 64, BF16)
        table = torch.arange(pages - 6, pages, dtype=torch.int32, device="cuda")[None]
        near = paged.attention(one.q, *(x[pages - 6:] for x in big), table - (pages - 6), one.cu, one.lengths, max_new=new)
        assert torch.equal(paged.attention(one.q, *big, table, one.cu, one.lengths, max_new=new), near) and bool(torch.isfinite(near).all())


# ---- all, as they are used ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("new", [1, 4, 60])
def test_written_read_and_attended_to(rows, new):
    """Attention over the codes is that over the words that are read back, as a cache of words."""
    c = Case4([new] * 3, [100, 0, 333], 8, 2, 128, 64, rows)
    cos, sin = tables(400, 64)
    q = paged.append(c.q, c.k, c.v, c.k_cache, c.v_cache, *c.args(), cos, sin)
    got = paged.attention(q, c.k_cache, c.v_cache, *c.args(), max_new=new)
    check(got, c.attention(q=q), rows, c.most())
    words = [values(x, 128).to(BF16) for x in (c.k_cache, c.v_cache)]
    check(paged.attention(q, *words, *c.args(), max_new=new), c.attention(q=q), rows, c.most())
    cu = torch.tensor([0] + [sum(c.length[:i + 1]) for i in range(3)], dtype=torch.int32, device="cuda")
    for got, cache in zip(paged.read(c.k_cache, c.v_cache, c.table, cu, c.lengths, rows=sum(c.length), head_dim=128), (c.k_cache, c.v_cache)):
        assert torch.equal(got.double(), torch.cat([c.gathered(cache, b).transpose(0, 1) for b in range(3)]))


@pytest.mark.parametrize("new", [1, 20])
def test_on_another_stream_and_in_a_graph(new):
    """A step captured once and replayed with other rows and lengths, on a stream of its own; two graphs of it in turn."""
    c = Case4([new] * 3, [0, 63, 200], 8, 2, 128, 64, F32, spare=6)
    cos, sin = tables(400, 64)
    table = torch.cat([c.table, torch.full((3, 1), -1, dtype=torch.int32, device="cuda")], dim=1)
    free = sorted(set(range(c.pages)) - set(c.table.flatten().tolist()))
    for b in range(3):
        table[b, -(-c.length[b] // 64)] = free[b]

    def step(q, k, v, lengths):
        r = paged.append(q, k, v, c.k_cache, c.v_cache, table, c.cu, lengths, cos, sin)
        return (paged.attention(r, c.k_cache, c.v_cache, table, c.cu, lengths, max_new=new, max_length=300),) + \
            paged.read(c.k_cache, c.v_cache, table, c.cu, lengths, rows=c.total, head_dim=128)

    side = torch.cuda.Stream()
    q, k, v, lengths = c.q.clone(), c.k.clone(), c.v.clone(), c.lengths.clone()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(q, k, v, lengths)
        side.synchronize()
        graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
        outs = []
        for graph in graphs:
            with torch.cuda.graph(graph, stream=side):
                outs.append(step(q, k, v, lengths))
        g = torch.Generator(device="cuda").manual_seed(5)
        for i in range(4):
            for t in (q, k, v):
                t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
            lengths.copy_(c.lengths + i)
            graphs[i % 2].replay()
            got, kc, vc = [x.clone() for x in outs[i % 2]], c.k_cache.clone(), c.v_cache.clone()
            assert all(torch.equal(x, y) for x, y in zip(step(q, k, v, lengths), got)) and torch.equal(kc, c.k_cache) and torch.equal(vc, c.v_cache)
    side.synchronize()


def test_refusals():
    c = Case4([2], [5], 4, 2, 64, 16, F32)
    calls = lambda k, v, q=c.q: (lambda: paged.append(q, c.k, c.v, k, v, *c.args()), lambda: paged.attention(q, k, v, *c.args()))  # noqa: E731
    wide = torch.zeros(c.pages, 2, 16, 64, dtype=torch.uint8, device="cuda")
    for call in calls(wide, wide) + calls(c.k_cache[:, :, :, :18], c.v_cache[:, :, :, :18]) + calls(c.k_cache, c.v_cache[:1]):
        with pytest.raises(ValueError):
            call()
    for call in calls(c.k_cache, wide.to(torch.int8)) + calls(c.k_cache.to(torch.int8), c.v_cache.to(torch.int8)):
        with pytest.raises(TypeError):
            call()
    get = lambda k=c.k_cache, v=c.v_cache, rows=2, hd=64, **kw: paged.read(k, v, *c.args(), rows=rows, head_dim=hd, **kw)  # noqa: E731
    get()
    for kw, error in (({"hd": None}, ValueError), ({"hd": 32}, ValueError), ({"hd": 96}, ValueError), ({"hd": 60}, _native.NativeError), ({"rows": -1}, ValueError), ({"dtype": torch.float16}, TypeError),
                      ({"k": c.k_cache.cpu()}, TypeError), ({"v": c.v_cache.cpu()}, TypeError), ({"k": wide, "v": wide}, ValueError)):
        with pytest.raises(error):
            get(**kw)
    words = torch.zeros(c.pages, 2, 16, 64, device="cuda")
    with pytest.raises(TypeError):
        get(k=words, v=words, dtype=BF16)
    with pytest.raises(ValueError):
        get(k=words, v=words, hd=32)
    with pytest.raises(TypeError):
        paged.PagedCache(4, 2, 64, dtype="int8")


# ---- caps and scales far from one ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("new", [1, 3, 5, 9, 90, 300])
@pytest.mark.parametrize("cap", [0.01, 1.0, 60.0, 257.0, 1e5, 1e30])
def test_caps_of_any_size(rows, new, cap):
    """A score that is small beside its cap is almost as it was; one that is large is the cap."""
    held_to_64_bits(Case4([new] * 3, [0, 65, 400], 8, 2, 128, 32, rows, seed=new), softcap=cap)


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("new", [1, 6, 90])
@pytest.mark.parametrize("cap", [3.0, 1e8])
@pytest.mark.parametrize("size", [2.0 ** -66, 2.0 ** 50])
def test_caps_with_keys_of_any_size(rows, new, cap, size):
    c = Case4([new] * 3, [0, 65, 400], 8, 2, 64, 32, rows)
    c.hold(size * values(c.k_cache, 64), values(c.v_cache, 64))
    held_to_64_bits(c, softcap=cap, scale=0.25 / size)
