"""What a call's tables may say and what is made of it: lengths past the page table, offsets past the rows, positions past the rotation, windows of
any size, pages that nobody reads."""
import pytest
import torch

from paged_ref import BF16, TYPES, Case, check

pytestmark = pytest.mark.gpu
if torch.cuda.is_available():
    from mojolearn_b200 import _native, paged, torch_ops


def tables(positions, half):
    a = torch.arange(positions, device="cuda")[:, None] * 0.01 * (1 + torch.arange(half, device="cuda"))
    return a.cos(), a.sin()


def both(c, lengths, cu, **kw):
    """Append and attention into outputs of sevens, and the caches before."""
    before = c.k_cache.clone(), c.v_cache.clone()
    q, out = (torch.full((c.total, c.heads, c.hd), 7.0, dtype=c.rows, device="cuda") for _ in range(2))
    paged.append(c.q, c.k, c.v, c.k_cache, c.v_cache, c.table, cu, lengths, out=q)
    appended = int(_native.lib().b200i_decode_status(torch.cuda.current_device()))
    paged.attention(c.q, c.k_cache, c.v_cache, c.table, cu, lengths, max_new=max(c.new), out=out, **kw)
    return before, q, out, appended


@pytest.mark.parametrize("rows,cache", TYPES)
@pytest.mark.parametrize("new", [1, 3, 90])
@pytest.mark.parametrize("what", ["length", "length at the limit", "offset"])
def test_a_sequence_that_its_tables_do_not_hold_is_left_out(rows, cache, new, what):
    """The second of three says more positions than its table has room for, or the last more rows than the call has: nothing of it is written, and
    that is reported; the others are as they were."""
    c = Case([new] * 3, [10, 64 * 3 - new, 40], 4, 2, 64, 64, rows, cache, seed=new)
    c.table = c.table[:, :3].contiguous()
    bad = 2 if what == "offset" else 1
    lengths, cu = c.lengths.clone(), c.cu.clone()
    if what == "offset":
        cu[3] += 5
    else:
        lengths[1] = 64 * 3 + 1 if what == "length at the limit" else 1 << 30
    (kb, vb), q, out, appended = both(c, lengths, cu)
    assert appended == 14
    with pytest.raises(_native.NativeError, match="more positions than its page table"):
        torch_ops.check_status()
    want = c.attention()
    mine = slice(bad * new, bad * new + new)
    assert bool((q[mine] == 7.0).all()) and bool((out[mine] == 7.0).all())
    pages = [int(p) for p in c.table[bad] if p >= 0]
    assert torch.equal(kb[pages], c.k_cache[pages]) and torch.equal(vb[pages], c.v_cache[pages])
    for b in {0, 1, 2} - {bad}:
        at = slice(b * new, b * new + new)
        assert torch.equal(q[at], c.q[at])
        check(out[at], want[at], rows, c.most())


@pytest.mark.parametrize("rows,cache", TYPES)
@pytest.mark.parametrize("hd,half", [(64, 32), (64, 2), (24, 12)])
def test_a_position_past_the_rotation_is_not_written(rows, cache, hd, half):
    c = Case([1, 20], [30, 25], 4, 2, hd, 16, rows, cache)
    cos, sin = tables(40, half)
    whole = tables(60, half)
    kb, vb = c.k_cache.clone(), c.v_cache.clone()
    want = paged.append(c.q, c.k, c.v, kw := c.k_cache.clone(), vw := c.v_cache.clone(), *c.args(), *whole)
    torch_ops.check_status()
    out = torch.full((21, 4, hd), 7.0, dtype=rows, device="cuda")
    paged.append(c.q, c.k, c.v, c.k_cache, c.v_cache, *c.args(), cos, sin, out=out)
    with pytest.raises(_native.NativeError, match="past the rotation"):
        torch_ops.check_status()
    assert torch.equal(out[:16], want[:16]) and bool((out[16:] == 7.0).all())
    for pos in range(25, 45):  # of the second sequence
        page, slot = int(c.table[1, pos // 16]), pos % 16
        for got, before, after in ((c.k_cache, kb, kw), (c.v_cache, vb, vw)):
            assert torch.equal(got[page, :, slot], (after if pos < 40 else before)[page, :, slot])


@pytest.mark.parametrize("rows,cache", TYPES)
@pytest.mark.parametrize("new", [9, 90])
@pytest.mark.parametrize("window", [(1 << 31) - 1, 1 << 31, (1 << 63) - 1])
def test_windows_wider_than_any_cache(rows, cache, new, window):
    """No window at all, also where some rows stand before the beginning of their cache."""
    c = Case([new] * 2, [0, 300], 4, 4, 64, 16, rows, cache, lengths=[2, new + 300])
    kw = {"max_new": new}
    want = paged.attention(c.q, c.k_cache, c.v_cache, *c.args(), **kw)
    assert torch.equal(paged.attention(c.q, c.k_cache, c.v_cache, *c.args(), window=window, **kw), want)
    check(want, c.attention(), rows, c.most())


@pytest.mark.parametrize("rows,cache", TYPES)
@pytest.mark.parametrize("page", [16, 32, 128])
@pytest.mark.parametrize("new", [1, 4, 70, 300])
@pytest.mark.parametrize("nobody", [-1, 1 << 30])
def test_pages_below_the_window_need_no_number(rows, cache, page, new, nobody):
    """Pages that no row sees any more may be given to others: their place in the table is not read as a page."""
    c = Case([new] * 3, [0, 100, 700], 4, 2, 64, page, rows, cache, seed=new)
    call = lambda: paged.attention(c.q, c.k_cache, c.v_cache, *c.args(), max_new=new, window=50)  # noqa: E731
    want = call()
    for b, n in enumerate(c.length):
        c.table[b, :max(0, n - new + 1 - 50) // page] = nobody
    assert torch.equal(call(), want)
    torch_ops.check_status()


def test_a_lazily_copied_cache_is_written_alone():
    """Storage that two tensors share until one of them is written."""
    c = Case([3], [20], 4, 2, 64, 16, BF16, BF16)
    k, v = torch._lazy_clone(c.k_cache), torch._lazy_clone(c.v_cache)
    kb, vb = c.k_cache.clone(), c.v_cache.clone()
    paged.append(c.q, c.k, c.v, k, v, *c.args())
    assert torch.equal(c.k_cache, kb) and torch.equal(c.v_cache, vb)
    assert not torch.equal(k, kb) and not torch.equal(v, vb)


@pytest.mark.parametrize("rows,cache", TYPES)
@pytest.mark.parametrize("heads,hd,half", [(4, 72, 36), (4, 64, 32), (5, 128, 3)])
def test_queries_rotated_in_their_place(rows, cache, heads, hd, half):
    c = Case([1, 20], [30, 25], heads, 1, hd, 16, rows, cache)
    cos, sin = tables(60, half)
    q, want = c.q.contiguous(), paged.append(c.q, c.k, c.v, c.k_cache, c.v_cache, *c.args(), cos, sin)
    kb, vb = c.k_cache.clone(), c.v_cache.clone()
    assert paged.append(q, c.k, c.v, c.k_cache, c.v_cache, *c.args(), cos, sin, out=q) is q
    assert torch.equal(q, want) and torch.equal(c.k_cache, kb) and torch.equal(c.v_cache, vb)
    torch_ops.check_status()
