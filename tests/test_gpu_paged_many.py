"""Attention where a row's output is multiplied tile after tile, and where rows do not come out finite and are done again."""
import pytest
import torch

from paged_ref import BF16, TYPES, Case, check

pytestmark = pytest.mark.gpu
if torch.cuda.is_available():
    from mojolearn_b200 import paged, torch_ops


def climbing(new, past, heads, kv, hd, page, per_tile):
    """A case whose scores climb by about `per_tile` (a factor of e to that) from one 128 keys to the next, along one column."""
    c = Case(new, past, heads, kv, hd, page, BF16, BF16, seed=hd)
    c.q[:, :, 7] = 1.0
    for b, n in enumerate(c.length):
        slope = torch.arange(n, device="cuda") * (per_tile / 128 * hd ** 0.5)
        for i in range(-(-n // page)):
            c.k_cache[int(c.table[b, i]), :, :min(page, n - i * page), 7] = slope[i * page:(i + 1) * page].to(BF16)
    return c


@pytest.mark.parametrize("new,heads,kv", [([300], 4, 4), ([40, 3], 8, 2), ([128, 129], 2, 2), ([70, 20], 8, 1)])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("per_tile", [7.0, 30.0])
def test_an_output_that_is_multiplied_in_every_tile(new, heads, kv, hd, per_tile):
    """Both halves of a row's output are multiplied before a tile's products are added: right, and the same words however the warps run."""
    c = climbing(new, [1500 + 77 * i for i in range(len(new))], heads, kv, hd, 64, per_tile)
    call = lambda: paged.attention(c.q, c.k_cache, c.v_cache, *c.args(), max_new=max(new))  # noqa: E731
    got = call()
    check(got, c.attention(), BF16, c.most())
    for _ in range(20):
        assert torch.equal(call(), got)
    torch_ops.check_status()


@pytest.mark.parametrize("new,past", [(300, 40), (60, 200), (7, 9000), (130, 12000)])
@pytest.mark.parametrize("column", [5, 100])
def test_a_row_done_again_is_written_after_its_other_words(new, past, column):
    """A value that is not finite in one column only, which some rows of a block see and others do not: those are done again as a whole, and
    the same words come out however the warps that store them run."""
    c = Case([new], [past], 8, 2, 128, 32, BF16, BF16, seed=new)
    for back in (1, new // 2, new - 2):
        pos = c.length[0] - back
        c.v_cache[int(c.table[0, pos // 32]), :, pos % 32, column] = float("nan")
    call = lambda: paged.attention(c.q, c.k_cache, c.v_cache, *c.args(), max_new=new)  # noqa: E731
    want, got = c.attention(), call()
    seen = torch.isnan(want)
    assert torch.equal(torch.isnan(got), seen) and bool(seen.any()) and not bool(seen.all(-1).any())
    check(torch.where(seen, torch.zeros_like(got), got), torch.where(seen, 0.0, want), BF16, 6.0)
    for _ in range(20):
        assert torch.equal(call().view(torch.int16), got.view(torch.int16))
    torch_ops.check_status()


@pytest.mark.parametrize("rows,cache", TYPES)
@pytest.mark.parametrize("new,past", [(1, 131000), (5, 30000), (300, 9000), (40, 60000)])
@pytest.mark.parametrize("what", ["value", "key", "masked value"])
def test_what_is_not_finite_in_a_long_past(rows, cache, new, past, what):
    """Every row that sees it, or is beside it, is done again over the whole past: right, without a wait that runs out, and in a time that a wait for
    the others bears (a kernel's waits run out after about a second)."""
    c = Case([new, 1], [past, 700], 8, 2, 128, 64, rows, cache, seed=new)
    pos = c.length[0] - 1 if what == "masked value" else 3
    (c.k_cache if what == "key" else c.v_cache)[int(c.table[0, pos // 64]), :, pos % 64, 9] = float("nan")
    call = lambda: paged.attention(c.q, c.k_cache, c.v_cache, *c.args(), max_new=new)  # noqa: E731
    call()
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    begin.record()
    got = call()
    end.record()
    torch_ops.check_status()
    assert begin.elapsed_time(end) < 250.0
    want = c.attention()
    seen = torch.isnan(want)
    assert torch.equal(torch.isnan(got), seen) and int(seen.any(-1).sum()) == (8 if what == "masked value" else 8 * new)
    check(torch.where(seen, torch.zeros_like(got), got), torch.where(seen, 0.0, want), rows, 6.0)
