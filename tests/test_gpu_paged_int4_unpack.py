"""More than 512 bfloat16 rows of a sequence and key head over a cache in 4 bits: the words are made once, in the workspace, and attended to there."""
import ctypes

import pytest
import torch

from paged_int4_ref import Case4
from paged_ref import BF16, check

pytestmark = pytest.mark.gpu
if torch.cuda.is_available():
    from mojolearn_b200 import _native, paged, torch_ops


def widened(c, positions):
    """The case's page table with room for `positions`; the numbers behind its own mean nothing."""
    more = positions // c.page - c.table.shape[1]
    return torch.cat([c.table, torch.full((c.table.shape[0], more), 1 << 30, dtype=torch.int32, device="cuda")], dim=1)


def attend(c, table=None, **kw):
    kw = {"max_new": max(c.new), "max_length": max(c.length), **kw}
    return paged.attention(c.q, c.k_cache, c.v_cache, c.table if table is None else table, c.cu, c.lengths, **kw)


def launches(call):
    before = _native.lib().b200i_launch_count()
    call()
    return _native.lib().b200i_launch_count() - before


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("heads,kv,hd,new", [(8, 2, 64, 150), (5, 5, 40, 530), (2, 1, 128, 300)])
def test_a_table_with_room_to_grow(page, heads, kv, hd, new):
    """The same words, by the same kernels."""
    c = Case4([new, 1, new], [700, 40, 0], heads, kv, hd, page, BF16, seed=hd)
    want = attend(c)
    check(want, c.attention(), BF16, c.most())
    made = launches(lambda: attend(c))
    assert made == 1 + launches(lambda: attend(c, max_new=512 // (heads // kv)))  # unpacking, and what follows it anyway
    with pytest.raises(_native.NativeError, match="max_new"):
        torch_ops.check_status()  # (of the call for the launches of fewer rows)
    for positions in (2048, 4096, 8192):
        table = widened(c, positions)
        assert torch.equal(attend(c, table), want) and launches(lambda: attend(c, table)) == made
    torch_ops.check_status()


def test_a_table_too_wide_for_words_takes_no_room_for_them():
    c = Case4([300], [2000], 8, 2, 128, 64, BF16, spare=0)
    want = attend(c)
    table = widened(c, 1 << 19)

    def peak(table):
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        out = attend(c, table)
        return out, torch.cuda.max_memory_allocated() - before

    got, most = peak(table)
    assert torch.equal(got, want)
    words = 2304 * 2 * 128 * 4  # of the narrow table's 36 pages
    assert peak(c.table)[1] - most >= words - (1 << 20)  # (the allocator gives a block away whole where less than 1 MB of it would be left, so either peak may be up to that much more)


@pytest.mark.parametrize("bound", [1, 64, 700, 1 << 20])
@pytest.mark.parametrize("window", [0, 90])
def test_bounds_on_lengths_only_cut_the_work(bound, window):
    c = Case4([260, 1, 3], [4000, 10, 700], 4, 2, 128, 64, BF16)
    got = attend(c, max_length=bound, window=window)
    check(got, c.attention(window), BF16, c.most())
    assert torch.equal(attend(c, widened(c, 8192), max_length=bound, window=window), got)
    torch_ops.check_status()


def test_without_room_for_words_the_codes_are_read():
    """Through the C entry point: with the room asked for without a table, with that and what is too little for words, and with less than either."""
    c = Case4([300], [900], 8, 2, 128, 64, BF16)
    want, ptr, lib = attend(c), (lambda t: ctypes.c_void_p(t.data_ptr())), _native.lib()
    shape = 1, 2, 300, 1, 8, 2, 128, 300, 1200, 0
    full, least = (int(lib.b200i_paged_attention_table_workspace_bytes(0, *shape, positions)) for positions in (c.table.shape[1] * 64, 0))
    assert full > least > 0
    q, made = c.q.contiguous(), []
    for room in (full, full - 16, least, least - 16):
        out, ws = torch.zeros_like(q), torch.empty(room, dtype=torch.uint8, device="cuda")
        call = lambda: _native.call("b200i_paged_attention", 0, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream), ptr(out), ptr(q), 1024, ptr(c.k_cache), ptr(c.v_cache), 1, 2,  # noqa: E731
                                    ptr(c.table), ptr(c.cu), ptr(c.lengths), 300, 1, 8, 2, 128, c.pages, 64, c.table.shape[1], 300, 1200, 128 ** -0.5, 0, 0.0, ptr(ws), room)
        if room < least:
            with pytest.raises(_native.NativeError, match="workspace"):
                call()
            continue
        made.append(launches(call))
        assert torch.equal(out, want)
    assert made[0] == made[1] + 1 == made[2] + 1
    torch_ops.check_status()
