"""More than 512 bfloat16 rows of a sequence and key head over a cache in 4 bits: the words are made once, in the workspace, and attended to there."""
import ctypes

import pytest
import torch

from paged_int4_ref import Case4, packed, parts
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


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("room", [0, 8192])
def test_a_page_outside_the_pool_is_reported(page, room):
    """It counts as a page of zeros, as one of scale zero does."""
    c = Case4([150, 1], [800, 90], 8, 2, 64, page, BF16)
    zeros = []
    for cache in (c.k_cache, c.v_cache):
        codes, scale = parts(cache)
        scale[int(c.table[0, 2])] = 0.0
        zeros.append(packed(codes, scale))
    c.k_cache, c.v_cache = zeros
    table = widened(c, room) if room else c.table.clone()
    want = attend(c, table)
    check(want, c.attention(), BF16, c.most())
    torch_ops.check_status()
    for wrong in (c.pages, -1, 1 << 30):
        table[0, 2] = wrong
        got = attend(c, table)
        with pytest.raises(_native.NativeError, match="outside the pool"):
            torch_ops.check_status()
        assert torch.equal(got, want)


@pytest.mark.parametrize("window", [0, 70])
@pytest.mark.parametrize("page", [16, 256])
def test_what_is_not_seen_has_no_influence(page, window):
    """NaN past the lengths, in pages of nobody, before a window, and in the memory that the workspace takes; page numbers of pages that no row sees mean nothing."""
    c = Case4([150, 0, 2], [500, 40, 33], 8, 2, 64, page, BF16, pad=3)
    out = torch.full_like(c.q.contiguous(), 7.0)
    want = attend(c, window=window, out=out)[:c.first[-1]].clone()
    assert bool((out[c.first[-1]:] == 7.0).all())
    check(want, c.attention(window)[:c.first[-1]], BF16, c.most())
    seen = torch.zeros(c.pages, page, dtype=torch.bool, device="cuda")
    for b, n in enumerate(c.length):
        for pos in range(max(0, n - c.new[b] + 1 - window) if window else 0, n if c.new[b] else 0):
            seen[int(c.table[b, pos // page]), pos % page] = True
    for name in ("k_cache", "v_cache"):
        codes, scale = parts(getattr(c, name))
        setattr(c, name, packed(torch.where(seen[:, None, :, None, None], codes, 15), torch.where(seen[:, None, :, None], scale, float("nan"))))
    table = widened(c, 4096)
    for b, n in enumerate(c.length):
        table[b, :max(0, n - c.new[b] + 1 - window) // page if window else 0] = -5
        if not c.new[b]:
            table[b] = -5
    for byte in (0xFF, 0x7F, 0x80):
        full = torch.full((64 << 20,), byte, dtype=torch.uint8, device="cuda")
        del full  # what the call's workspace is cut from
        assert torch.equal(attend(c, table, window=window)[:c.first[-1]], want)
    torch_ops.check_status()


@pytest.mark.parametrize("room", [0, 4096])
def test_on_another_stream_and_in_a_graph(room):
    """Captured twice and replayed in turn with other rows, lengths and pages, each graph with a workspace of its own."""
    c = Case4([140, 140], [100, 400], 8, 2, 64, 64, BF16, spare=6)
    table = torch.cat([c.table, torch.full((2, 1), -1, dtype=torch.int32, device="cuda")], dim=1) if not room else widened(c, room)
    free = sorted(set(range(c.pages)) - set(c.table.flatten().tolist()))
    for b in range(2):
        table[b, -(-c.length[b] // 64)] = free[b]
    q, lengths, side = c.q.clone(), c.lengths.clone(), torch.cuda.Stream()

    def step():
        return paged.attention(q, c.k_cache, c.v_cache, table, c.cu, lengths, max_new=140, max_length=620)

    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        side.synchronize()
        graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
        for graph in graphs:
            with torch.cuda.graph(graph, stream=side):
                outs.append(step())
        g = torch.Generator(device="cuda").manual_seed(5)
        for i in range(4):
            q.copy_(torch.randn(q.shape, generator=g, device="cuda"))
            lengths.copy_(c.lengths + 3 * i)
            order = torch.randperm(c.pages, generator=g, device="cuda").to(torch.int32)
            table[:, :10] = torch.where(table[:, :10] >= 0, order[table[:, :10].clamp(0, c.pages - 1)], table[:, :10])
            graphs[0].replay(), graphs[1].replay()
            got = [x.clone() for x in outs]
            want = step()
            assert torch.equal(got[0], want) and torch.equal(got[1], want)
            c.table, c.length = table, lengths.tolist()
            check(want, c.attention(q=q), BF16, c.most())
    side.synchronize()
    torch_ops.check_status()
