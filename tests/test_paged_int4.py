"""The paged cache in 4 bits without a device: refusals of the C entry points and of the Python calls, the definition's own words, and the workspace."""
import ctypes

import pytest
import torch

from mojolearn_b200 import _native, paged
from paged_int4_ref import packed, parts, quantised, values

PLACE = [ctypes.c_void_p(1 << (20 + i)) for i in range(6)]  # never read: the calls are refused first
GOOD = {"out_type": 1, "cache_type": 2, "rows": 2, "batch": 1, "n_kv": 2, "head_dim": 64, "pages": 3, "page": 16, "max_pages": 2}
BAD = [({"rows": 0}, b"positive"), ({"batch": -1}, b"positive"), ({"head_dim": 132}, b"head_dim"), ({"head_dim": 12}, b"head_dim"), ({"page": 8}, b"page"), ({"page": 48}, b"page"),
       ({"cache_type": 3}, b"4 bits"), ({"out_type": 2}, b"4 bits"), ({"out_type": 1, "cache_type": 0}, b"float32"), ({"pages": 1 << 28}, b"2^31"), ({"rows": 1 << 31}, b"31 bits")]


def read(a, k=PLACE[0], v=PLACE[1], k_cache=PLACE[2], v_cache=PLACE[3]):
    buf = ctypes.create_string_buffer(256)
    status = _native.lib().b200i_paged_read(-1, None, k, v, k_cache, v_cache, a["out_type"], a["cache_type"], PLACE[4], PLACE[4], PLACE[4],
                                            *[a[n] for n in ("rows", "batch", "n_kv", "head_dim", "pages", "page", "max_pages")], ctypes.cast(buf, ctypes.c_void_p), 256)
    return status, buf.value


@pytest.mark.parametrize("change,message", BAD)
def test_extents_and_types_that_are_refused(change, message):
    status, said = read(dict(GOOD, **change))
    assert status == 1 and said.startswith(b"paged_read") and message in said


@pytest.mark.parametrize("kw,message", [({"k": None}, b"null"), ({"v_cache": None}, b"null"), ({"k": ctypes.c_void_p((1 << 20) + 8)}, b"16-byte"), ({"k_cache": ctypes.c_void_p((1 << 22) + 4)}, b"16-byte"),
                                        ({"v": ctypes.c_void_p((1 << 20) + 496)}, b"over one another"), ({"k": ctypes.c_void_p((1 << 22) + 16)}, b"over one another"),
                                        ({"v": ctypes.c_void_p((1 << 23) + 3 * 2 * 16 * 36 - 16)}, b"over one another")])
def test_storage_that_is_refused(kw, message):
    status, said = read(GOOD, **kw)
    assert status == 1 and message in said


@pytest.mark.parametrize("cache_type", [-1, 3, 7])
def test_other_types_of_caches(cache_type):
    buf = ctypes.create_string_buffer(256)
    lib, one, err = _native.lib(), PLACE[0], [ctypes.cast(buf, ctypes.c_void_p), 256]
    tail = [2, 1, 4, 2, 64, 3, 16, 2]
    assert lib.b200i_paged_attention(-1, None, one, one, 256, one, one, 0, cache_type, one, one, one, *tail, 2, 32, 0.1, 0, 0.0, None, 0, *err) == 1 and b"4 bits" in buf.value
    assert lib.b200i_paged_append(-1, None, one, one, one, one, one, one, 256, 128, 128, 0, cache_type, None, None, 0, 0, None, None, 1e-6, 0, one, one, one, *tail, *err) == 1
    assert b"4 bits" in buf.value


def test_host_tensors_are_refused():
    k = torch.zeros(3, 2, 16, 36, dtype=torch.uint8)
    i = torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(TypeError):
        paged.read(k, k, i, torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), rows=1, head_dim=64)
    with pytest.raises(TypeError):
        paged.attention(torch.zeros(1, 4, 64), k, k, i, torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))


def test_the_definition():
    """A scale has five significant bits and is the smallest of them that seven times reach the largest word; the nearest code, ties to even; bytes there and back."""
    x = torch.randn(3, 2, 16, 72, dtype=torch.float64, generator=torch.Generator().manual_seed(1)) * torch.logspace(-8, 8, 16, dtype=torch.float64)[:, None]
    codes, scale = quantised(x)
    wide = torch.nn.functional.pad(x, (0, 24)).unflatten(-1, (3, 32))
    most = wide.abs().amax(-1)
    part = torch.frexp(scale)[0] * 32
    assert torch.equal(part, part.round()) and bool((7 * scale >= most).all())
    below = torch.ldexp((part - 1) / 32, torch.frexp(scale)[1])
    assert bool((7 * below < most).all())
    left = (wide - (codes - 8) * scale[..., None]).abs() / scale[..., None]
    assert bool((left <= 0.5).all()) and int(codes.min()) >= 1 and int(codes.max()) <= 15
    back = parts(packed(codes, scale))
    assert torch.equal(back[0], codes) and torch.equal(back[1], scale)
    held = values(packed(codes, scale), 72)
    assert torch.equal(held, held.to(torch.bfloat16).double())
    tie = torch.tensor([7.0, 0.5, 1.5, 2.5, -0.5, -1.5] + [0.0] * 26)
    assert quantised(tie)[0][0, :6].sub(8).tolist() == [7, 0, 2, 2, 0, -2]


@pytest.mark.parametrize("row_type,rows,laid,keys", [(0, 1, 2, 256), (0, 2, 2, 256), (0, 3, 8, 128), (0, 9, 16, 128), (0, 17, 24, 128), (1, 4, 4, 256), (1, 5, 8, 128), (1, 16, 16, 128), (1, 24, 24, 128)])
def test_the_workspace_of_a_few_rows(row_type, rows, laid, keys):
    """Two parts of as many rows as are laid out a block, and a block at most for every four tiles; none where a sequence's keys are not cut."""
    need = lambda length: _native.lib().b200i_paged_attention_workspace_bytes(-1, row_type, 2, rows, 1, 8, 8, 128, rows, length, 0)  # noqa: E731
    assert need(8 * 128) == 0
    blocks = min((1 if rows > 16 else 2) * 148, -(-8 * (5120 // keys) // 4))
    assert need(5120) == blocks * (2 * laid * 130 * 4 + 32)


def test_the_workspace_of_many_rows_has_room_for_words():
    """More than 512 bfloat16 rows a sequence and key head: pages of words for as many positions as are named, up to 256 MB of them; extents that overflow nothing."""
    need = lambda batch, new, length, row_type=1, cache=2: _native.lib().b200i_paged_attention_workspace_bytes(-1, row_type, cache, batch * new, batch, 8, 8, 128, new, length, 0)  # noqa: E731
    words = lambda batch, length: -(-length // 256) * 256 * batch * 8 * 128 * 4  # noqa: E731
    for batch, new, length in ((1, 513, 16384), (1, 2048, 1000), (4, 600, 8192)):
        more = need(batch, new, length) - need(batch, new, length, cache=1)
        assert words(batch, length) <= more <= words(batch, length) * 1.01 + 4096
    for call in ((1, 512, 16384), (1, 600, 16384, 0), (2, 600, 40000), (1 << 20, 1024, 1 << 30), (1 << 29, 1024, (1 << 31) - 1)):
        assert need(*call) == need(*call, *([1] if len(call) == 3 else []), cache=1)
