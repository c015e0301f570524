"""Arguments of the paged cache's C entry points that are refused before anything reaches the device."""
import ctypes

import pytest

from mojolearn_b200 import _native

PLACE = ctypes.c_void_p(1 << 20)  # never read: the calls are refused first


def attend(out=ctypes.c_void_p(1 << 22), q=PLACE, ldq=256, rows=2, ws=None, ws_bytes=0, window=0, softcap=0.0, scale=0.1):
    buf = ctypes.create_string_buffer(256)
    status = _native.lib().b200i_paged_attention(-1, None, out, q, ldq, PLACE, PLACE, 0, 1, PLACE, PLACE, PLACE, rows, 1, 4, 2, 64, 3, 16, 2, 2, 32, scale, window, softcap, ws, ws_bytes,
                                                 ctypes.cast(buf, ctypes.c_void_p), 256)
    return status, buf.value


@pytest.mark.parametrize("off", [1, 2, 4, 8, 12])
def test_a_workspace_between_16_byte_boundaries(off):
    status, message = attend(ws=ctypes.c_void_p((1 << 21) + off), ws_bytes=1 << 20)
    assert status == 1 and b"workspace" in message and b"16-byte" in message


@pytest.mark.parametrize("out,q,ldq,rows", [(0, 0, 256, 2), (1024, 0, 256, 2), (2032, 0, 256, 2), (0, 2032, 256, 2), (2048, 4096, 1024, 3), (4096, 0, 1024, 3)])
def test_an_output_over_the_queries(out, q, ldq, rows):
    """A row that does not come out finite is done again from its query, so that has to be there still."""
    status, message = attend(out=ctypes.c_void_p((1 << 20) + out), q=ctypes.c_void_p((1 << 20) + q), ldq=ldq, rows=rows)
    assert status == 1 and b"output" in message and b"queries" in message


@pytest.mark.parametrize("out,q,ldq,rows", [(2048, 0, 256, 2), (0, 2048, 256, 2), (1024, 0, 2048, 2), (5120, 4096, 1024, 3)])
def test_an_output_beside_the_queries(out, q, ldq, rows):
    """Column blocks of one matrix, and rows one after another: whatever refuses this call, it is not that."""
    assert b"queries" not in attend(out=ctypes.c_void_p((1 << 20) + out), q=ctypes.c_void_p((1 << 20) + q), ldq=ldq, rows=rows, ws=PLACE, ws_bytes=8)[1]


def append(out, q=1 << 20, k=1 << 21, v=1 << 22, ldq=256):
    buf = ctypes.create_string_buffer(256)
    p = ctypes.c_void_p
    # norm kind 7 is refused, before the device and after the places
    status = _native.lib().b200i_paged_append(-1, None, p(out), PLACE, PLACE, p(q), p(k), p(v), ldq, 128, 128, 0, 1, None, None, 0, 0, None, None, 1e-6, 7, PLACE, PLACE, PLACE, 2, 1, 4, 2, 64,
                                              3, 16, 2, ctypes.cast(buf, ctypes.c_void_p), 256)
    assert status == 1
    return buf.value


@pytest.mark.parametrize("out,ldq", [((1 << 20) + 1024, 256), ((1 << 20) - 16, 256), (1 << 20, 512), (1 << 21, 256), ((1 << 22) + 512, 256)])
def test_rotated_queries_over_rows_that_are_read(out, ldq):
    assert b"output" in append(out, ldq=ldq)


def test_rotated_queries_beside_the_rows_or_in_their_place():
    for out in (1 << 23, 1 << 20, (1 << 20) + 2048, (1 << 21) + 1024):
        assert b"norm kind" in append(out)


def workspace(rows, batch, max_new, max_length, row_type=1, heads=32, kv=8):
    return _native.lib().b200i_paged_attention_workspace_bytes(-1, row_type, 1, rows, batch, heads, kv, 128, max_new, max_length, 0)


@pytest.mark.parametrize("row_type,block", [(0, 2 * 128 * 130 * 4 + 32), (1, 2 * 256 * 130 * 4 + 32)])
def test_a_short_call_has_a_short_workspace(row_type, block):
    """Parts of as many blocks as the call can have steps: 17 tokens over 300 keys, 8 key heads, tiles of 64 or 128 keys."""
    tiles = -(-300 // (128 if row_type else 64)) + 1
    assert workspace(17, 1, 17, 300, row_type) == min(148, 8 * tiles) * block
    assert workspace(5, 1, 5, 1, row_type) == 8 * 2 * block
    for call in ((2048, 1, 2048, 16384), (4096, 4, 1024, 1024), (17, 1, 17, 1 << 31), (1 << 30, 1, 1 << 30, 1 << 62), (40, 30, 17, 100)):
        assert workspace(*call, row_type) == 148 * block
