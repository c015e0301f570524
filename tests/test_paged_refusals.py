"""Arguments of the paged cache's C entry points that are refused before anything reaches the device."""
import ctypes

import pytest

from mojolearn_b200 import _native

PLACE = ctypes.c_void_p(1 << 20)  # never read: the calls are refused first


def attend(out=PLACE, q=PLACE, ldq=256, rows=2, ws=None, ws_bytes=0, window=0, softcap=0.0, scale=0.1):
    buf = ctypes.create_string_buffer(256)
    status = _native.lib().b200i_paged_attention(-1, None, out, q, ldq, PLACE, PLACE, 0, 1, PLACE, PLACE, PLACE, rows, 1, 4, 2, 64, 3, 16, 2, 2, 32, scale, window, softcap, ws, ws_bytes,
                                                 ctypes.cast(buf, ctypes.c_void_p), 256)
    return status, buf.value


@pytest.mark.parametrize("off", [1, 2, 4, 8, 12])
def test_a_workspace_between_16_byte_boundaries(off):
    status, message = attend(ws=ctypes.c_void_p((1 << 21) + off), ws_bytes=1 << 20)
    assert status == 1 and b"workspace" in message and b"16-byte" in message
