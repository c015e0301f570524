"""The paged cache's refusals that need no device."""
import ctypes

import pytest
import torch

from mojolearn_b200 import _native, paged


def test_host_tensors_are_refused():
    q = torch.zeros(2, 4, 64)
    k = torch.zeros(3, 2, 16, 64)
    i = torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(TypeError):
        paged.attention(q, k, k, i, torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    with pytest.raises(TypeError):
        paged.append(q, q[:, :2], q[:, :2], k, k, i, torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    with pytest.raises(TypeError):
        paged.attention(q.half(), k, k, i, None, None)


GOOD = {"row_type": 0, "cache_type": 1, "rows": 2, "batch": 1, "n_heads": 4, "n_kv": 2, "head_dim": 64, "pages": 3, "page": 16, "max_pages": 2}
BAD = [({"rows": 0}, b"positive"), ({"batch": -1}, b"positive"), ({"n_heads": 5}, b"multiple"), ({"head_dim": 132}, b"head_dim"), ({"head_dim": 12}, b"head_dim"),
       ({"page": 8}, b"page"), ({"page": 48}, b"page"), ({"row_type": 1, "cache_type": 0}, b"float32"), ({"row_type": 2}, b"float32"), ({"pages": 1 << 28}, b"2^31"),
       ({"rows": 1 << 31}, b"31 bits"), ({"max_pages": 1 << 28}, b"31 bits")]


@pytest.mark.parametrize("change,message", BAD)
def test_c_abi_refusals_come_before_the_device(change, message):
    a = dict(GOOD, **change)
    buf = ctypes.create_string_buffer(256)
    one = ctypes.c_void_p(1 << 20)  # never read: the extents are refused first
    lib = _native.lib()
    tail = [a[n] for n in ("rows", "batch", "n_heads", "n_kv", "head_dim", "pages", "page", "max_pages")]
    err = [ctypes.cast(buf, ctypes.c_void_p), 256]
    assert lib.b200i_paged_attention(-1, None, one, one, 256, one, one, a["row_type"], a["cache_type"], one, one, one, *tail, 2, 32, 0.1, 0, 0.0, None, 0, *err) == 1
    assert message in buf.value and buf.value.startswith(b"paged_attention")
    assert lib.b200i_paged_append(-1, None, one, one, one, one, one, one, 256, 128, 128, a["row_type"], a["cache_type"], None, None, 0, 0, None, None, 1e-6, 0, one, one, one,
                                  *tail, *err) == 1
    assert message in buf.value and buf.value.startswith(b"paged_append")
