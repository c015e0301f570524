"""Whose rows `paged.read` gives: many sequences in a block's rows, most of them without rows, offsets that leave rows to nobody, and rows behind the last sequence."""
import ctypes
import random

import pytest
import torch

from paged_ref import BF16

pytestmark = pytest.mark.gpu
if torch.cuda.is_available():
    from mojolearn_b200 import _native, torch_ops


def held(cu, lengths, rows, capacity):
    """Of each row the first sequence that ends behind it, where that began before it and its tables hold it, and its position there."""
    out = []
    for t in range(rows):
        b = next((b for b in range(len(lengths)) if t < cu[b + 1]), None)
        if b is None or t < cu[b] or not 0 <= cu[b] <= cu[b + 1] <= rows or lengths[b] > capacity:
            out.append(None)
        else:
            out.append((b, lengths[b] - cu[b + 1] + t))
    return out


def offsets(kind, batch, seed):
    r = random.Random(seed)
    new = [r.choice([0, 0, 0, 1, 1, 5, 40]) if kind != "sparse" else int(r.random() < 0.01) for _ in range(batch)]
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    if kind == "begins late":
        cu = [x + 7 for x in cu]
    if kind == "any":  # what no caller means: whatever it says, a row has at most one sequence
        for _ in range(1 + batch // 8):
            cu[r.randrange(batch + 1)] = r.randint(-3, cu[-1] + 3)
    return cu


@pytest.mark.parametrize("kind", ["ragged", "sparse", "begins late", "any"])
@pytest.mark.parametrize("batch", [1, 31, 32, 33, 700])
@pytest.mark.parametrize("pad", [0, 1, 45, 20000])
def test_rows_and_their_sequences(kind, batch, pad):
    page, kv, hd, capacity = 16, 2, 8, 48
    cu = offsets(kind, batch, batch + pad)
    rows = max(cu) + pad
    if rows < 1:
        rows = 1
    lengths = [max(0, min(capacity, cu[b + 1] - cu[b])) for b in range(batch)]
    g = torch.Generator(device="cuda").manual_seed(batch)
    cache = [torch.randn(batch * 3, kv, page, hd, generator=g, device="cuda").to(BF16) for _ in range(2)]
    table = torch.randperm(batch * 3, generator=g, device="cuda").to(torch.int32).view(batch, 3)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    got, cu_there, lengths_there = [torch.full((rows, kv, hd), 7.0, device="cuda") for _ in range(2)], ints(cu), ints(lengths)
    _native.call("b200i_paged_read", 0, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream), *[ctypes.c_void_p(x.data_ptr()) for x in got + cache], 0, 1,
                 *[ctypes.c_void_p(x.data_ptr()) for x in (table, cu_there, lengths_there)], rows, batch, kv, hd, batch * 3, page, 3)
    if kind != "any":
        torch_ops.check_status()
    else:
        try:
            torch_ops.check_status()
        except _native.NativeError:
            pass
    where = held(cu, lengths, rows, capacity)
    at = [t for t, x in enumerate(where) if x is not None]
    assert at or kind in ("sparse", "any") or max(cu) == min(cu)
    nobody = torch.ones(rows, dtype=torch.bool, device="cuda")
    nobody[at] = False
    assert all(bool((have[nobody] == 7.0).all()) for have in got)
    if not at:
        return
    seq, pos = (torch.tensor([where[t][i] for t in at], device="cuda") for i in (0, 1))
    for have, x in zip(got, cache):
        want = x[table[seq, pos.clamp(min=0) // page].long(), :, pos.clamp(min=0) % page].float()
        assert torch.equal(have[at], torch.where(pos[:, None, None] < 0, 0.0, want))
