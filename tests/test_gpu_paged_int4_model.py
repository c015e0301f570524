"""`PagedLM` and `PagedCache` on a cache in 4 bits."""
import numpy as np
import pytest
import torch

from paged_int4_ref import values
from test_gpu_paged_serving import model

pytestmark = pytest.mark.gpu
if torch.cuda.is_available():
    from mojolearn_b200 import paged, torch_ops
    from mojolearn_b200.models import PagedLM


def test_a_pool_in_4_bits():
    cache = paged.PagedCache(8, 2, 72, page=16, layers=2, dtype="int4")
    assert cache.dtype == "int4" and len(cache.k) == 2 and cache.k[0].shape == (8, 2, 16, 54) and cache.k[0].dtype == torch.uint8
    assert paged.row_bytes(72) == 54 and paged.row_bytes(128) == 72 and paged.row_bytes(8) == 18
    a = cache.open()
    tables = cache.extend([a], [17])
    k, v = paged.read(cache.k[0], cache.v[0], *tables, rows=17, head_dim=72)
    assert not bool(k.any()) and not bool(v.any()), "an empty cache holds zeros"


def test_one_layer_fed_in_pieces_and_at_once():
    """What a layer writes follows from its input alone, whose bits no product or norm before it changes with the other rows of a call: the same codes
    however the tokens are fed, and logits to the rounding of 32-bit sums."""
    lm = model(layers=1)
    served = PagedLM(lm, 60, page=16, cache="int4")
    ids = np.random.default_rng(1).integers(0, 256, 150).astype(np.int32)
    a, b = served.open(), served.open()
    whole = served.feed([a], [ids])
    for at in list(range(0, 40)) + list(range(40, 150, 11)):
        piece = served.feed([b], [ids[at:at + 1] if at < 40 else ids[at:at + 11]])
    assert float((whole - piece).norm() / whole.norm()) <= 2e-5
    held = []
    for s in (a, b):
        pages = torch.tensor(served.cache.held[s], device="cuda")
        held.append([values(x[0][pages], 32).transpose(0, 1).flatten(1, 2)[:, :150] for x in (served.cache.k, served.cache.v)])
    assert torch.equal(held[0][0], held[1][0]) and torch.equal(held[0][1], held[1][1]) and bool(held[0][0].any())
    lm.check_status()


def test_the_first_row_of_a_layer_is_its_value():
    """A sequence's first token attends to itself alone: its output is the value as it is held, and that is within half a step of it. So logits of a first
    token on a cache in 4 bits are those of one on float32 to what half a step makes of them."""
    lm = model(layers=1)
    rows = []
    for cache in ("float32", "bfloat16", "int4"):
        served = PagedLM(lm, 8, page=16, cache=cache)
        rows.append(served.feed([served.open()], [[7]])[0])
        got = served.cache
        k, v = paged.read(got.k[0], got.v[0], *got.extend([0], [0])[:1], torch.tensor([0, 1], dtype=torch.int32, device="cuda"), torch.tensor([1], dtype=torch.int32, device="cuda"),
                          rows=1, head_dim=32, dtype=torch.float32)
        if cache == "float32":
            want = k, v
        else:
            # half a step of a scale that is up to 17 / 16 of a seventh of the group's largest word; of bfloat16 half of 2^-7
            share = 2.0 ** -8 if cache == "bfloat16" else 0.5 / 7 * 17 / 16
            for x, y in zip((k, v), want):
                assert float((x - y).abs().max()) <= share * float(y.abs().max()) * (1 + 1e-6)
    assert bool(torch.isfinite(rows[2]).all())
    torch_ops.check_status()


def test_greedy_continuations_do_not_depend_on_who_is_served_beside():
    """One layer: the codes that a sequence writes are its own, so a continuation is the same alone and beside others, but for ties of logits within their rounding."""
    lm = model(layers=1)
    served = PagedLM(lm, 120, page=16, cache="int4")
    r = np.random.default_rng(2)
    prompts = [r.integers(0, 256, n).astype(np.int32) for n in (40, 1, 130)]
    together = served.generate(prompts, 8, chunk=32)
    assert [len(x) for x in together] == [48, 9, 138] and len(served.cache.free) == 120
    for p, x in zip(prompts, together):
        alone = served.generate([p], 8, chunk=64)[0]
        assert np.array_equal(alone, x)
