"""Weights of up to 24 bfloat16 rows over a cache in 4 bits: how far an output is off does not change with the number of rows."""
import pytest
import torch

from paged_int4_ref import Case4, packed, parts
from paged_ref import BF16

pytestmark = pytest.mark.gpu
if torch.cuda.is_available():
    from mojolearn_b200 import paged, torch_ops


@pytest.mark.parametrize("new,group", [(1, 1), (4, 1), (1, 7), (2, 7), (2, 8), (17, 1), (3, 7), (5, 4), (3, 8), (24, 1)])
@pytest.mark.parametrize("hd", [32, 64, 96, 128])
@pytest.mark.parametrize("past", [6, 3000])
def test_a_weight_has_two_pieces(new, group, hd, past):
    """An output is off by its own rounding, 2^-8 of itself, and by what is left of the weights, of the sum of weight times |value|: 2^-16 where a weight is held
    as two pieces of 8 bits. A score (eight sums of 16 products, cut at 2^-23 of up to 50, times 0.18 at most) and its power of two are off by less than 2^-16, as is
    the weights' sum by both: 2^-14 in all. With one piece it is up to 2^-8, which shows where an output is small beside its terms."""
    c = Case4([new, new], [past, 5], 2 * group, 2, hd, 32, BF16, seed=hd + new)
    got = paged.attention(c.q, c.k_cache, c.v_cache, *c.args(), max_new=new)
    torch_ops.check_status()
    want = c.attention()
    codes, scale = parts(c.v_cache)
    c.v_cache = packed(8 + (codes - 8).abs(), scale)  # (codes are from 1 to 15)
    terms = c.attention()
    assert bool(((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -14 * terms).all())
