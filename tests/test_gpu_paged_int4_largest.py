"""The largest words that a cache in 4 bits holds, 7 times 2^90, where weights exceed one: sums that leave 32 bits on the way do not reach the answer."""
import pytest
import torch

from paged_int4_ref import Case4, packed, quantised, values
from paged_ref import BF16, F32, check

pytestmark = pytest.mark.gpu
if torch.cuda.is_available():
    from mojolearn_b200 import paged, torch_ops


@pytest.mark.parametrize("rows", [F32, BF16])
@pytest.mark.parametrize("new", [1, 3, 20, 90, 300])
@pytest.mark.parametrize("rise", [7.5, 60.0, 95.0, 120.0])
def test_values_of_the_largest_size_under_rising_scores(rows, new, rise):
    """Every 256 keys scores are `rise` powers of two larger than before: where weights are taken from the scores so far, a sum is up to 2^(90 + 3 + rise + 8)."""
    c = Case4([new, 1], [1000, 200], 4, 2, 64, 32, rows, seed=new)
    c.q = torch.full_like(c.q, 1.0)
    k = torch.zeros_like(values(c.k_cache, 64))
    for b, n in enumerate(c.length):
        for first in range(0, n, 32):
            k[int(c.table[b, first // 32])] = rise * 0.6931471805599453 / 8.0 * (first // 256)  # scores are 8 times a key's word
    v = values(c.v_cache, 64)
    v = v / v.abs().amax() * 7 * 2.0 ** 90
    c.k_cache, c.v_cache = packed(*quantised(k)), packed(*quantised(v))
    got = paged.attention(c.q, c.k_cache, c.v_cache, *c.args(), max_new=new)
    torch_ops.check_status()
    check(got, c.attention(), rows, c.most())
