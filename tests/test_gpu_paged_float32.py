"""Attention of float32 rows, held to what its arithmetic leaves, row by row and word by word: that no piece of a word and no product of pieces is
missing in a few rows or columns.

Scores of normal inputs have a deviation of one. A score of many rows is a sum of 24 (bfloat16 cache) or 48 matrix products of pieces in the
tensor pipe, which cuts off up to 2^-23 of it each time, half of that on average: 48 * 2^-24 = 2.9e-6 of its size. Across the keys of a row
that is a deviation of 2.9e-6 of the weights and so of the output; pieces left out (2^-24 of a product), exponentials (2^-22) and sums add a
tenth to it. A row's error is held to twice that in its norm, 6.5e-6. A word's is four deviations of it at most, of values
whose largest is three of theirs or more: 8.5e-6 of the largest. Few rows (fused multiply-adds in 32 bits) are below that. A second piece of a
weight or a word that is left out is 2^-9 of it, a third 2^-17: 7.6e-6 in every word."""
import pytest
import torch

from paged_ref import BF16, F32, Case

pytestmark = pytest.mark.gpu
if torch.cuda.is_available():
    from mojolearn_b200 import paged, torch_ops


@pytest.mark.parametrize("cache", [F32, BF16])
@pytest.mark.parametrize("heads,kv,hd", [(12, 12, 64), (16, 2, 128), (5, 1, 80), (4, 4, 8)])
@pytest.mark.parametrize("new,past", [([1, 1, 1], [0, 300, 2000]), ([2, 3, 1], [500, 17, 90]), ([129, 1, 70], [0, 1000, 333]), ([300, 64], [128, 0]), ([1], [9000])])
def test_every_row_is_exact_to_its_arithmetic(cache, heads, kv, hd, new, past):
    c = Case(new, past, heads, kv, hd, 32, F32, cache, seed=heads + len(new))
    got, want = paged.attention(c.q, c.k_cache, c.v_cache, *c.args(), max_new=max(new)).double(), c.attention()
    torch_ops.check_status()
    off = got - want
    assert float(off.abs().max()) <= 8.5e-6 * c.most()
    assert float((off.norm(dim=-1) / want.norm(dim=-1)).max()) <= 6.5e-6
