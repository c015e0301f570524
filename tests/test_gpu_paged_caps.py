"""Capped scores and scales far from one, on every kernel of the paged attention."""
import pytest
import torch

from paged_ref import BF16, F32, TYPES, Case, check

pytestmark = pytest.mark.gpu
if torch.cuda.is_available():
    from mojolearn_b200 import paged


def held(c, **kw):
    got = paged.attention(c.q, c.k_cache, c.v_cache, *c.args(), max_new=max(c.new), **kw)
    check(got, c.attention(softcap=kw["softcap"], scale=kw.get("scale")), c.rows, c.most())
    return got


@pytest.mark.parametrize("rows,cache", TYPES)
@pytest.mark.parametrize("new", [1, 3, 90, 300])
@pytest.mark.parametrize("cap", [60.0, 255.0, 257.0, 1e3, 1e5, 1e8, 1e30])
def test_caps_far_above_the_scores(rows, cache, new, cap):
    """A score that is small beside its cap is almost as it was."""
    held(Case([new] * 3, [0, 65, 400], 8, 2, 128, 32, rows, cache, seed=new), softcap=cap)


@pytest.mark.parametrize("rows,cache", TYPES)
@pytest.mark.parametrize("new", [1, 90])
@pytest.mark.parametrize("cap", [3.0, 1e3, 1e8])
@pytest.mark.parametrize("size", [2.0 ** -66, 2.0 ** -20, 2.0 ** 20, 2.0 ** 50])
def test_caps_with_keys_of_any_size(rows, cache, new, cap, size):
    c = Case([new] * 3, [0, 65, 400], 8, 2, 64, 32, rows, cache)
    c.k_cache.mul_(size)
    held(c, softcap=cap, scale=0.25 / size)


@pytest.mark.parametrize("rows,cache", TYPES)
@pytest.mark.parametrize("new", [1, 90])
@pytest.mark.parametrize("part", [0.35, 1.0])
def test_scores_about_where_the_formula_changes(rows, cache, new, part):
    """Scores 65536 part + e of a cap of 65536, e about one: exact products, whose caps have to keep their order and their differences. A score of
    that size is held to 2^-7 in 32 bits, and the cap's own arithmetic adds a few of them: weights within 2^-5 (a slope of tanh below 0.9)."""
    c = Case([new] * 2, [0, 300], 4, 2, 64, 32, rows, cache)
    near = torch.tensor(65536.0 * part).to(BF16)
    c.q.zero_()
    c.q[:, :, 0] = 1.0
    c.q[:, :, 1] = 1.0
    c.k_cache[..., 0] = near.to(c.k_cache.dtype)
    c.k_cache[..., 1] = c.k_cache[..., 1].to(BF16).to(c.k_cache.dtype)
    got = paged.attention(c.q, c.k_cache, c.v_cache, *c.args(), max_new=new, softcap=65536.0, scale=1.0)
    off = (got.double() - c.attention(softcap=65536.0, scale=1.0)).abs().max()
    assert float(off) <= (2.0 ** -5 + 2.0 ** -7) * c.most()


@pytest.mark.parametrize("rows,cache", TYPES)
@pytest.mark.parametrize("new", [1, 3, 90])
@pytest.mark.parametrize("cap,scale", [(1e-20, 1e20), (1e-25, 1.0), (1e-40, 1.0), (1e-300, 0.125)])
def test_caps_next_to_nothing(rows, cache, new, cap, scale):
    """Scores capped to next to nothing weigh all keys alike, whatever the scale; a product of zero among them too."""
    c = Case([new] * 2, [0, 300], 4, 2, 64, 32, rows, cache)
    for b in range(2):
        c.k_cache[int(c.table[b, 0]), :, 0] = 0.0
    held(c, softcap=cap, scale=scale)


@pytest.mark.parametrize("rows,cache", TYPES)
@pytest.mark.parametrize("new", [1, 3, 90])
def test_a_scale_and_a_cap_whose_quotient_leaves_32_bits(rows, cache, new):
    c = Case([new] * 2, [0, 300], 4, 2, 64, 32, rows, cache)
    c.k_cache.mul_(2.0 ** 50)
    held(c, softcap=1e30, scale=2.0 ** -52)
