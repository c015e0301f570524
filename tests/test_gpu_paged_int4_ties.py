"""Words whose codes in 4 bits are easily missed: float32 words exactly between two codes or one 24-bit step beside it, norms whose squares leave 32 bits, a type's largest words."""
import pytest
import torch

from paged_int4_ref import Case4, parts
from paged_ref import rotated
from test_gpu_paged_int4 import ROWS, tables, written

pytestmark = pytest.mark.gpu
if torch.cuda.is_available():
    from mojolearn_b200 import paged, torch_ops


@pytest.mark.parametrize("hd", [40, 64, 72, 128])
@pytest.mark.parametrize("beside", [-1, 0, 1])
@pytest.mark.parametrize("top", [7.0, 7.3, 3.9])
def test_float32_words_at_and_beside_ties(hd, beside, top):
    """Every half between two codes for a scale of one to five bits, as it is, the next word above it and the next below."""
    c = Case4([28], [3], 2, 2, hd, 16, torch.float32, seed=hd)
    scale = torch.tensor([1.0, 17 / 16, 1.5, 31 / 16], device="cuda").repeat(7)[:, None, None]
    halves = (torch.arange(hd, device="cuda") % 14 - 6.5).float()[None, None]
    x = (halves * scale).expand(28, 2, hd).contiguous()
    if beside:
        x = torch.nextafter(x, torch.full_like(x, float("inf") if beside > 0 else float("-inf")))
    x[:, :, ::32] = (torch.tensor(top, device="cuda") * scale).expand(28, 2, hd)[:, :, ::32]  # what the scale follows
    before = c.k_cache.clone(), c.v_cache.clone()
    paged.append(torch.zeros_like(x), x, x, c.k_cache, c.v_cache, *c.args())
    torch_ops.check_status()
    for have, want in zip((c.k_cache, c.v_cache), written(c, x, x, before)):
        assert torch.equal(have, want)


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("half", [0, 3, 32])
@pytest.mark.parametrize("size,weight", [(2.0 ** 90, 1.0), (2.0 ** 63, 1.0), (2.0 ** -70, 1.0), (2.0 ** -100, 1.0), (2.0 ** 40, 2.0 ** -90), (2.0 ** -40, 2.0 ** 100)])
def test_norms_of_words_of_any_size(rows, half, size, weight):
    """Squares that leave 32 bits, and weights that bring words to the ends of the scales: the codes are those of 64 bits."""
    c = Case4([70], [9], 4, 2, 64, 16, rows, seed=5)
    k = c.k * size
    cos, sin = tables(96, half) if half else (None, None)
    w = (torch.rand(64, device="cuda") + 0.5) * weight
    before = c.k_cache.clone(), c.v_cache.clone()
    paged.append(c.q, k, c.v, c.k_cache, c.v_cache, *c.args(), cos, sin, q_norm=w, k_norm=w, eps=1e-45)
    pos = torch.arange(9, 79, device="cuda")
    for have, want in zip((c.k_cache, c.v_cache), written(c, rotated(k, pos, cos, sin, w, 1e-45), c.v, before)):
        assert torch.equal(have, want)


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("half", [0, 3, 32])
def test_the_largest_words_are_cut(rows, half):
    """The type's largest and lowest words are finite, and so is what a rotation makes of them in 64 bits: cut to 7 times the largest scale."""
    c = Case4([64], [0], 2, 2, 64, 16, rows, seed=6)
    big = torch.finfo(rows).max
    x = torch.where(torch.rand(64, 2, 64, device="cuda") < 0.5, -big, big).to(rows)
    x[:, 0, ::5] = 1.0
    cos, sin = tables(64, half) if half else (None, None)
    before = c.k_cache.clone(), c.v_cache.clone()
    paged.append(torch.zeros_like(x), x, x, c.k_cache, c.v_cache, *c.args(), cos, sin)
    for have, want in zip((c.k_cache, c.v_cache), written(c, rotated(x, torch.arange(64, device="cuda"), cos, sin), x, before)):
        assert torch.equal(have, want)
    assert bool(torch.isfinite(parts(c.k_cache)[1]).all()) and bool(torch.isfinite(parts(c.v_cache)[1]).all())
