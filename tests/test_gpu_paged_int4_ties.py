"""Values and keys in 4 bits that lie exactly between two codes, or one 24-bit step beside it, as float32 rows that hold words of few bits do."""
import pytest
import torch

from paged_int4_ref import Case4
from test_gpu_paged_int4 import written

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
