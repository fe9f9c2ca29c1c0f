"""Attention over values near the largest of their type, all of one sign: the sums ahead of the division stay finite where those of weights up to one do."""
import numpy as np
import pytest
import torch

from cache_util import DEV, batch_of, filled_cache, largest, reference, tolerance

pytestmark = pytest.mark.gpu


# one row, a few, a chunk whose tiles several CTAs share, and one whose tiles are whole; f32
@pytest.mark.parametrize("specs,wide,dtype", [([(2000, 1)], False, torch.bfloat16), ([(2000, 4)], False, torch.bfloat16),
                                              ([(2000, 300)], True, torch.bfloat16), ([(100, 100)] * 80, True, torch.bfloat16),
                                              ([(2000, 20)], False, torch.float32)])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("quantized", [True, False])
def test_sums_stay_finite(specs, wide, dtype, dim, quantized):
    """Scores all alike, so that every weight is one; the sum of 2000 values of up to 2^115 is below 2^126."""
    batch, pages = batch_of(specs, 16, **(dict(width=4096, hints=False) if wide else {}))
    cache = filled_cache(pages, 16, 2, dim, quantized, v_std=2.0 ** 112)
    if quantized:
        cache.v |= 0x88  # levels of 0.08 and above
    else:
        cache.v.abs_().clamp_(max=2.0 ** 115)
    g = torch.Generator(device=DEV).manual_seed(3)
    q = torch.randn(batch.rows, 8, dim, device=DEV, generator=g).to(dtype)
    out = cache.attention(q, batch, 0.0)
    assert torch.isfinite(out).all()
    ref, spread, reach = reference(cache, batch, q, 0.0)
    off = np.abs(out.cpu().double().numpy() - ref)
    assert (off <= tolerance(ref, spread, reach, dim, specs[0][0], dtype == torch.float32, largest(cache))).all()
