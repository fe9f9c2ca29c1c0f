"""The attention kernel for many rows where every CTA has many row tiles, one after another, of few steps each: results are written out and the
next queries brought in over and over, by warps that are through at different times."""
import numpy as np
import pytest
import torch

from cache_util import DEV, batch_of, filled_cache, largest, reference, spoil_unused, tolerance
from unifur_b200 import _lib

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def short_prompts(count, most):
    """(tokens in the cache, the call's rows): a few to `most` rows, some with tokens ahead of them."""
    rng = np.random.default_rng(count)
    rows = rng.integers(3, most + 1, count)
    return [(int(n + a), int(n)) for n, a in zip(rows, rng.integers(0, 90, count) * (rng.random(count) < 0.5))]


# Row tiles are 256 rows (128 with a dim of 256) of a head: part of one to a sequence, or two and a bit, of which the last have idle warps.
@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("count,heads,group,dim,most", [(60, 16, 2, 64, 90), (40, 16, 2, 128, 90), (24, 16, 5, 128, 120), (40, 16, 3, 256, 40), (50, 8, 9, 64, 70)])
def test_every_run_gives_the_same(count, heads, group, dim, most, quantized):
    specs = short_prompts(count, most)
    batch, pages = batch_of(specs, 16, width=4096, hints=False, spare_rows=(1, 1))
    tiles = sum(-(-n * group // (128 if dim == 256 else 256)) for _, n in specs) * heads
    assert tiles > 3 * 148
    cache = filled_cache(pages, 16, heads, dim, quantized)
    spoil_unused(cache, batch)
    g = torch.Generator(device=DEV).manual_seed(7)
    q = torch.randn(batch.rows, heads * group, dim, device=DEV, generator=g).to(BF16)
    before = _lib.launch_count()
    first = torch.full_like(q, 7.0)
    cache.attention(q, batch, out=first)
    assert _lib.launch_count() - before >= 2  # the kernel for many rows and its join
    ref, spread, reach = reference(cache, batch, q, dim ** -0.5)
    off = np.abs(first.cpu().double().numpy() - ref)
    real = ~np.isnan(ref)
    assert (off <= tolerance(ref, spread, reach, dim, max(n for n, _ in specs), False, largest(cache)))[real].all()
    out, differs = torch.empty_like(first), torch.zeros((), dtype=torch.int64, device=DEV)
    for _ in range(200):
        out.fill_(7.0)
        cache.attention(q, batch, out=out)
        differs += (out != first).sum()
    assert int(differs) == 0
    assert _lib.load().nf4_device_status(None, None, None) == 0


@pytest.mark.parametrize("quantized", [True, False])
def test_a_prompt_beside_them(quantized):
    """Row tiles that several CTAs share, between those of which a CTA has many."""
    specs = short_prompts(30, 60)[:15] + [(900, 700)] + short_prompts(30, 60)[15:] + [(3000, 40)]
    batch, pages = batch_of(specs, 16, spare_rows=(0, 2))
    cache = filled_cache(pages, 16, 8, 128, quantized)
    g = torch.Generator(device=DEV).manual_seed(8)
    q = torch.randn(batch.rows, 32, 128, device=DEV, generator=g).to(BF16)
    before = _lib.launch_count()
    first = cache.attention(q, batch)
    assert _lib.launch_count() - before >= 2
    ref, spread, reach = reference(cache, batch, q, 128 ** -0.5)
    off = np.abs(first.cpu().double().numpy() - ref)
    real = ~np.isnan(ref)
    assert (off <= tolerance(ref, spread, reach, 128, 3000, False, largest(cache)))[real].all()
    rows = slice(0, batch.rows - 2)
    for _ in range(100):
        assert torch.equal(cache.attention(q, batch)[rows], first[rows])
