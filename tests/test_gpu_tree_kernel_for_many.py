"""The kernel for many rows of trees, which every test here asks the library about: a page table with room for many tokens, or hints of many, stand for it where a batch is
small.  Its ways in: pages of a bf16 cache by boxes or by small copies, codes expanded where they are used or ahead."""
import numpy as np
import pytest
import torch

from cache_util import DEV, batch_of, filled_cache, largest, spoil_unused, tolerance
from tree_kernels import takes_the_kernel_for_many
from tree_util import masks_of, tree_reference
from unifur_b200 import _lib

pytestmark = pytest.mark.gpu

FORMS = ["bf16", "nf4", "nf4 ahead"]


def wide_batch(form, specs, page_size, group):
    """Rows of no sequence, of which the host cannot know, for many; a cache is expanded ahead where there may be more than 1024 rows of a head."""
    ahead = form == "nf4 ahead"
    batch, pages = batch_of(specs, page_size, width=65536 // page_size, hints=False, spare_rows=(1, 1100 if ahead else 300))
    if ahead:
        batch.max_length = max(2000, *(n for n, _ in specs))
    else:
        batch.max_rows = 1024 // group
    return batch, pages


def check(form, specs, heads, group, dim, page_size, kind="tree", seed=0, scale=None, k_std=1.0, v_std=1.0, q_std=1.0):
    batch, pages = wide_batch(form, specs, page_size, group)
    cache = filled_cache(pages, page_size, heads, dim, form != "bf16", seed=seed + 1, k_std=k_std, v_std=v_std)
    spoil_unused(cache, batch)
    masks = masks_of(kind, specs, batch, np.random.default_rng(seed + 3))
    g = torch.Generator(device=DEV).manual_seed(seed + 2)
    q = (torch.randn(batch.rows, heads * group, dim, device=DEV, generator=g) * q_std).bfloat16()
    out = torch.full_like(q, 7.0)
    assert takes_the_kernel_for_many(cache, batch, heads * group)
    before = _lib.launch_count()
    cache.tree_attention(q, masks, batch, scale, out=out)
    assert _lib.launch_count() - before == (3 if form == "nf4 ahead" else 2)
    ref, spread, reach = tree_reference(cache, batch, q, masks, dim ** -0.5 if scale is None else scale)
    rows = slice(1, 1 + sum(n for _, n in specs))
    assert bool((out[:1] == 7.0).all()) and bool((out[rows.stop:] == 7.0).all()), "rows of no sequence were written"
    off = np.abs(out[rows].cpu().double().numpy() - ref[rows])
    # scores off by up to e move a weight by a factor between exp(-2 e) and exp(2 e), of which `tolerance` has 2 e: see the test of pieces of every number of steps
    two_e = np.minimum(4 * 2.0 ** -11 * reach[rows][..., None], 50.0)
    may = tolerance(ref[rows], spread[rows], reach[rows], dim, max(n for n, _ in specs), False, largest(cache)) + (np.expm1(two_e) - two_e) * spread[rows]
    may = np.where(spread[rows] == 0, 0, may)  # what sees nothing is zeros
    worst = float((off / np.maximum(may, 1e-300)).max())
    assert worst <= 1, f"off by {float(off.max())}, {worst} of what it may be"
    assert _lib.load().nf4_device_status(None, None, None) == 0


# the third has nodes without a token (a length below the rows) and a sequence of no tokens
SPECS = [[(1, 1)], [(300, 40), (65, 64), (1, 1)], [(0, 7), (20, 33), (700, 17), (0, 0), (2100, 12)], [(129, 2), (128, 128), (256, 100), (64, 64)], [(1100, 300), (40, 3)]]
SHAPES = [(2, 7, 128, 64), (1, 4, 64, 16), (1, 3, 256, 48), (2, 2, 128, 80), (1, 16, 64, 64)]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("shape", range(5))
@pytest.mark.parametrize("which", range(5))
def test_uneven_batches(which, shape, form):
    """Masks are trees, whatever bits, or none, another for each batch of a shape."""
    check(form, SPECS[which], *SHAPES[shape], ["tree", "any", "none"][(which + shape) % 3])


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("k_std,v_std,q_std,scale", [(1e4, 1.0, 1e-4, None), (1e-6, 1e6, 1e6, 0.1), (1.0, 1e-6, 1.0, 0.0), (1.0, 1.0, 1.0, -0.3),
                                                     (3e5, 3e5, 1e-5, 0.05), (1.0, 1.0, 30.0, None)])
def test_magnitudes(dim, form, k_std, v_std, q_std, scale):
    """Keys, values and queries outside f16's range; scores all alike; a scale below zero; sharp scores."""
    check(form, [(700, 40), (150, 150)], 1, 4, dim, 64, k_std=k_std, v_std=v_std, q_std=q_std, scale=scale)


# pages of sixteen tokens are a bf16 cache's small copies, of 64 boxes
@pytest.mark.parametrize("form,page_size", [("bf16", 16), ("bf16", 64), ("nf4", 16), ("nf4", 64), ("nf4 ahead", 32)])
@pytest.mark.parametrize("heads,group,dim", [(4, 4, 128), (4, 4, 64), (3, 5, 256)])
def test_pages_that_there_are_not(form, page_size, heads, group, dim):
    """In sequences of one step, of few, and ones that are divided, between whole ones: theirs are NaNs, and the others' bits as they are with all pages there."""
    rng = np.random.default_rng(3)
    specs = [(int(n), int(k)) for n, k in zip(rng.choice([60, 100, 128, 129, 300, 700], 90), rng.integers(10, 40, 90))]
    specs[7], specs[50] = (5000, 30), (4000, 35)
    batch, pages = wide_batch(form, specs, page_size, group)
    cache = filled_cache(pages, page_size, heads, dim, form != "bf16")
    masks = masks_of("tree", specs, batch, rng)
    q = torch.randn(batch.rows, heads * group, dim, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).bfloat16()
    assert takes_the_kernel_for_many(cache, batch, heads * group)
    whole = cache.tree_attention(q, masks, batch)
    assert bool(torch.isfinite(whole[1:1 + sum(n for _, n in specs)]).all())
    bad = sorted({7, *(int(s) for s in rng.choice(90, 30, replace=False) if s != 50)})
    for s in bad:  # a page that has a token of the context
        length, n = specs[s]
        batch.page_table[s, int(rng.integers(0, (length - n - 1) // page_size + 1))] = [-1, pages, 2 ** 31 - 1, -2 ** 31][s % 4]
    starts = batch.row_starts.tolist()
    for _ in range(5):
        out = cache.tree_attention(q, masks, batch)
        for s in range(90):
            rows = slice(starts[s], starts[s + 1])
            if s in bad:
                assert bool(torch.isnan(out[rows]).all()), f"sequence {s}, {specs[s]}"
            else:
                assert torch.equal(out[rows], whole[rows]), f"sequence {s}, {specs[s]}"
    assert _lib.load().nf4_device_status(None, None, None) == 0
