"""Attention of bf16 tensors over an NF4 cache whose tokens are of unlike size: f16 operands have a step's (or a tile's) largest in common, and a row has
to be right beside tokens far larger than its own, those that it must not see above all."""
import numpy as np
import pytest
import torch

from cache_util import DEV, batch_of, filled_cache, reference
from unifur_b200 import _lib

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def tokens_scaled(cache, batch, page_size, name, factors):
    """Multiplies the scales of a single sequence's tokens (k or v), in all heads."""
    t = torch.arange(len(factors), device=DEV)
    page = batch.page_table[0, t // page_size].long()
    scales = getattr(cache, name + "_scales")
    scales[page, :, t % page_size] = scales[page, :, t % page_size] * torch.as_tensor(factors, dtype=torch.float32, device=DEV)[:, None, None]


def scales_of(cache, batch, page_size, name, length):
    """The largest scale of each token, any head."""
    t = np.arange(length)
    page = batch.page_table[0].cpu().numpy()[t // page_size]
    return getattr(cache, name + "_scales").cpu().double().numpy()[page, :, t % page_size].max((1, 2))


def check(cache, batch, q, page_size, scale=None):
    """Every result against 64 bits.  Half steps of f16, 2^-11, that count relative to what they round: three for a key (level, scale, their product),
    which move a weight by twice their share of the largest sum of |q k| (numerator and denominator); one for the weight, three for the value; f32
    sums; 2^-8 of the result for bf16.  And those that count beside larger numbers: a key or value is off by 2^-37 of the sequence's largest, a
    token's part by 2^-31 of the largest that is seen by the row or 15 rows behind it.  Rows whose own scores are so large that their half steps
    move them by more than 1/2 (those that see keys of 2^20 and more) are left out: e^(2 * 1/2) bounds nothing there."""
    dim, group = q.shape[-1], q.shape[1] // cache.heads()
    scale = dim ** -0.5 if scale is None else scale
    got = cache.attention(q, batch, scale)
    ref, spread, reach = reference(cache, batch, q, scale)
    length, n = int(batch.lengths[0]), int(batch.row_starts[1])
    high_k, high_v = (scales_of(cache, batch, page_size, name, length) for name in ("k", "v"))
    sees = length - n + np.arange(n) + 1
    near = np.array([high_v[:min(length, s + -(-15 // group))].max() for s in sees])[:, None, None]
    moved = 3 * 2.0 ** -11 * reach + 2.0 ** -37 * high_k.max() * abs(scale) * np.abs(q.cpu().double().numpy()).sum(-1) + 2.0 ** -24 * (dim + 8) * reach
    moved = np.where(moved <= 0.5, moved, np.nan)
    limit = 2.0 ** -8 * np.abs(ref) + (np.expm1(2 * moved)[..., None] + 4 * 2.0 ** -11 + 2.0 ** -24 * (2 * length + 64)) * spread * (1 + 2.0 ** -7) + \
        2.0 ** -37 * high_v.max() + length * 2.0 ** -31 * near
    off = np.abs(got.cpu().double().numpy() - ref)
    assert np.isfinite(limit).any((1, 2))[:len(limit) // 2].all()
    limit = np.where(np.isnan(limit), np.inf, limit)
    assert (off <= limit).all(), f"{float((off / limit).max())} of what it may be, first at row {int(np.argwhere(off > limit)[0][0])}"
    assert _lib.load().nf4_device_status(None, None, None) == 0
    return got, limit


def rows(batch, q_heads, dim, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(5)
    return (torch.randn(batch.rows, q_heads, dim, device=DEV, generator=g) * std).to(BF16)


# group: with the first of each dim keys and values are expanded ahead of the kernel, with the second inside it
@pytest.mark.parametrize("dim,group", [(64, 4), (64, 2), (128, 4), (128, 2), (256, 4), (256, 1)])
@pytest.mark.parametrize("k_by,v_by,scale", [(0, 25, 0.0), (0, 25, None), (25, 0, None), (20, 20, None), (0, -30, None)])
def test_a_prompt_and_larger_tokens_behind(dim, group, k_by, v_by, scale):
    """200 tokens of which the last hundred are larger, or smaller, in a first step that has both."""
    batch, pages = batch_of([(200, 200)], 16, width=4096, hints=False)
    cache = filled_cache(pages, 16, 2, dim, True)
    q = rows(batch, 2 * group, dim)
    before = _lib.launch_count()
    plain, limit = check(cache, batch, q, 16, scale)
    assert _lib.launch_count() - before >= 2
    for name, by in (("k", k_by), ("v", v_by)):
        tokens_scaled(cache, batch, 16, name, np.where(np.arange(200) >= 100, 2.0 ** by, 1.0))
    got, limit2 = check(cache, batch, q, 16, scale)
    # rows ahead do not change by more than both may be off
    assert (np.abs((got - plain)[:84].cpu().double().numpy()) <= (limit + limit2)[:84]).all()


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_a_short_prompt_and_larger_tokens_behind(dim):
    """The kernel for few rows: 30 tokens, tiles of sixteen rows are four of them; the last ten are larger."""
    batch, pages = batch_of([(30, 30)], 16)
    cache = filled_cache(pages, 16, 1, dim, True)
    q = rows(batch, 4, dim)
    before = _lib.launch_count()
    plain, limit = check(cache, batch, q, 16)
    assert _lib.launch_count() - before == 1
    tokens_scaled(cache, batch, 16, "v", np.where(np.arange(30) >= 20, 2.0 ** 28, 1.0))
    got, limit2 = check(cache, batch, q, 16)
    assert (np.abs((got - plain)[:16].cpu().double().numpy()) <= (limit + limit2)[:16]).all()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("specs,wide", [([(3000, 1)], False), ([(900, 4)], False), ([(700, 300)], True), ([(700, 90)], True)])
def test_tokens_of_all_sizes(specs, wide, dim):
    """Values between 2^-10 and 2^10, keys between 1/4 and 4."""
    batch, pages = batch_of(specs, 16, **(dict(width=4096, hints=False) if wide else {}))
    cache = filled_cache(pages, 16, 2, dim, True)
    rng = np.random.default_rng(1)
    tokens_scaled(cache, batch, 16, "k", 2.0 ** rng.uniform(-2, 2, specs[0][0]))
    tokens_scaled(cache, batch, 16, "v", 2.0 ** rng.uniform(-10, 10, specs[0][0]))
    check(cache, batch, rows(batch, 8, dim, 0.5), 16)


@pytest.mark.parametrize("k_by,v_by,q_by", [(-110, 0, 100), (0, -110, 0), (100, 90, -100)])
@pytest.mark.parametrize("n", [4, 300])
def test_near_the_ends_of_the_range(n, k_by, v_by, q_by):
    """Scales next to the smallest and largest of their type, with queries that make ordinary scores of them."""
    batch, pages = batch_of([(500, n)], 16, **(dict(width=4096, hints=False) if n > 16 else {}))
    cache = filled_cache(pages, 16, 2, 128, True)
    q = (rows(batch, 8, 128).float() * 2.0 ** q_by).to(BF16)
    tokens_scaled(cache, batch, 16, "k", np.full(500, 2.0 ** k_by))
    tokens_scaled(cache, batch, 16, "v", np.full(500, 2.0 ** v_by))
    check(cache, batch, q, 16)
