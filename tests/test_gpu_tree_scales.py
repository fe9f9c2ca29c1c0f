"""Attention of trees over an NF4 cache whose nodes are of unlike size: f16 operands have units in common, and a node has to be right beside nodes of other
branches that are far larger than all that it sees."""
import numpy as np
import pytest
import torch

from cache_util import DEV, batch_of, filled_cache
from test_gpu_cache_scales import rows, scales_of, tokens_scaled
from tree_kernels import takes_the_kernel_for_many
from tree_util import packed, tree_reference, unpacked
from unifur_b200 import _lib

pytestmark = pytest.mark.gpu


def visible(masks, context, n):
    """[n, context + n]: the tokens that each node sees."""
    return np.concatenate((np.ones((n, context), bool), unpacked(masks.cpu().numpy())[:, :n]), 1)


def check(cache, batch, q, masks, page_size, many):
    """Every result of one sequence against 64 bits.  Half steps of f16, 2^-11, that count relative to what they round: three for a key (level, scale, their product),
    which move a weight by twice their share of the largest sum of |q k| (numerator and denominator); one for the weight, three for the value; f32
    sums; 2^-8 of the result for bf16.  And those that count beside other numbers, as the header has them.  Few rows: a token's part is off by 2^-31 of the largest value that
    the row or one of 15 on either side of it sees.  Many: a key or value by 2^-37 of the largest among the step's tokens (128, or 64 with a dim of 256), a token's
    part by 2^-28 of its own value.  Rows whose keys' half steps move their scores by more than 1/2 are left out: e^(2 * 1/2) bounds nothing there."""
    dim, group = q.shape[-1], q.shape[1] // cache.heads()
    length, n = int(batch.lengths[0]), batch.rows
    assert takes_the_kernel_for_many(cache, batch, q.shape[1]) == many
    got = cache.tree_attention(q, masks, batch)
    ref, spread, reach = tree_reference(cache, batch, q, masks, dim ** -0.5)
    sees = visible(masks, length - n, n)
    high_k, high_v = (scales_of(cache, batch, page_size, name, length) for name in ("k", "v"))
    moved = 3 * 2.0 ** -11 * reach + 2.0 ** -24 * (dim + 8) * reach
    if many:
        step = 64 if dim == 256 else 128
        near_k, near_v = (np.repeat([h[t:t + step].max() for t in range(0, length, step)], step)[:length] for h in (high_k, high_v))
        moved += 2.0 ** -37 * (sees * near_k).max(1)[:, None] * dim ** -0.5 * np.abs(q.cpu().double().numpy()).sum(-1)
        beside = (2.0 ** -37 * (sees * near_v).max(1) + 2.0 ** -28 * (sees * high_v).sum(1))[:, None, None]
    else:
        away = -(-15 // group)
        beside = length * 2.0 ** -31 * np.array([(sees[max(i - away, 0):i + away + 1] * high_v).max() for i in range(n)])[:, None, None]
    moved = np.where(moved <= 0.5, moved, np.nan)
    limit = 2.0 ** -8 * np.abs(ref) + (np.expm1(2 * moved)[..., None] + 4 * 2.0 ** -11 + 2.0 ** -24 * (2 * length + 64)) * spread * (1 + 2.0 ** -7) + beside
    assert np.isfinite(limit).mean() > 0.5
    off = np.abs(got.cpu().double().numpy() - ref)
    limit = np.where(np.isnan(limit), np.inf, limit)
    assert (off <= limit).all(), f"{float((off / limit).max())} of what it may be, first at row {int(np.argwhere(off > limit)[0][0])}"
    assert _lib.load().nf4_device_status(None, None, None) == 0


def branches(n, alone, rng, apart=0):
    """Masks of nodes that see themselves and a third of the others, and of `alone` none but itself; those from number `apart` on none ahead of it."""
    bits = rng.random((n, n)) < 0.3
    bits[:, alone] = False
    bits[apart:, :apart] = False
    bits[np.arange(n), np.arange(n)] = True
    return torch.from_numpy(packed(bits, -(-n // 32))).to(DEV)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("k_by,v_by", [(0, 0), (0, 25), (0, 60), (20, 20), (0, -30)])
@pytest.mark.parametrize("context,n,group", [(8, 64, 4), (0, 30, 2), (100, 40, 8), (3, 12, 16)])
def test_few_rows_beside_a_larger_node_of_another_branch(context, n, group, k_by, v_by, dim):
    batch, pages = batch_of([(context + n, n)], 16)
    cache = filled_cache(pages, 16, 2, dim, True)
    factors = np.ones((2, context + n))
    factors[0, context + 5], factors[1, context + 5] = 2.0 ** k_by, 2.0 ** v_by
    for name, by in zip("kv", factors):
        tokens_scaled(cache, batch, 16, name, by)
    check(cache, batch, rows(batch, 2 * group, dim), branches(n, [5], np.random.default_rng(n)), 16, False)


# the last: expanded ahead
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("k_by,v_by", [(0, 0), (0, 25), (0, 40), (0, 100), (15, 20), (0, -30), (0, -100)])
@pytest.mark.parametrize("context,n,group", [(0, 300, 2), (128, 400, 1), (128, 290, 3), (0, 300, 4)])
def test_many_rows_beside_larger_nodes_of_another_branch(context, n, group, k_by, v_by, dim):
    """Larger nodes in a step whose nodes most others do not see, ahead of the steps that these see."""
    batch, pages = batch_of([(context + n, n)], 16, width=4096, hints=False)
    cache = filled_cache(pages, 16, 2, dim, True)
    step, large = 64 if dim == 256 else 128, [3, 7]
    factors = np.ones((2, context + n))
    for node in large:
        factors[0, context + node], factors[1, context + node] = 2.0 ** k_by, 2.0 ** v_by
    for name, by in zip("kv", factors):
        tokens_scaled(cache, batch, 16, name, by)
    check(cache, batch, rows(batch, 2 * group, dim), branches(n, large, np.random.default_rng(n), step), 16, True)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("by", [[0, 100, 0, -100, 60, -20], [-110, 90, 0, 50, -60, 90], [0, -3, -6, -9, -12, -15], [100, 40, -20, -80, -110, 10], [-110, -50, 10, 70, 100, 100]])
def test_steps_that_rise_and_fall(by, dim):
    """Each step of tokens of another size, up and down over the whole range of f32; rows see some steps, and others not."""
    step, n = 64 if dim == 256 else 128, 6 * (64 if dim == 256 else 128)
    batch, pages = batch_of([(n, n)], 16, width=4096, hints=False)
    cache = filled_cache(pages, 16, 1, dim, True)
    tokens_scaled(cache, batch, 16, "v", np.repeat(2.0 ** np.array(by), step))
    rng = np.random.default_rng(2)
    bits = np.repeat(rng.random((n, 6)) < 0.4, step, 1) & (rng.random((n, n)) < 0.5)
    bits[np.arange(n), np.arange(n)] = True
    check(cache, batch, rows(batch, 2, dim, 0.5), torch.from_numpy(packed(bits, -(-n // 32))).to(DEV), 16, True)
