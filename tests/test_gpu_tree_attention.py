"""Attention of trees of drafted tokens over the paged cache, against 64 bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from cache_util import DEV, batch_of, filled_cache, largest, spoil_unused, tolerance  # noqa: E402
from tree_util import masks_of, tree_reference  # noqa: E402
from unifur_b200 import _lib  # noqa: E402
from unifur_b200.kv_cache import CacheBatch  # noqa: E402

# (tokens in the cache, the tree's nodes) of each sequence
FEW = [[(1, 1)], [(40, 3)], [(16, 1), (17, 2)], [(200, 2), (0, 0), (1, 1), (333, 1)], [(9, 9), (100, 3)], [(3, 5), (260, 4)]]
MANY = [[(300, 40), (65, 64), (1, 1)], [(130, 130)], [(20, 33), (128, 31)], [(700, 17), (0, 7), (2100, 12)], [(1100, 300)]]


def check(specs, heads, group, dim, page_size, quantized, dtype, kind="tree", seed=0, hints=True, scale=None, k_std=1.0, v_std=1.0, q_std=1.0):
    batch, pages = batch_of(specs, page_size, spare_rows=(1, 2), seed=seed, hints=hints)
    cache = filled_cache(pages, page_size, heads, dim, quantized, seed=seed + 1, k_std=k_std, v_std=v_std)
    spoil_unused(cache, batch)
    masks = masks_of(kind, specs, batch, np.random.default_rng(seed + 3))
    g = torch.Generator(device=DEV).manual_seed(seed + 2)
    wide = (torch.randn(batch.rows, heads * group * dim + 24, device=DEV, generator=g) * q_std).to(dtype)
    q = wide[:, 16:16 + heads * group * dim].unflatten(1, (heads * group, dim))
    out = torch.full((batch.rows, heads * group, dim), 7.0, device=DEV, dtype=dtype)
    got = cache.tree_attention(q, masks, batch, scale, out=out)
    assert got.data_ptr() == out.data_ptr()
    ref, spread, reach = tree_reference(cache, batch, q, masks, dim ** -0.5 if scale is None else scale)
    rows = slice(1, batch.rows - 2)
    assert bool((out[:1] == 7.0).all()) and bool((out[-2:] == 7.0).all()), "rows of no sequence were written"
    off = np.abs(out[rows].cpu().double().numpy() - ref[rows])
    may = tolerance(ref[rows], spread[rows], reach[rows], dim, max(n for n, _ in specs), dtype == torch.float32, largest(cache))
    may = np.where(spread[rows] == 0, 0, may)  # what sees nothing is zeros
    worst = float((off / np.maximum(may, 1e-300)).max())
    assert worst <= 1, f"off by {float(off.max())}, {worst} of what it may be"
    assert _lib.load().nf4_device_status(None, None, None) == 0
    return cache, batch, q, masks, got


@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("heads,group,dim,page_size", [(4, 4, 128, 64), (2, 4, 64, 16), (1, 5, 256, 48), (3, 1, 128, 32), (2, 4, 128, 48)])
@pytest.mark.parametrize("kind", ["tree", "any", "none"])
@pytest.mark.parametrize("specs", FEW)
def test_few_rows(specs, kind, heads, group, dim, page_size, quantized):
    check(specs, heads, group, dim, page_size, quantized, torch.bfloat16, kind)


@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("heads,group,dim,page_size", [(2, 7, 128, 64), (1, 4, 64, 16), (1, 3, 256, 48), (2, 1, 128, 80), (1, 16, 64, 64)])
@pytest.mark.parametrize("kind", ["tree", "any", "none"])
@pytest.mark.parametrize("specs", MANY)
def test_many_rows(specs, kind, heads, group, dim, page_size, quantized):
    check(specs, heads, group, dim, page_size, quantized, torch.bfloat16, kind)


@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("heads,group,dim,page_size", [(2, 3, 128, 64), (1, 5, 64, 16), (1, 2, 256, 48)])
@pytest.mark.parametrize("kind", ["tree", "any", "none"])
@pytest.mark.parametrize("specs", [FEW[1], FEW[3], FEW[5], MANY[0], MANY[2], MANY[3]])
def test_f32(specs, kind, heads, group, dim, page_size, quantized):
    check(specs, heads, group, dim, page_size, quantized, torch.float32, kind)


@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("specs", [[(200, 1), (5000, 3)], [(9000, 20), (300, 1), (40, 40)], [(20000, 60)]])
def test_without_hints(specs, dtype, quantized):
    check(specs, 2, 4, 128, 32, quantized, dtype, hints=False)


@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("specs", [[(3000, 2)], [(700, 40)]])
@pytest.mark.parametrize("k_std,v_std,q_std,scale", [(1e4, 1.0, 1e-4, None), (1e-6, 1e6, 1e6, 0.1), (1.0, 1e-6, 1.0, 0.0), (1.0, 1.0, 1.0, -0.3),
                                                     (3e5, 3e5, 1e-5, 0.05), (1.0, 1.0, 30.0, None)])
def test_magnitudes(specs, quantized, k_std, v_std, q_std, scale):
    """Keys, values and queries outside f16's range; scores all alike; a scale below zero; sharp scores."""
    check(specs, 1, 4, 128, 64, quantized, torch.bfloat16, k_std=k_std, v_std=v_std, q_std=q_std, scale=scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("quantized", [True, False])
def test_many_sequences(quantized, dtype):
    rng = np.random.default_rng(5)
    specs = [(int(n), int(min(n, k))) for n, k in zip(rng.integers(0, 200, 90), rng.integers(0, 20, 90))]
    check(specs, 2, 2, 64, 16, quantized, dtype)


@pytest.mark.parametrize("hint", [(1, 1), (3, 100000), (1000, 16)])
def test_wrong_hints_change_no_result(hint):
    specs = [(300, 70), (900, 1), (64, 64)]
    cache, batch, q, masks, right = check(specs, 2, 4, 128, 32, True, torch.bfloat16)
    wrong = CacheBatch(batch.page_table, batch.lengths, batch.row_starts, batch.rows, *hint)
    out = cache.tree_attention(q, masks, wrong)[1:-2].double()
    right = right[1:-2].double()
    assert float((out - right).norm() / right.norm()) < 2.0 ** -7


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [2, 30])
def test_masks_of_a_chain_are_causal_attention(dtype, rows):
    specs = [(400, rows), (rows, rows), (90, 1)]
    batch, pages = batch_of(specs, 32)
    cache = filled_cache(pages, 32, 2, 128, True)
    chain = torch.cat([torch.arange(-1, n - 1) for _, n in specs]).to(torch.int32).to(DEV)
    masks, positions = cache.tree_masks(chain, batch)
    assert positions.tolist() == [n - k + i for n, k in specs for i in range(k)]
    q = torch.randn(batch.rows, 8, 128, device=DEV).to(dtype)
    a, b = cache.tree_attention(q, masks, batch).double(), cache.attention(q, batch).double()
    # two results that are each off by their type's rounding and f16 operands' (bf16), or by sums of f32
    assert float((a - b).norm() / b.norm()) < (2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -18)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [2, 90])
def test_a_page_that_there_is_not(dtype, rows):
    specs = [(200, rows), (300, rows)]
    batch, pages = batch_of(specs, 32)
    cache = filled_cache(pages, 32, 2, 128, True)
    batch.page_table[0, 1] = pages + 5
    q = torch.randn(batch.rows, 8, 128, device=DEV).to(dtype)
    out = cache.tree_attention(q, masks_of("tree", specs, batch, np.random.default_rng(0)), batch)
    assert bool(torch.isnan(out[:rows]).all()) and bool(torch.isfinite(out[rows:]).all())


@pytest.mark.parametrize("quantized", [True, False])
def test_results_are_the_same_every_time_and_beside_other_sequences(quantized):
    specs = [(5000, 20), (700, 2), (64, 1), (3000, 33)]
    batch, pages = batch_of(specs, 64)
    cache = filled_cache(pages, 64, 4, 128, quantized)
    masks = masks_of("tree", specs, batch, np.random.default_rng(1))
    q = torch.randn(batch.rows, 28, 128, device=DEV).bfloat16()
    first = cache.tree_attention(q, masks, batch)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for i in range(20):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(cache.tree_attention(q, masks, batch))
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for o in outs)


@pytest.mark.parametrize("heads,group,dim,page_size", [(4, 4, 128, 32), (2, 16, 64, 16), (2, 5, 256, 48)])
@pytest.mark.parametrize("quantized", [True, False])
def test_pieces_of_every_number_of_steps_are_the_same_every_time(quantized, heads, group, dim, page_size):
    """Sequences of one step, of few, and ones that the shares cut anywhere, between others of unlike scales: what a piece takes of the one before it
    or after it is none of its own."""
    rng = np.random.default_rng(6)
    specs = [(int(n), int(min(n, k))) for n, k in zip(rng.choice([60, 128, 129, 300, 700], 90), rng.integers(20, 60, 90))]
    batch, pages = batch_of(specs, page_size, seed=1)
    cache = filled_cache(pages, page_size, heads, dim, quantized, seed=2)
    for i, (table, length) in enumerate(zip(batch.page_table.tolist(), batch.lengths.tolist())):
        used = table[:-(-length // page_size)]
        for t in (cache.k_scales, cache.v_scales) if quantized else (cache.k, cache.v):
            t[used] *= 2.0 ** float(rng.integers(-12, 12))
    masks = masks_of("tree", specs, batch, rng)
    q = torch.randn(batch.rows, heads * group, dim, device=DEV).bfloat16()
    first = cache.tree_attention(q, masks, batch)
    ref, spread, reach = tree_reference(cache, batch, q, masks, dim ** -0.5)
    off = np.abs(first.cpu().double().numpy() - ref)
    # Keys of such sizes make scores whose errors e = 2 * 2^-11 * reach (a level's rounding and its product's with the scale) are not small, as
    # `tolerance` takes them to be.  A weight is exp(score) over the sum of all: with scores off by up to e it is between exp(-2 e) and exp(2 e) times
    # what it should be, so that a result is off by up to (exp(2 e) - 1) * sum(weight * |value|), of which `tolerance` has 2 e.
    two_e = np.minimum(4 * 2.0 ** -11 * reach[..., None], 50.0)
    may = tolerance(ref, spread, reach, dim, 700, False, largest(cache)) + (np.expm1(two_e) - two_e) * spread
    worst = np.unravel_index(np.argmax(off / may), off.shape)
    assert bool((off <= may).all()), f"{int((off > may).sum())} of {off.size}, {worst}: off by {off[worst]} where {may[worst]} is allowed, 2 e {two_e[worst[:2]]}"
    for _ in range(60):
        assert torch.equal(cache.tree_attention(q, masks, batch), first)


def test_no_words_no_rows_no_sequences():
    specs = [(50, 3), (7, 7)]
    batch, pages = batch_of(specs, 16)
    cache = filled_cache(pages, 16, 2, 64, True)
    q = torch.randn(batch.rows, 4, 64, device=DEV).bfloat16()
    none = torch.zeros(batch.rows, 0, dtype=torch.int32, device=DEV)
    zero = torch.zeros(batch.rows, 1, dtype=torch.int32, device=DEV)
    a = cache.tree_attention(q, none, batch)
    assert torch.equal(a, cache.tree_attention(q, zero, batch)) and bool((a[3:] == 0).all()) and bool((a[:3] != 0).any())
    empty = CacheBatch(batch.page_table[:0], batch.lengths[:0], batch.row_starts[:1], 0)
    assert cache.tree_attention(q[:0], zero[:0], empty).shape == (0, 4, 64)
