"""The operators for trees as a program calls them: values that are cut, pools beyond 32 bits, graphs in turn, many rows to a head, what is refused."""
import numpy as np
import pytest
import torch

from cache_util import DEV, batch_of, filled_cache, largest, tolerance
from test_gpu_cache_cut import both, ints
from tree_util import masks_of, tree_reference
from unifur_b200 import _lib
from unifur_b200.kv_cache import CacheBatch, PagedKvCache, Rotation

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def normal(*shape, dtype=BF16, seed=7):
    return torch.randn(*shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed)).to(dtype)


def pools(cache):
    return [t for t in (cache.k, cache.v, cache.k_scales, cache.v_scales) if t is not None]


# attention of few rows, of many (over a long context that the host knows of), of f32
@pytest.mark.parametrize("rows,dtype,long", [(4, BF16, False), (50, BF16, True), (50, F32, False)])
@pytest.mark.parametrize("quantized", [True, False])
def test_what_is_cut(rows, dtype, long, quantized):
    """Lengths beyond the page table, row starts beyond the call's rows and numbers below zero: what the cut values give, and nothing else is written."""
    heads, group, dim = 2, 4, 128
    given, cut = both(rows)
    if long:
        for b in (given, cut):
            table = torch.full((3, 8192), -1, dtype=torch.int32, device=DEV)
            table[:, :4] = b.page_table
            b.page_table, b.max_rows, b.max_length = table, 0, 0
        given.lengths, cut.lengths = ints(64, -7, 60), ints(64, 0, 60)
    cache = filled_cache(12, 16, heads, dim, quantized)
    q, masks = normal(cut.rows, heads * group, dim, dtype=dtype), masks_of("tree", [(64, 3), (0, 2), (60, rows)], cut, np.random.default_rng(1))
    outs = []
    for b in (given, cut):
        whole = torch.full((cut.rows + 4, heads * group, dim), 7.0, device=DEV, dtype=dtype)
        before = _lib.launch_count()
        cache.tree_attention(q, masks, b, out=whole[2:-2])
        assert not long or _lib.launch_count() - before >= 2
        assert (whole[:2] == 7).all() and (whole[-2:] == 7).all()
        outs.append(whole)
    assert torch.equal(*outs) and torch.isfinite(outs[0]).all()
    assert (outs[0][2 + 3:2 + 5] == 0).all()  # the rows of the sequence without tokens
    ref, spread, reach = tree_reference(cache, cut, q, masks, dim ** -0.5)
    off = np.abs(outs[0][2:-2].cpu().double().numpy() - ref)
    assert (off <= tolerance(ref, spread, reach, dim, 64, dtype == F32, largest(cache))).all()


@pytest.mark.parametrize("quantized", [True, False])
def test_the_other_operators_with_what_is_cut(quantized):
    given, cut = both(9)
    q, k, v = normal(3, cut.rows, 2, 64)
    parents = torch.full((cut.rows,), -1, dtype=torch.int32, device=DEV)
    kept, counts = ints(0, 2, 0, 1, 1, 8).view(3, 2), ints(2, 2, 2)
    seen = []
    for b in (given, cut):
        cache = filled_cache(12, 16, 2, 64, quantized)
        rotated = cache.append_rotated(k, v, b, Rotation.new(64, 64, DEV), None, q, torch.full_like(q, 7.0))
        masks, positions = cache.tree_masks(parents, b, out=(torch.zeros(b.rows, 1, dtype=torch.int32, device=DEV), torch.zeros(b.rows, dtype=torch.int32, device=DEV)))
        seen.append([rotated.nan_to_num(9.0), masks, positions, cache.keep(kept, counts, b), *pools(cache)])
    for a, b in zip(*seen):
        assert torch.equal(a, b)
    assert seen[0][3].tolist() == [63, 0, 53]


@pytest.mark.parametrize("quantized", [True, False])
def test_a_pool_beyond_32_bits(quantized):
    """Pages at the end of a pool whose bytes need more than 32 bits: what a small pool gives."""
    heads, dim, page_size = 8, 256, 64
    pages = ((1 << 32) // (heads * page_size * dim // 2 if quantized else heads * page_size * dim * 2)) + 40
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("not enough memory on the device")
    small = filled_cache(12, page_size, heads, dim, quantized)
    big = PagedKvCache(*(torch.empty(pages, *t.shape[1:], dtype=t.dtype, device=DEV) if t is not None else None
                         for t in (small.k, small.v, small.k_scales, small.v_scales)))
    for a, b in zip(pools(big), pools(small)):
        a[-12:] = b
    rotation = Rotation.new(400, 128, DEV)
    for specs, dtype in (([(300, 3), (200, 2)], BF16), ([(300, 100), (200, 70)], BF16), ([(300, 40), (200, 9)], F32)):
        batch, _ = batch_of(specs, page_size, spare_pages=0)
        there = CacheBatch(torch.where(batch.page_table < 0, batch.page_table, batch.page_table + (pages - 12)), batch.lengths, batch.row_starts,
                           batch.rows, batch.max_rows, batch.max_length)
        k, v = normal(2, batch.rows, heads, dim, dtype=dtype)
        q, masks = normal(batch.rows, 2 * heads, dim, dtype=dtype, seed=3), masks_of("tree", specs, batch, np.random.default_rng(2))
        turned = [c.append_rotated(k, v, b, rotation, None, q) for c, b in ((small, batch), (big, there))]
        assert torch.equal(*turned)
        assert torch.equal(big.tree_attention(turned[0], masks, there), small.tree_attention(turned[0], masks, batch))
        kept, counts = ints(0, 2, 1, 1).view(2, 2), ints(2, 1)
        assert torch.equal(small.keep(kept, counts, batch), big.keep(kept, counts, there))
        for a, b in zip(pools(big), pools(small)):
            assert torch.equal(a[-12:], b)


@pytest.mark.parametrize("specs", [[(900, 3), (64, 2)], [(20000, 30), (3000, 40)]])
def test_graphs_in_turn(specs):
    """Two captured calls, replayed in any order and twice in a row, beside eager ones: each has a workspace of its own."""
    batch, pages = batch_of(specs, 32)
    cache = filled_cache(pages, 32, 2, 128, True)
    masks = masks_of("tree", specs, batch, np.random.default_rng(3))
    qs = [normal(batch.rows, 8, 128, seed=i) for i in range(2)]
    want = [cache.tree_attention(q, masks, batch) for q in qs]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for q in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(cache.tree_attention(q, masks, batch))
        graphs.append(g)
    for i in (0, 1, 1, 0, 0, 1):
        outs[i].zero_()
        graphs[i].replay()
        assert torch.equal(cache.tree_attention(qs[1 - i], masks, batch), want[1 - i])
        assert torch.equal(outs[i], want[i])


@pytest.mark.parametrize("hint", [None, (300, 16), (4, 100000)])
@pytest.mark.parametrize("heads,group,dim", [(1, 8, 128), (2, 8, 64), (1, 5, 256)])
def test_a_cache_that_is_expanded_ahead(heads, group, dim, hint):
    """More than a thousand rows to a head; and hints that are wrong, so that it is expanded for fewer tokens than there are, or not."""
    specs = [(900, 300), (33, 33), (700, 290)]
    batch, pages = batch_of(specs, 32)
    if hint:
        batch.max_rows, batch.max_length = hint
    cache = filled_cache(pages, 32, heads, dim, True)
    q, masks = normal(batch.rows, heads * group, dim), masks_of("tree", specs, batch, np.random.default_rng(4))
    out = cache.tree_attention(q, masks, batch)
    ref, spread, reach = tree_reference(cache, batch, q, masks, dim ** -0.5)
    off = np.abs(out.cpu().double().numpy() - ref)
    assert (off <= tolerance(ref, spread, reach, dim, 900, False, largest(cache))).all()
    for _ in range(10):
        assert torch.equal(cache.tree_attention(q, masks, batch), out)


def test_what_is_refused():
    specs = [(40, 5)]
    batch, pages = batch_of(specs, 16)
    cache = filled_cache(pages, 16, 2, 64, True)
    q, k = normal(5, 8, 64), normal(5, 2, 64)
    masks, words = torch.zeros(5, 1, dtype=torch.int32, device=DEV), torch.zeros(5, dtype=torch.int32, device=DEV)
    rotation = Rotation.new(50, 64, DEV)
    for call, word in [
        (lambda: cache.tree_attention(q, masks.long(), batch), "masks"), (lambda: cache.tree_attention(q, masks[:4], batch), "masks"),
        (lambda: cache.tree_attention(q, masks.cpu(), batch), "device"), (lambda: cache.tree_attention(q, words, batch), "masks"),
        (lambda: cache.tree_attention(q, torch.zeros(5, 2, dtype=torch.int32, device=DEV)[:, :1], batch), "masks"),
        (lambda: cache.tree_masks(words[:4], batch), "parents"), (lambda: cache.tree_masks(words.long(), batch), "parents"),
        (lambda: cache.tree_masks(words, batch, out=(masks, words[:3])), "positions"),
        (lambda: cache.append_rotated(k, k.float(), batch, rotation), "one type"), (lambda: cache.append_rotated(k, k, batch, rotation, None, q.float()), "one type"),
        (lambda: cache.append_rotated(k, k, batch, Rotation(rotation.table.double())), "table"),
        (lambda: cache.append_rotated(k, k, batch, Rotation(rotation.table.cpu())), "device"),
        (lambda: cache.append_rotated(k, k, batch, Rotation(rotation.table[:, :32])), "table"),
        (lambda: cache.append_rotated(k, k, batch, rotation, words[:4]), "positions"), (lambda: cache.append_rotated(k, k, batch, rotation, None, None, q), "without q"),
        (lambda: cache.append_rotated(k, k, batch, rotation, None, q, q[:, :4]), "shape"), (lambda: cache.append_rotated(k[:, :1], k, batch, rotation), "k must"),
        (lambda: cache.keep(masks, words[:1], batch), "kept"), (lambda: cache.keep(masks[:1], words, batch), "counts"),
        (lambda: cache.keep(masks[:1], words[:1], batch, out=words), "out"), (lambda: cache.keep(words[:1], words[:1], batch), "kept"),
    ]:
        with pytest.raises(ValueError, match=word):
            call()
    for call in (lambda: cache.append_rotated(k, k, batch, Rotation(torch.zeros(50, 24, device=DEV))), lambda: cache.append_rotated(k, k, batch, Rotation(torch.zeros(50, 128, device=DEV)))):
        with pytest.raises(_lib.Nf4Error, match="rotary_dim"):
            call()
    with pytest.raises(_lib.Nf4Error, match="aligned"):
        cache.append_rotated(k, k, batch, Rotation(torch.zeros(64 * 51, device=DEV)[1:64 * 50 + 1].view(50, 64)))
    with pytest.raises(_lib.Nf4Error, match="scale"):
        cache.tree_attention(q, masks, batch, float("inf"))


def test_rows_of_larger_tensors_at_odd_places():
    """Rows that are not 16-byte aligned are copied; results go where they are asked for."""
    specs = [(70, 9), (30, 4)]
    batch, pages = batch_of(specs, 16)
    caches = [filled_cache(pages, 16, 2, 64, True) for _ in range(2)]
    masks, rotation = masks_of("tree", specs, batch, np.random.default_rng(5)), Rotation.new(80, 32, DEV, pairs=True)
    wide = normal(batch.rows, 8 * 64 + 2 * 128 + 9)
    q, k, v = wide[:, 1:513], wide[:, 515:643], wide[:, 645:773]
    got = caches[0].append_rotated(k, v, batch, rotation, None, q)
    want = caches[1].append_rotated(k.contiguous(), v.contiguous(), batch, rotation, None, q.contiguous())
    assert torch.equal(got, want)
    for a, b in zip(*(pools(c) for c in caches)):
        assert torch.equal(a, b)
    out = torch.zeros(batch.rows, 2, 8, 64, dtype=BF16, device=DEV)
    assert torch.equal(caches[0].tree_attention(q.unflatten(1, (8, 64)), masks, batch, out=out[:, 1]), caches[1].tree_attention(q.contiguous(), masks, batch).view(-1, 8, 64))
    assert bool((out[:, 0] == 0).all())


@pytest.mark.parametrize("heads,group,dim,page_size", [(2, 4, 128, 16), (2, 8, 64, 48), (1, 4, 256, 16)])
def test_a_page_that_there_is_not_among_small_ones(heads, group, dim, page_size):
    """Each head's and each step's: pages -1 and behind the pool, in the first and the last steps of the sequence."""
    specs = [(700, 30), (900, 30), (500, 30), (300, 30)]
    batch, pages = batch_of(specs, page_size)
    cache = filled_cache(pages, page_size, heads, dim, False)
    batch.page_table[0, 0] = -1
    batch.page_table[2, (500 - 31) // page_size] = pages
    q = torch.randn(batch.rows, heads * group, dim, device=DEV).bfloat16()
    out = cache.tree_attention(q, masks_of("tree", specs, batch, np.random.default_rng(0)), batch)
    for s in range(4):
        rows = out[30 * s:30 * s + 30]
        assert bool(torch.isnan(rows).all()) if s in (0, 2) else bool(torch.isfinite(rows).all())


@pytest.mark.parametrize("heads,group,dim,page_size", [(4, 4, 128, 16), (2, 8, 64, 16), (2, 8, 64, 112), (2, 5, 256, 16)])
def test_small_pages_are_as_large_ones(heads, group, dim, page_size):
    """A bf16 cache of the same tokens in small pages and in large ones: sequences of one step to many, every time the same bits."""
    rng = np.random.default_rng(8)
    specs = [(int(n), int(min(n, k))) for n, k in zip(rng.choice([1, 60, 128, 129, 300, 700, 2500], 60), rng.integers(10, 50, 60))]
    outs = []
    for size in (page_size, 128):
        batch, pages = batch_of(specs, size)
        cache = filled_cache(pages, size, heads, dim, False)
        cache.k.zero_(), cache.v.zero_()
        for s, (n, _) in enumerate(specs):
            g = torch.Generator(device=DEV).manual_seed(s)
            k, v = (torch.randn(n, heads, dim, device=DEV, generator=g).bfloat16() for _ in range(2))
            for t0 in range(0, n, size):
                page, some = int(batch.page_table[s, t0 // size]), min(size, n - t0)
                cache.k[page, :, :some], cache.v[page, :, :some] = k[t0:t0 + some].transpose(0, 1), v[t0:t0 + some].transpose(0, 1)
        q = torch.randn(batch.rows, heads * group, dim, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1000)).bfloat16()
        masks = masks_of("tree", specs, batch, np.random.default_rng(3))
        outs.append([cache.tree_attention(q, masks, batch) for _ in range(5)])
    assert all(torch.equal(o, outs[0][0]) for o in outs[0] + outs[1])
