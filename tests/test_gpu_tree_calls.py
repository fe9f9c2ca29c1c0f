"""Masks of trees, appending with rotation, keeping a path, and the operators of a step with drafted tokens together."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from cache_util import DEV, batch_of, filled_cache, largest, stored, tolerance  # noqa: E402
from tree_util import ancestors, packed, random_parents, tree_reference  # noqa: E402
from unifur_b200.kv_cache import CacheBatch, PagedKvCache, Rotation  # noqa: E402
from unifur_b200.quantize import PackedNf4Tensor  # noqa: E402


def pools(cache):
    return [t for t in (cache.k, cache.v, cache.k_scales, cache.v_scales) if t is not None]


# ---- masks and positions ------------------------------------------------------------------------
@pytest.mark.parametrize("specs", [[(1, 1)], [(50, 32), (40, 33), (9, 0), (3, 5)], [(5000, 700), (64, 64)], [(300, 129)] * 40])
@pytest.mark.parametrize("words", [None, 1, 40])
def test_masks_and_positions(specs, words):
    rng = np.random.default_rng(len(specs))
    batch, pages = batch_of(specs, 16, spare_rows=(2, 1))
    cache = filled_cache(pages, 16, 1, 64, True)
    parents = random_parents(specs, (2, 1), rng)
    if words is None:
        masks, positions = cache.tree_masks(torch.from_numpy(parents).to(DEV), batch)
    else:
        out = (torch.full((batch.rows, words), 5, dtype=torch.int32, device=DEV), torch.full((batch.rows,), 5, dtype=torch.int32, device=DEV))
        masks, positions = cache.tree_masks(torch.from_numpy(parents).to(DEV), batch, out=out)
        assert bool((masks[:2] == 5).all()) and bool((masks[-1:] == 5).all()) and int(positions[1]) == 5 and int(positions[-1]) == 5
    starts = batch.row_starts.tolist()
    for s, (length, n) in enumerate(specs):
        seen, depth = ancestors(parents, starts[s], n)
        rows = slice(starts[s], starts[s + 1])
        assert (masks[rows].cpu().numpy() == packed(seen, masks.shape[1])).all()
        assert (positions[rows].cpu().numpy() == length - n + depth).all()


def test_parents_that_are_none_make_roots():
    specs = [(20, 6)]
    batch, pages = batch_of(specs, 16)
    cache = filled_cache(pages, 16, 1, 64, True)
    parents = torch.tensor([0, 1, 5, -7, 100000, 1], dtype=torch.int32, device=DEV)  # of itself, of a later one, of none
    masks, positions = cache.tree_masks(parents, batch)
    assert masks[:, 0].tolist() == [1, 2, 4, 8, 16, 2 | 32] and positions.tolist() == [14, 14, 14, 14, 14, 15]


def test_a_long_chain():
    n = 2050
    batch, pages = batch_of([(n, n)], 64)
    cache = filled_cache(pages, 64, 1, 64, True)
    masks, positions = cache.tree_masks(torch.arange(-1, n - 1, dtype=torch.int32, device=DEV), batch)
    assert (masks.cpu().numpy() == packed(np.tril(np.ones((n, n), bool)), -(-n // 32))).all()
    assert positions.tolist() == list(range(n))


@pytest.mark.parametrize("near,words", [(1, None), (3, None), (40, 130), (5000, None), (40, 7), (2, 100)])
@pytest.mark.parametrize("hints", [True, False])
def test_deep_trees_of_thousands_of_nodes(near, words, hints):
    """Ways that go through most words of a row, or leap over many; with masks for fewer nodes and for more."""
    specs = [(4500, 4300), (3, 3), (2049, 2049), (257, 256)]
    rng = np.random.default_rng(near)
    batch, pages = batch_of(specs, 64, spare_rows=(1, 1), hints=hints)
    cache = filled_cache(pages, 64, 1, 64, True)
    starts = batch.row_starts.tolist()
    parents = np.zeros(batch.rows, np.int32)
    for s, (_, n) in enumerate(specs):
        i = np.arange(n)
        parents[starts[s]:starts[s + 1]] = np.where(i == 0, -1, np.maximum(i - rng.integers(1, near + 1, n), -1))
    words = words or -(-4300 // 32)
    out = (torch.full((batch.rows, words), 5, dtype=torch.int32, device=DEV), torch.full((batch.rows,), 5, dtype=torch.int32, device=DEV))
    masks, positions = (t.cpu().numpy() for t in cache.tree_masks(torch.from_numpy(parents).to(DEV), batch, out=out))
    for t in (masks, positions):
        assert (t[0] == 5).all() and (t[-1] == 5).all()
    for s, (length, n) in enumerate(specs):
        seen, depth = ancestors(parents, starts[s], n)
        rows = slice(starts[s], starts[s + 1])
        assert (masks[rows] == packed(seen, words)).all() and (positions[rows] == length - n + depth).all()


# ---- appending with rotation --------------------------------------------------------------------
def turned(x, positions, table, pairs):
    """In f32, each product and sum rounded; and a sum of magnitudes for tolerances."""
    half, x = table.shape[1] // 2, x.float()
    turn = table[positions.long()][:, None]
    cos, sin = turn[..., :half], turn[..., half:]
    out = x.clone()
    one, two = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if pairs else (slice(0, half), slice(half, 2 * half))
    a, b = x[..., one], x[..., two]
    out[..., one] = a * cos - b * sin
    out[..., two] = b * cos + a * sin
    return out


ROTATED = [(4, 7, 128, 64, 128, False), (2, 4, 64, 16, 64, True), (3, 1, 64, 48, 32, False), (2, 2, 256, 16, 256, False), (1, 5, 256, 32, 176, True),
           (2, 3, 128, 16, 64, False), (1, 1, 128, 64, 16, True), (8, 4, 128, 32, 96, False)]


@pytest.mark.parametrize("heads,group,dim,page_size,rotary,pairs", ROTATED)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("specs,given", [([(1, 1)], False), ([(333, 5), (64, 64), (1, 1), (3, 5)], False), ([(90, 20), (0, 0), (33, 17)], True),
                                         ([(1500, 1400)], False)])
def test_append_rotated(specs, given, quantized, dtype, heads, group, dim, page_size, rotary, pairs):
    batch, pages = batch_of(specs, page_size, spare_rows=(2, 3))
    cache, plain = (filled_cache(pages, page_size, heads, dim, quantized, seed=1) for _ in range(2))
    g = torch.Generator(device=DEV).manual_seed(2)
    wide = torch.randn(batch.rows, (2 + group) * heads * dim + 24, device=DEV, generator=g).to(dtype)
    wide[3 % batch.rows] = 0.0
    q, k, v = (wide[:, a:b].unflatten(1, (-1, dim)) for a, b in ((8, 8 + group * heads * dim), (16 + group * heads * dim, 16 + (group + 1) * heads * dim),
                                                              (24 + (group + 1) * heads * dim, None)))
    rotation = Rotation.new(1600, rotary, DEV, base=500.0, pairs=pairs)
    own = torch.zeros(batch.rows, dtype=torch.int64)
    at = 2
    for length, n in specs:
        own[at:at + n] = torch.arange(length - n, length)
        at += n
    in_sequence = torch.zeros(batch.rows, dtype=torch.bool)
    in_sequence[2:-3] = True
    positions = torch.randint(0, 1600, (batch.rows,), generator=g, device=DEV, dtype=torch.int32) if given else own.to(DEV)
    out = torch.full((batch.rows, group * heads, dim), 7.0, device=DEV, dtype=dtype)
    got = cache.append_rotated(k, v, batch, rotation, positions if given else None, q, out)
    assert got.data_ptr() == out.data_ptr()
    # the cache has what append makes of the rotated f32 rows, bit for bit, and nothing else
    safe = positions.clamp(min=0)
    k32 = turned(k, safe, rotation.table, pairs)
    plain.append(k32, v.float(), batch)
    for a, b in zip(pools(cache), pools(plain)):
        assert torch.equal(torch.nan_to_num(a.float()), torch.nan_to_num(b.float()))
    want = turned(q, safe, rotation.table, pairs).to(dtype)
    there = in_sequence & (positions.cpu() >= 0)
    assert torch.equal(out[there], want[there])
    assert bool((out[~in_sequence] == 7.0).all())
    assert bool(torch.isnan(out[in_sequence & ~there]).all())
    # without queries, and in place
    again = filled_cache(pages, page_size, heads, dim, quantized, seed=1)
    assert again.append_rotated(k, v, batch, rotation, positions if given else None) is None
    for a, b in zip(pools(cache), pools(again)):
        assert torch.equal(a, b)
    held = q.clone()
    assert again.append_rotated(k, v, batch, rotation, positions if given else None, held, held).data_ptr() == held.data_ptr()
    assert torch.equal(held[there], want[there])


def test_the_cache_of_rotated_keys_is_the_quantizers():
    specs = [(100, 70)]
    batch, pages = batch_of(specs, 32)
    cache = PagedKvCache.new(pages, 32, 2, 128, DEV)
    rotation = Rotation.new(100, 128, DEV)
    k, v = torch.randn(2, 70, 2, 128, device=DEV).bfloat16()
    cache.append_rotated(k, v, batch, rotation)
    packed_k = PackedNf4Tensor.quantize(turned(k, torch.arange(30, 100, device=DEV), rotation.table, False).flatten())
    got, _ = cache.read(batch)
    assert torch.equal(got.flatten(), packed_k.dequantize())


def test_table_of_the_rotation():
    for positions, dim, base in ((5, 16, 10.0), (3000, 64, 1e6)):
        t = Rotation.new(positions, dim, DEV, base=base).table.cpu().double().numpy()
        angles = np.arange(positions)[:, None] * base ** (-2.0 * np.arange(dim // 2) / dim)
        # rounded to f32 once, from angles that are off by a few of 64 bits' roundings
        assert np.abs(t - np.concatenate((np.cos(angles), np.sin(angles)), 1)).max() <= 2.0 ** -25 + 8 * 2.0 ** -53 * positions


@pytest.mark.parametrize("quantized", [True, False])
def test_positions_outside_the_table_and_places_that_there_are_not(quantized):
    specs = [(40, 40), (20, 20)]
    batch, pages = batch_of(specs, 16)
    batch.page_table[0, 1], batch.page_table[1, 0] = -3, pages
    cache = filled_cache(pages, 16, 2, 64, quantized)
    before = [t.clone() for t in pools(cache)]
    rotation = Rotation.new(30, 64, DEV)
    q, k, v = torch.randn(3, 60, 2, 64, device=DEV)
    out = cache.append_rotated(k, v, batch, rotation, None, q)
    own = torch.cat((torch.arange(40), torch.arange(20)))
    assert bool(torch.isnan(out[own >= 30]).all()) and torch.equal(out[own < 30], turned(q, own.to(DEV).clamp(max=29), rotation.table, False)[own < 30])
    # written: tokens 0-15 of the first, 16-19 of the second (32-39 are behind the table)
    changed = sum(int((a != b).flatten(3).any(-1).any(1).sum()) for a, b in zip(before[:2], pools(cache)[:2]))
    assert changed == 2 * (16 + 4)
    none = Rotation(torch.empty(0, 64, device=DEV))
    assert bool(torch.isnan(cache.append_rotated(k, v, batch, none, None, q)).all())


def test_numbers_that_are_none():
    specs = [(4, 4)]
    batch, pages = batch_of(specs, 16)
    cache = PagedKvCache.new(pages, 16, 1, 64, DEV, quantized=False)
    rotation = Rotation.new(4, 32, DEV)
    k = torch.randn(4, 1, 64, device=DEV)
    k[1, 0, 3], k[2, 0, 40], k[3, 0, 7] = float("nan"), float("inf"), -float("inf")
    q = cache.append_rotated(k, k, batch, rotation, None, k.clone())
    want = turned(k, torch.arange(4, device=DEV), rotation.table, False)
    assert torch.equal(torch.isnan(q), torch.isnan(want)) and torch.equal(torch.nan_to_num(q), torch.nan_to_num(want))
    back, _ = cache.read(batch)
    assert torch.equal(torch.isnan(back), torch.isnan(want))


# ---- keeping a path -----------------------------------------------------------------------------
KEPT = [
    ([(40, 9)], [[0, 2, 5]]), ([(8, 8), (300, 20), (5, 0), (64, 1)], [[0, 1, 2, 3, 4, 5, 6, 7], [3, 4, 5, 6, 19], [], [0]]),
    ([(50, 40), (3, 5)], [[], [0, 1, 4]]),                          # nothing kept; two of the nodes have no token
    ([(700, 600)], [list(range(1, 600, 2))]),                        # a path over many pages, longer than a step of the kernel
    ([(700, 600)], [list(range(1, 600))]),                           # each node to the place of the one before
]


@pytest.mark.parametrize("heads,dim,page_size", [(4, 128, 64), (3, 64, 16), (16, 256, 48)])
@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("specs,paths", KEPT)
def test_keep(specs, paths, quantized, heads, dim, page_size):
    batch, pages = batch_of(specs, page_size, spare_rows=(1, 1))
    cache = filled_cache(pages, page_size, heads, dim, quantized, seed=3)
    want = [t.clone() for t in pools(cache)]
    table = batch.page_table.cpu()
    for s, ((length, n), path) in enumerate(zip(specs, paths)):
        for j, node in enumerate(path):
            old, new = length - n + node, length - n + j
            if old >= 0 and new >= 0:
                for t in want:
                    t[table[s, new // page_size], :, new % page_size] = t[table[s, old // page_size], :, old % page_size]
    most = max(1, max(len(p) for p in paths))
    kept = torch.zeros(len(specs), most, dtype=torch.int32)
    for row, path in zip(kept, paths):
        row[:len(path)] = torch.tensor(path, dtype=torch.int32)
    counts = torch.tensor([len(p) for p in paths], dtype=torch.int32, device=DEV)
    was = batch.lengths.clone()
    lengths = cache.keep(kept.to(DEV), counts, batch)
    assert torch.equal(batch.lengths, was)
    assert lengths.tolist() == [max(0, length - n + len(p)) for (length, n), p in zip(specs, paths)]
    for a, b in zip(pools(cache), want):
        assert torch.equal(a, b)
    # lengths in place, of paths that leave everything where it is
    first = torch.arange(most, dtype=torch.int32, device=DEV).expand(len(specs), most).contiguous()
    assert cache.keep(first, counts, batch, out=batch.lengths).data_ptr() == batch.lengths.data_ptr()
    assert torch.equal(batch.lengths, lengths)
    for a, b in zip(pools(cache), want):
        assert torch.equal(a, b)


def test_paths_end_at_what_is_no_path():
    specs = [(20, 6)] * 6
    batch, pages = batch_of(specs, 16)
    cache = filled_cache(pages, 16, 1, 64, True)
    kept = torch.tensor([[0, 2, 2, 3], [0, 6, 7, 8], [-1, 0, 1, 2], [3, 1, 4, 5], [0, 1, 2, 3], [0, 1, 2, 3]], dtype=torch.int32, device=DEV)
    counts = torch.tensor([4, 4, 4, 4, 100, -5], dtype=torch.int32, device=DEV)
    assert cache.keep(kept, counts, batch).tolist() == [14 + 2, 14 + 1, 14, 14 + 1, 14 + 4, 14]


@pytest.mark.parametrize("quantized", [True, False])
def test_keep_skips_pages_that_there_are_not(quantized):
    specs = [(40, 30), (40, 30)]
    batch, pages = batch_of(specs, 16)
    cache = filled_cache(pages, 16, 2, 64, quantized)
    batch.page_table[0, 2], batch.page_table[1, 0] = -1, pages
    before = [t.clone() for t in pools(cache)]
    kept = torch.tensor([[1, 4, 25], [1, 4, 25]], dtype=torch.int32, device=DEV)
    counts = torch.tensor([3, 3], dtype=torch.int32, device=DEV)
    assert cache.keep(kept, counts, batch).tolist() == [13, 13]
    changed = sum(int((a != b).flatten(3).any(-1).any(1).sum()) for a, b in zip(before[:2], pools(cache)[:2]))
    assert changed == 2 * 2  # the first sequence's two; 25 is in no page, and the second's places are in none


# ---- together -----------------------------------------------------------------------------------
@pytest.mark.parametrize("quantized", [True, False])
def test_steps_with_drafted_tokens_give_what_their_paths_alone_give(quantized):
    """Two layers' caches: trees are appended, verified and cut to a path, step after step, one by one and as replays of one captured step.
    Each step's attention is the 64-bit result over what is cached, and at the end the caches hold what appending
    the accepted tokens alone gives."""
    heads, group, dim, page_size, n, most = 2, 4, 128, 16, 3, 12
    g = torch.Generator(device=DEV).manual_seed(3)
    rng = np.random.default_rng(4)
    lengths0 = [15, 1, 40]
    table = torch.randperm(18, device=DEV, generator=g).to(torch.int32).view(n, 6)
    rotation = Rotation.new(96, dim, DEV)
    starts = torch.arange(0, n * most + 1, most, dtype=torch.int32, device=DEV)
    first = torch.tensor(np.cumsum([0] + lengths0), dtype=torch.int32, device=DEV)
    prefix = torch.randn(2, 2, sum(lengths0), heads, dim, device=DEV, generator=g).bfloat16()
    steps = 4
    parents = torch.from_numpy(np.stack([random_parents([(0, most)] * n, (0, 0), rng, roots=0) for _ in range(steps)])).to(DEV)
    kv = torch.randn(steps, 2, 2, n * most, heads, dim, device=DEV, generator=g).bfloat16()
    qs = torch.randn(steps, 2, n * most, heads * group, dim, device=DEV, generator=g).bfloat16()
    paths, counts = torch.zeros(steps, n, 6, dtype=torch.int32), torch.zeros(steps, n, dtype=torch.int32)
    for i in range(steps):
        for s in range(n):
            node, path = int(rng.integers(0, most)), []
            while node >= 0:
                path.insert(0, node)
                node = int(parents[i, s * most + node])
            path = path[:6]
            paths[i, s, :len(path)], counts[i, s] = torch.tensor(path, dtype=torch.int32), len(path)
    paths, counts = paths.to(DEV), counts.to(DEV)

    def begin():
        caches = [PagedKvCache.new(18, page_size, heads, dim, DEV, quantized) for _ in range(2)]
        lengths = torch.tensor(lengths0, dtype=torch.int32, device=DEV)
        for c, (k, v) in zip(caches, prefix):
            c.append_rotated(k, v, CacheBatch(table, lengths, first, sum(lengths0)), rotation)
        return caches, lengths

    def step(caches, lengths, up, rows, q_rows, path, count):
        lengths += most
        batch = CacheBatch(table, lengths, starts, n * most, most, 96)
        masks, positions = caches[0].tree_masks(up, batch)
        outs = []
        for c, (k, v), q in zip(caches, rows, q_rows):
            turned_q = c.append_rotated(k, v, batch, rotation, positions, q)
            outs.append((turned_q, c.tree_attention(turned_q, masks, batch)))
        caches[1].keep(path, count, batch)
        caches[0].keep(path, count, batch, out=lengths)
        return masks, outs

    caches, lengths = begin()
    eager = []
    for i in range(steps):
        held = [PagedKvCache(*(None if t is None else t.clone() for t in c._args())) for c in caches]
        at = lengths + most
        masks, outs = step(caches, lengths, parents[i], kv[i], qs[i], paths[i], counts[i])
        batch = CacheBatch(table, at, starts, n * most)
        for c, (k, v), (q, a) in zip(held, kv[i], outs):
            _, positions = c.tree_masks(parents[i], batch)
            c.append_rotated(k, v, batch, rotation, positions)
            ref, spread, reach = tree_reference(c, batch, q, masks, dim ** -0.5)
            off = np.abs(a.cpu().double().numpy() - ref)
            assert (off <= tolerance(ref, spread, reach, dim, 96, False, largest(c))).all()
        eager.append([a.clone() for _, a in outs])

    # the accepted tokens alone
    alone, at = begin()
    for i in range(steps):
        for s in range(n):
            for j in range(int(counts[i, s])):
                at[s] += 1
                one = torch.zeros(n + 1, dtype=torch.int32, device=DEV)
                one[s + 1:] = 1
                row = s * most + int(paths[i, s, j])
                for c, (k, v) in zip(alone, kv[i]):
                    c.append_rotated(k[row:row + 1], v[row:row + 1], CacheBatch(table, at, one, 1), rotation)
    assert torch.equal(at, lengths)
    for a, b in zip(caches, alone):
        for name in ("k", "v"):
            x, y = stored(a, name), stored(b, name)
            for s in range(n):
                t = np.arange(int(lengths[s]))
                page = table[s].cpu().numpy()[t // page_size]
                assert (x[page, :, t % page_size] == y[page, :, t % page_size]).all()

    caches, lengths = begin()
    ins = [t[0].clone() for t in (parents, kv, qs, paths, counts)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(caches, lengths, *ins)  # warm-up
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            _, outs = step(caches, lengths, *ins)
        fresh, _ = begin()
        for a, b in zip(caches, fresh):
            for x, y in zip(pools(a), pools(b)):
                x.copy_(y)
        lengths.copy_(torch.tensor(lengths0, dtype=torch.int32))
        for i in range(steps):
            for t, all_ in zip(ins, (parents, kv, qs, paths, counts)):
                t.copy_(all_[i])
            graph.replay()
            assert all(torch.equal(a, b) for (_, a), b in zip(outs, eager[i]))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(lengths, at)
