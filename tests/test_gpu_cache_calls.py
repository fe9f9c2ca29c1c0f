"""The cache's operators as a program calls them: rows inside larger tensors, padded batches, shared pages, graphs in turn, pools beyond 32 bits."""
import numpy as np
import pytest
import torch

from cache_util import DEV, batch_of, filled_cache, largest, reference, spoil_unused, tolerance
from unifur_b200 import _lib
from unifur_b200.kv_cache import CacheBatch, PagedKvCache

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def rows_of(batch, heads, dim, dtype=BF16, seed=7):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(batch.rows, heads, dim, device=DEV, generator=g).to(dtype)


def check(cache, batch, q, got, scale=None):
    """`got` against 64 bits; rows of no sequence are not looked at."""
    dim = q.shape[-1]
    ref, spread, reach = reference(cache, batch, q, dim ** -0.5 if scale is None else scale)
    real = ~np.isnan(ref)
    off = np.abs(got.cpu().double().numpy() - ref)
    limit = tolerance(ref, spread, reach, dim, int(batch.lengths.max()), q.dtype == F32, largest(cache))
    assert (off <= limit)[real].all(), np.nanmax(np.where(real, off / limit, 0))


# One row to a sequence, a chunk, f32: the three kernels.
@pytest.mark.parametrize("n,dtype", [(1, BF16), (70, BF16), (33, F32)])
@pytest.mark.parametrize("quantized", [True, False])
def test_rows_inside_a_larger_tensor(n, dtype, quantized):
    heads, group, dim = 2, 3, 128
    batch, pages = batch_of([(150, n), (n, n)], 32, spare_rows=(2, 3))
    whole = torch.randn(batch.rows, (group + 2) * heads * dim + 8, device=DEV).to(dtype)
    q, k, v = whole[:, :group * heads * dim], whole[:, group * heads * dim:(group + 1) * heads * dim], whole[:, -heads * dim:]
    caches = [filled_cache(pages, 32, heads, dim, quantized) for _ in range(2)]
    caches[0].append(k, v, batch)
    caches[1].append(k.contiguous().view(-1, heads, dim), v.contiguous(), batch)
    for name in ("k", "v", "k_scales", "v_scales"):
        a, b = (getattr(c, name) for c in caches)
        assert a is None or torch.equal(a, b)
    want = caches[0].attention(q.contiguous(), batch)
    wide = torch.full((batch.rows, group * heads * dim + 16), 7.0, device=DEV, dtype=dtype)
    out = wide[:, 8:-8]
    assert caches[0].attention(q, batch, out=out) is out
    assert torch.equal(out[2:-3], want[2:-3])
    assert (wide[:, :8] == 7).all() and (wide[:, -8:] == 7).all() and (out[:2] == 7).all() and (out[-3:] == 7).all()
    odd = torch.empty(q.numel() + 1, device=DEV, dtype=dtype)[1:].view(q.shape)  # not 16-byte aligned
    assert torch.equal(caches[0].attention(odd.copy_(q), batch)[2:-3], want[2:-3])
    dense = caches[0].read(batch, dtype)
    strided = [torch.full((batch.rows, heads, dim), 7.0, device=DEV, dtype=dtype) for _ in range(2)]
    caches[0].read(batch, dtype, strided)
    for a, b in zip(dense, strided):
        assert torch.equal(a[2:-3], b[2:-3]) and (b[:2] == 7).all() and (b[-3:] == 7).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("specs", [[(0, 0), (70, 3), (50, 0), (0, 2), (3, 5), (1, 1)], [(0, 0), (300, 90), (50, 0), (0, 40), (3, 100), (129, 129)]])
def test_sequences_without_rows_or_tokens(specs, quantized, dtype):
    """Empty sequences, and rows whose token is negative: they see nothing and become zeros, whatever the pool holds."""
    batch, pages = batch_of(specs, 16, spare_rows=(1, 2))
    cache = filled_cache(pages, 16, 2, 128, quantized)
    spoil_unused(cache, batch)
    q = rows_of(batch, 4, 128, dtype)
    out = torch.full_like(q, 7.0)
    cache.attention(q, batch, out=out)
    check(cache, batch, q, out)
    assert (out[:1] == 7).all() and (out[-2:] == 7).all()
    starts = batch.row_starts.tolist()
    for s, (length, n) in enumerate(specs):
        blind = out[starts[s]:starts[s] + max(0, n - length)]
        assert (blind == 0).all()


def test_nothing_to_do():
    cache = filled_cache(3, 16, 2, 64, True)
    before = [t.clone() for t in (cache.k, cache.v, cache.k_scales, cache.v_scales)]
    empty = lambda *s: torch.empty(*s, dtype=torch.int32, device=DEV)  # noqa: E731
    for batch in (CacheBatch(empty(0, 4), empty(0), torch.zeros(1, dtype=torch.int32, device=DEV), 0),
                  CacheBatch(empty(0, 0), empty(0), torch.zeros(1, dtype=torch.int32, device=DEV), 5),
                  CacheBatch(torch.zeros(2, 0, dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV),
                             torch.zeros(3, dtype=torch.int32, device=DEV), 0)):
        x = torch.zeros(batch.rows, 2, 64, device=DEV)
        cache.append(x, x, batch)
        assert cache.read(batch)[0].shape == x.shape and cache.attention(x, batch).shape == x.shape
    assert all(torch.equal(a, b) for a, b in zip(before, (cache.k, cache.v, cache.k_scales, cache.v_scales)))


def test_what_is_refused():
    batch, pages = batch_of([(20, 2)], 16)
    cache, q = filled_cache(pages, 16, 2, 64, True), torch.zeros(2, 4, 64, device=DEV)
    kv = q[:, :2]
    for call, word in ((lambda: cache.attention(q.half(), batch), "bf16 or f32"), (lambda: cache.attention(q[:, :3], batch), "multiple"),
                       (lambda: cache.attention(q[:1], batch), "must be"), (lambda: cache.attention(q.cpu(), batch), "device"),
                       (lambda: cache.attention(q, batch, out=q.bfloat16()), "shape and type"), (lambda: cache.attention(q, batch, float("nan")), "finite"),
                       (lambda: cache.attention(q, batch, out=torch.zeros(2, 4, 66, device=DEV)[..., :64]), "aligned"),
                       (lambda: cache.append(kv, kv.bfloat16(), batch), "one type"), (lambda: cache.append(q, kv, batch), "must be"),
                       (lambda: cache.read(batch, torch.float16), "bf16 or f32"),
                       (lambda: cache.read(batch, BF16, (kv, kv)), "dtype"),
                       (lambda: cache.append(kv, kv, CacheBatch(batch.page_table.long(), batch.lengths, batch.row_starts, 2)), "int32"),
                       (lambda: cache.append(kv, kv, CacheBatch(batch.page_table, batch.lengths, batch.row_starts[:1], 2)), "sequences"),
                       (lambda: PagedKvCache(cache.k.transpose(0, 1), cache.v, cache.k_scales, cache.v_scales).append(kv, kv, batch), "cache"),
                       (lambda: PagedKvCache(cache.k, cache.v).append(kv, kv, batch), "scales"),
                       (lambda: PagedKvCache.new(2, 24, 2, 64, DEV).append(kv, kv, batch), "page_size"),
                       (lambda: PagedKvCache.new(2, 16, 2, 192, DEV).append(torch.zeros(2, 2, 192, device=DEV), torch.zeros(2, 2, 192, device=DEV), batch), "head_dim")):
        with pytest.raises(Exception, match=word):
            call()
    torch.cuda.synchronize()


@pytest.mark.parametrize("n", [1, 50])
def test_shared_pages(n):
    """Two sequences with the same pages of a prefix get what they get with pages of their own."""
    batch, pages = batch_of([(96 + n, n), (96 + n, n)], 32)
    cache = filled_cache(pages, 32, 2, 128, True)
    q = rows_of(batch, 4, 128)
    table = batch.page_table.cpu()
    for pool in (cache.k, cache.v, cache.k_scales, cache.v_scales):
        pool[table[1, :3].long()] = pool[table[0, :3].long()]
    want = cache.attention(q, batch)
    table[1, :3] = table[0, :3]
    got = cache.attention(q, CacheBatch(table.to(DEV), batch.lengths, batch.row_starts, batch.rows, batch.max_rows, batch.max_length))
    assert torch.equal(got, want)


@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("page_size", [256, 4096])
@pytest.mark.parametrize("specs", [[(5000, 1), (300, 2)], [(5000, 200), (300, 30)]])
def test_large_pages(specs, page_size, quantized):
    batch, pages = batch_of(specs, page_size, spare_pages=0)
    cache = filled_cache(pages, page_size, 1, 64, quantized)
    q = rows_of(batch, 4, 64)
    check(cache, batch, q, cache.attention(q, batch))


@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("group,dim", [(80, 64), (65, 128), (33, 256)])
def test_many_query_heads_to_a_head(group, dim, quantized):
    batch, pages = batch_of([(400, 1), (77, 2)], 16)
    cache = filled_cache(pages, 16, 1, dim, quantized)
    q = rows_of(batch, group, dim)
    check(cache, batch, q, cache.attention(q, batch))


def test_graphs_in_turn():
    """A captured decode step and a captured chunk, replayed in turn with eager calls between, on one stream."""
    cases = []
    for specs in ([(900, 1), (4000, 1)], [(700, 300), (200, 64)]):
        batch, pages = batch_of(specs, 64)
        cache = filled_cache(pages, 64, 4, 128, True)
        q = rows_of(batch, 28, 128)
        cases.append((cache, batch, q, cache.attention(q, batch)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graphs = []
        for cache, batch, q, _ in cases:
            cache.attention(q, batch)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = cache.attention(q, batch)
            graphs.append((graph, out))
        for i in range(6):
            for (graph, out), (cache, batch, q, want) in zip(graphs, cases):
                out.zero_()
                graph.replay()
                assert torch.equal(cache.attention(q, batch), want) and torch.equal(out, want)
    torch.cuda.current_stream().wait_stream(side)


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
    for name in ("k", "v", "k_scales", "v_scales"):
        if getattr(small, name) is not None:
            getattr(big, name)[-12:] = getattr(small, name)
    for specs, dtype in (([(300, 1), (200, 3)], BF16), ([(300, 100), (200, 70)], BF16), ([(300, 40), (200, 9)], F32)):
        batch, _ = batch_of(specs, page_size, spare_pages=0)
        there = CacheBatch(torch.where(batch.page_table < 0, batch.page_table, batch.page_table + (pages - 12)), batch.lengths, batch.row_starts,
                           batch.rows, batch.max_rows, batch.max_length)
        k, v = (rows_of(batch, heads, dim, dtype, seed) for seed in (1, 2))
        small.append(k, v, batch)
        big.append(k, v, there)
        q = rows_of(batch, 2 * heads, dim, dtype)
        assert torch.equal(big.attention(q, there), small.attention(q, batch))
        assert all(torch.equal(a, b) for a, b in zip(big.read(there, dtype), small.read(batch, dtype)))


# ---- the kernel for many rows, which a wide page table without hints stands for (one launch more than the kernel that streams the cache, or two) ----

def wide(specs, page_size, tokens=1 << 16, **more):
    return batch_of(specs, page_size, width=tokens // page_size, hints=False, **more)


def many(cache, batch, q, **more):
    before = _lib.launch_count()
    out = cache.attention(q, batch, **more)
    assert _lib.launch_count() - before >= 2
    return out


CHUNKS = [[(130, 130)], [(300, 40), (65, 64), (1, 1)], [(1000, 129), (257, 257)], [(20, 33), (128, 128)], [(513, 300), (0, 7)]]


@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("heads,group,dim,page_size", [(2, 7, 128, 64), (1, 4, 64, 16), (1, 3, 256, 48), (2, 2, 128, 80)])
@pytest.mark.parametrize("specs", CHUNKS)
def test_many_rows(specs, heads, group, dim, page_size, quantized):
    batch, pages = wide(specs, page_size, tokens=1 << 20 if dim == 64 else page_size * 1024, spare_rows=(1, 2))
    cache = filled_cache(pages, page_size, heads, dim, quantized)
    spoil_unused(cache, batch)
    q = rows_of(batch, heads * group, dim)
    out = torch.full_like(q, 7.0)
    many(cache, batch, q, out=out)
    check(cache, batch, q, out)
    assert (out[:1] == 7).all() and (out[-2:] == 7).all()


@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("k_std,v_std,q_std,scale", [(1e4, 1.0, 1e-4, None), (1e-6, 1e6, 1e6, 0.1), (1.0, 1e-6, 1.0, 0.0), (1.0, 1.0, 1.0, -0.3), (1.0, 1.0, 30.0, None)])
@pytest.mark.parametrize("n", [70, 300])
def test_magnitudes_of_many_rows(n, quantized, k_std, v_std, q_std, scale):
    batch, pages = wide([(700, n)], 16, tokens=1 << 20)
    cache = filled_cache(pages, 16, 1, 128, quantized, k_std=k_std, v_std=v_std)
    q = (rows_of(batch, 2, 128, F32) * q_std).bfloat16()
    check(cache, batch, q, many(cache, batch, q, scale=scale), scale)


@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("n", [90, 600])
def test_many_rows_and_a_page_that_there_is_not(n, quantized):
    """That sequence's rows behind it are NaNs, another's are right."""
    batch, pages = wide([(700, n), (300, 64)], 16, tokens=1 << 20)
    cache = filled_cache(pages, 16, 2, 64, quantized)
    q = rows_of(batch, 4, 64)
    want = many(cache, batch, q)
    batch.page_table[0, 2] = pages
    got = many(cache, batch, q)
    assert got[:n].isnan().all() and torch.equal(got[n:], want[n:])


def test_more_tokens_than_the_hint_says():
    """The room for expanded keys and values follows the hint; with more tokens they are expanded where they are used."""
    batch, pages = batch_of([(3000, 700), (2000, 300)], 64)
    cache = filled_cache(pages, 64, 2, 128, True)
    q = rows_of(batch, 32, 128)
    batch.max_rows, batch.max_length = 100000, 100
    check(cache, batch, q, many(cache, batch, q))


@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("n,dim", [(40, 128), (9, 256), (300, 64)])
def test_both_kernels_agree(n, dim, quantized):
    """The same batch with a narrow and with a wide page table."""
    specs = [(700, n), (31, 3), (300, 1)]
    narrow, pages = batch_of(specs, 16)
    table = torch.full((3, 4096), -1, dtype=torch.int32, device=DEV)
    table[:, :narrow.page_table.shape[1]] = narrow.page_table
    cache = filled_cache(pages, 16, 1, dim, quantized)
    q = rows_of(narrow, 8, dim)
    for batch in (narrow, CacheBatch(table, narrow.lengths, narrow.row_starts, narrow.rows)):
        check(cache, batch, q, cache.attention(q, batch))
