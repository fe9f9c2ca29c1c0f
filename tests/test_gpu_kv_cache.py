"""The paged cache on the GPU: what append writes and read gives back, against the quantizer and the values themselves."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from cache_util import DEV, batch_of, filled_cache, stored  # noqa: E402
from gpu_util import bits_equal  # noqa: E402
from unifur_b200.kv_cache import CacheBatch, PagedKvCache  # noqa: E402
from unifur_b200.quantize import PackedNf4Tensor  # noqa: E402

SPECS = [
    [(1, 1)],
    [(200, 1), (0, 0), (17, 1), (16, 1)],
    [(333, 5), (64, 64), (1, 1), (3, 5)],      # the last has two rows before its first token
    [(700, 700)],
]


def places(specs, batch, page_size, first):
    """(row, page, place) of every row that has a token."""
    table, row, got = batch.page_table.cpu().numpy(), first, []
    for s, (length, new) in enumerate(specs):
        for i in range(new):
            t = length - new + i
            if t >= 0:
                got.append((row, int(table[s, t // page_size]), t % page_size))
            row += 1
    return got


@pytest.mark.parametrize("heads,dim,page_size", [(4, 128, 64), (3, 64, 48), (2, 256, 16)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("specs", SPECS)
def test_append_writes_what_the_quantizer_gives_and_nothing_else(specs, quantized, dtype, heads, dim, page_size):
    batch, pages = batch_of(specs, page_size, spare_rows=(2, 3))
    cache = filled_cache(pages, page_size, heads, dim, quantized, seed=1)
    before = [t.clone() for t in (cache.k, cache.v, cache.k_scales, cache.v_scales) if t is not None]
    g = torch.Generator(device=DEV).manual_seed(2)
    wide = torch.randn(batch.rows, 2 * heads * dim + 16, device=DEV, generator=g).to(dtype)
    wide[:, 8] = 0.0
    wide[0:1, 24:88] = 0.0
    k, v = wide[:, 8:8 + heads * dim], wide[:, 16 + heads * dim:].unflatten(1, (heads, dim))  # rows of a wider tensor
    cache.append(k, v, batch)
    where = places(specs, batch, page_size, 2)
    touched = torch.zeros(pages, page_size, dtype=torch.bool, device=DEV)
    for row, page, place in where:
        touched[page, place] = True
    assert len(where) == int(touched.sum())
    now = [t for t in (cache.k, cache.v, cache.k_scales, cache.v_scales) if t is not None]
    for was, is_ in zip(before, now):
        keep = ~touched[:, None, :, None].expand_as(is_)
        assert torch.equal(was[keep], is_[keep])
    for name, x in (("k", k.unflatten(1, (heads, dim))), ("v", v)):
        for row, page, place in where:
            values = x[row].contiguous()
            if quantized:
                p = PackedNf4Tensor.quantize(values.float().flatten())
                assert torch.equal(getattr(cache, name)[page, :, place].flatten(), p.codes)
                assert torch.equal(getattr(cache, name + "_scales")[page, :, place].flatten(), p.absmax)
            else:
                assert torch.equal(getattr(cache, name)[page, :, place], values.bfloat16())
    # and back
    for out_type in (torch.float32, torch.bfloat16):
        back = [torch.full((batch.rows, heads, dim), 7.0, device=DEV, dtype=out_type) for _ in range(2)]
        got = cache.read(batch, out_type, out=tuple(back))
        assert got[0].data_ptr() == back[0].data_ptr()
        rows = {row for row, _, _ in where}
        for name, t in zip(("k", "v"), got):
            values = torch.from_numpy(stored(cache, name).astype(np.float32)).to(DEV)  # (a product of two f32, rounded once)
            for row, page, place in where:
                assert torch.equal(t[row], values[page, :, place].to(out_type))
            for row in range(batch.rows):
                in_sequence = 2 <= row < batch.rows - 3
                if row not in rows:
                    assert bool(torch.isnan(t[row]).all() if in_sequence else (t[row] == 7.0).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_blocks_of_any_content_are_quantized_as_the_reference_does(oracle, dtype):
    """Zeros, NaNs, infinities, subnormals, values next to the ends of a type's range."""
    heads, dim, page_size = 2, 128, 16
    rng = np.random.default_rng(4)
    x = rng.standard_normal((32, heads * dim)).astype(np.float32)
    x[1] = 0.0
    x[2, ::3] = np.nan
    x[3, 5] = np.inf
    x[4, 70] = -np.inf
    x[5] *= 1e-38
    x[6] *= 3e-45
    x[7] *= 1e38
    x[8] = -0.0
    x[9] *= 1e-31
    x[10] = np.nan
    t = torch.from_numpy(x).to(DEV).to(dtype)
    batch, pages = batch_of([(32, 32)], page_size)
    cache = PagedKvCache.new(pages, page_size, heads, dim, DEV)
    cache.append(t, t, batch)
    packed, absmax = oracle.quantize_packed(t.float().cpu().numpy())
    table = batch.page_table[0, :2].long()
    for codes, scales in ((cache.k, cache.k_scales), (cache.v, cache.v_scales)):
        assert codes[table].transpose(1, 2).cpu().numpy().tobytes() == packed.tobytes()
        assert bits_equal(scales[table].transpose(1, 2).contiguous().cpu().numpy().ravel(), absmax.ravel())


def test_places_that_there_are_not():
    """Pages outside the pool and lengths beyond the table: nothing is written, reading gives NaNs."""
    heads, dim, page_size = 2, 64, 16
    batch, pages = batch_of([(40, 40), (20, 20)], page_size)
    batch.page_table[0, 1], batch.page_table[1, 0] = -3, pages
    cache = filled_cache(pages, page_size, heads, dim, True)
    before = [t.clone() for t in (cache.k, cache.v)]
    x = torch.randn(60, heads, dim, device=DEV)
    cache.append(x, x, batch)
    k, v = cache.read(batch)
    gone = list(range(16, 32)) + list(range(40, 56))
    kept = [r for r in range(60) if r not in gone]
    for t in (k, v):
        assert bool(torch.isnan(t[gone]).all()) and not bool(torch.isnan(t[kept]).any())
    changed = sum(int((a != b).flatten(3).any(-1).any(1).sum()) for a, b in zip(before, (cache.k, cache.v)))
    assert changed <= 2 * len(kept)
    # a length beyond the table's pages is cut there, rows beyond the tensors too
    far = CacheBatch(batch.page_table, torch.tensor([1000, 20], dtype=torch.int32, device=DEV),
                     torch.tensor([0, 40, 5000], dtype=torch.int32, device=DEV), 60)
    cache.append(x, x, far)
    torch.cuda.synchronize()


def test_many_sequences_and_empty_ones():
    heads, dim, page_size = 1, 64, 16
    rng = np.random.default_rng(5)
    specs = [(int(n), int(min(n, k))) for n, k in zip(rng.integers(0, 60, 700), rng.integers(0, 4, 700))]
    batch, pages = batch_of(specs, page_size, spare_rows=(1, 1))
    cache = PagedKvCache.new(pages, page_size, heads, dim, DEV, quantized=False)
    x = torch.randn(batch.rows, heads, dim, device=DEV).bfloat16()
    cache.append(x, -x, batch)
    k, v = cache.read(batch, torch.bfloat16)
    assert torch.equal(k[1:-1], x[1:-1]) and torch.equal(v[1:-1], -x[1:-1])
