"""Attention over the paged cache against 64 bits, and the operators of a decode step together."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from cache_util import DEV, batch_of, filled_cache, largest, reference, spoil_unused, tolerance  # noqa: E402
from unifur_b200 import _lib  # noqa: E402
from unifur_b200.kv_cache import CacheBatch, PagedKvCache  # noqa: E402

# (tokens in the cache, the call's rows) of each sequence
ONE = [[(1, 1)], [(15, 1)], [(16, 1), (17, 1)], [(200, 1), (0, 0), (1, 1), (333, 1)], [(0, 1), (64, 1)], [(2100, 1), (50, 1)]]
FEW = [[(9, 2), (100, 3)], [(700, 5), (6, 6), (30, 1)], [(3, 5), (260, 8)]]      # (3, 5): two rows see nothing
CHUNKS = [[(130, 130)], [(300, 40), (65, 64), (1, 1)], [(1000, 129), (257, 257)], [(20, 33), (128, 128)], [(513, 300), (0, 7)]]


def check(specs, heads, group, dim, page_size, quantized, dtype, seed=0, hints=True, scale=None, k_std=1.0, v_std=1.0, q_std=1.0):
    batch, pages = batch_of(specs, page_size, spare_rows=(1, 2), seed=seed, hints=hints)
    cache = filled_cache(pages, page_size, heads, dim, quantized, seed=seed + 1, k_std=k_std, v_std=v_std)
    spoil_unused(cache, batch)
    g = torch.Generator(device=DEV).manual_seed(seed + 2)
    wide = (torch.randn(batch.rows, heads * group * dim + 24, device=DEV, generator=g) * q_std).to(dtype)
    q = wide[:, 16:16 + heads * group * dim].unflatten(1, (heads * group, dim))
    out = torch.full((batch.rows, heads * group, dim), 7.0, device=DEV, dtype=dtype)
    got = cache.attention(q, batch, scale, out=out)
    assert got.data_ptr() == out.data_ptr()
    ref, spread, reach = reference(cache, batch, q, dim ** -0.5 if scale is None else scale)
    rows = slice(1, batch.rows - 2)
    assert bool((out[:1] == 7.0).all()) and bool((out[-2:] == 7.0).all()), "rows of no sequence were written"
    off = np.abs(out[rows].cpu().double().numpy() - ref[rows])
    may = tolerance(ref[rows], spread[rows], reach[rows], dim, max(n for n, _ in specs), dtype == torch.float32, largest(cache))
    worst = float((off / np.maximum(may, 1e-300)).max())
    assert worst <= 1, f"off by {float(off.max())}, {worst} of what it may be"
    assert _lib.load().nf4_device_status(None, None, None) == 0
    return cache, batch, q, got


@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("heads,group,dim,page_size", [(4, 7, 128, 64), (2, 4, 64, 16), (1, 8, 256, 48), (3, 1, 128, 32), (2, 16, 64, 128), (2, 4, 128, 48)])
@pytest.mark.parametrize("specs", ONE + FEW)
def test_few_rows(specs, heads, group, dim, page_size, quantized):
    check(specs, heads, group, dim, page_size, quantized, torch.bfloat16)


@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("heads,group,dim,page_size", [(2, 7, 128, 64), (1, 4, 64, 16), (1, 3, 256, 48), (2, 1, 128, 80)])
@pytest.mark.parametrize("specs", CHUNKS)
def test_chunks(specs, heads, group, dim, page_size, quantized):
    check(specs, heads, group, dim, page_size, quantized, torch.bfloat16)


@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("heads,group,dim,page_size", [(2, 3, 128, 64), (1, 5, 64, 16), (1, 2, 256, 48)])
@pytest.mark.parametrize("specs", [ONE[3], ONE[5], FEW[1], FEW[2], CHUNKS[1], CHUNKS[3]])
def test_f32(specs, heads, group, dim, page_size, quantized):
    check(specs, heads, group, dim, page_size, quantized, torch.float32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("specs", [[(200, 1), (5000, 1)], [(90, 20), (300, 1), (40, 40)]])
def test_without_hints(specs, dtype):
    check(specs, 2, 4, 128, 32, True, dtype, hints=False)


@pytest.mark.parametrize("hint", [(1, 1), (3, 100000), (1000, 16)])
def test_wrong_hints_change_no_result(hint):
    specs = [(300, 70), (900, 1), (64, 64)]
    cache, batch, q, right = check(specs, 2, 4, 128, 32, True, torch.bfloat16)
    wrong = CacheBatch(batch.page_table, batch.lengths, batch.row_starts, batch.rows, *hint)
    out = cache.attention(q, wrong)[1:-2].double()
    right = right[1:-2].double()
    assert float((out - right).norm() / right.norm()) < 2.0 ** -7


@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("specs", [[(3000, 1)], [(700, 40)]])
@pytest.mark.parametrize("k_std,v_std,q_std,scale", [(1e4, 1.0, 1e-4, None), (1e-6, 1e6, 1e6, 0.1), (1.0, 1e-6, 1.0, 0.0), (1.0, 1.0, 1.0, -0.3),
                                                     (3e5, 3e5, 1e-5, 0.05), (1.0, 1.0, 30.0, None)])
def test_magnitudes(specs, quantized, k_std, v_std, q_std, scale):
    """Keys, values and queries outside f16's range; scores all alike; a scale below zero; sharp scores."""
    check(specs, 1, 4, 128, 64, quantized, torch.bfloat16, k_std=k_std, v_std=v_std, q_std=q_std, scale=scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [1, 90])
def test_a_page_that_there_is_not(dtype, rows):
    specs = [(200, rows), (300, rows)]
    batch, pages = batch_of(specs, 32)
    cache = filled_cache(pages, 32, 2, 128, True)
    batch.page_table[0, 1] = pages + 5
    q = torch.randn(batch.rows, 8, 128, device=DEV).to(dtype)
    out = cache.attention(q, batch)
    assert bool(torch.isnan(out[:rows]).all()) and bool(torch.isfinite(out[rows:]).all())


def test_results_are_the_same_every_time():
    specs = [(5000, 1), (700, 2), (64, 1), (3000, 1)]
    batch, pages = batch_of(specs, 64)
    cache = filled_cache(pages, 64, 4, 128, True)
    q = torch.randn(batch.rows, 28, 128, device=DEV).bfloat16()
    first = cache.attention(q, batch)
    for _ in range(20):
        assert torch.equal(cache.attention(q, batch), first)


def test_decode_steps_in_a_graph_and_beside_it(oracle):
    """Projections, append, attention and the output projection of a decoder layer: steps run one by one, and replays of one
    captured step whose lengths and rows change in place, give the same; each step is the 64-bit result of what is cached."""
    from unifur_b200._lib import LAYOUT_OUT_IN
    from unifur_b200.quantize import PackedNf4Tensor, linear_forward, linear_forward_grouped

    hidden, heads, group, dim, page_size, n = 512, 2, 2, 128, 16, 3
    g = torch.Generator(device=DEV).manual_seed(3)
    pack = lambda *s: PackedNf4Tensor.quantize((torch.randn(*s, device=DEV, generator=g) * 0.05).flatten())  # noqa: E731
    wq, wk, wv, wo = pack(heads * group * dim, hidden), pack(heads * dim, hidden), pack(heads * dim, hidden), pack(hidden, heads * group * dim)
    lengths0 = [15, 1, 40]
    table = torch.randperm(12, device=DEV, generator=g).to(torch.int32).view(n, 4)
    prefix = torch.randn(sum(lengths0), 2, heads * dim, device=DEV, generator=g).bfloat16()
    xs = torch.randn(6, n, hidden, device=DEV, generator=g).bfloat16()

    def begin():
        cache = PagedKvCache.new(12, page_size, heads, dim, DEV)
        lengths = torch.tensor(lengths0, dtype=torch.int32, device=DEV)
        starts = torch.tensor(np.cumsum([0] + lengths0), dtype=torch.int32, device=DEV)
        cache.append(prefix[:, 0], prefix[:, 1], CacheBatch(table, lengths, starts, sum(lengths0)))
        return cache, lengths

    starts = torch.arange(n + 1, dtype=torch.int32, device=DEV)

    def step(cache, lengths, x):
        lengths += 1
        batch = CacheBatch(table, lengths, starts, n, 1, 64)
        q, k, v = linear_forward_grouped(x, hidden, LAYOUT_OUT_IN, [{"packed": wq, "d_out": heads * group * dim}, {"packed": wk, "d_out": heads * dim},
                                                                    {"packed": wv, "d_out": heads * dim}])
        cache.append(k, v, batch)
        a = cache.attention(q, batch)
        return q, a, linear_forward(a, wo, heads * group * dim, hidden, LAYOUT_OUT_IN)

    cache, lengths = begin()
    eager = []
    for x in xs:
        q, a, y = step(cache, lengths, x)
        eager.append((a.clone(), y.clone()))
        ref, spread, reach = reference(cache, CacheBatch(table, lengths, starts, n), q.view(n, heads * group, dim), dim ** -0.5)
        off = np.abs(a.view(n, heads * group, dim).cpu().double().numpy() - ref)
        assert (off <= tolerance(ref, spread, reach, dim, 64, False, largest(cache))).all()

    cache, lengths = begin()
    x = xs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(cache, lengths, x)          # warm-up
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            _, a, y = step(cache, lengths, x)
        lengths.copy_(torch.tensor(lengths0, dtype=torch.int32))
        for i in range(len(xs)):
            x.copy_(xs[i])
            graph.replay()
            assert torch.equal(a, eager[i][0]) and torch.equal(y, eager[i][1])
    torch.cuda.current_stream().wait_stream(side)


def test_two_streams_at_once():
    specs = [(4000, 1), (900, 1)]
    batch, pages = batch_of(specs, 64)
    cache = filled_cache(pages, 64, 4, 128, True)
    q = torch.randn(batch.rows, 28, 128, device=DEV).bfloat16()
    want = cache.attention(q, batch)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for i in range(20):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(cache.attention(q, batch))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
