"""What the cache's entry points refuse, looked at without a GPU: every argument is checked before anything is launched."""
import ctypes

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def lib():
    from unifur_b200 import build

    build.build()
    from unifur_b200 import _lib

    return _lib.load()


def arguments(**changed):
    """A call that holds together as far as the host can see (the addresses are never followed), with what is changed."""
    from unifur_b200 import _lib

    cache, batch, args = _lib.Cache(), _lib.CacheBatch(), _lib.AttentionArgs()
    for s in (cache, batch, args):
        s.struct_bytes = ctypes.sizeof(s)
    cache.form, cache.num_pages, cache.page_size, cache.heads, cache.head_dim = _lib.CACHE_NF4, 8, 64, 4, 128
    cache.k = cache.v = cache.k_scales = cache.v_scales = 4096
    batch.sequences, batch.page_table, batch.lengths, batch.row_starts = 2, 4096, 4096, 4096
    batch.pages_per_sequence, batch.rows = 4, 2
    args.io_dtype, args.q_heads, args.scale, args.q, args.out, args.workspace, args.workspace_bytes = 0, 28, 0.1, 4096, 4096, 4096, 1 << 40
    for name, value in changed.items():
        target, field = name.split("__")
        setattr({"cache": cache, "batch": batch, "args": args}[target], field, value)
    return cache, batch, args


def attention(lib, **changed):
    cache, batch, args = arguments(**changed)
    return lib.nf4_cache_attention_dev(ctypes.byref(cache), ctypes.byref(batch), ctypes.byref(args), None), lib.nf4_last_error().decode()


BOTH = [
    ({"cache__struct_bytes": 8}, -1, "struct_bytes"), ({"batch__struct_bytes": 8}, -1, "struct_bytes"),
    ({"cache__form": 2}, -1, "form"), ({"cache__head_dim": 192}, -4, "head_dim"), ({"cache__head_dim": 0}, -4, "head_dim"),
    ({"cache__page_size": 0}, -4, "page_size"), ({"cache__page_size": 24}, -4, "page_size"), ({"cache__page_size": 1 << 17}, -4, "page_size"),
    ({"cache__heads": 0}, -4, "heads"), ({"cache__num_pages": 0}, -4, "pool"), ({"cache__num_pages": 1 << 30}, -4, "pool"),
    ({"cache__k": None}, -1, "null"), ({"cache__v_scales": None}, -1, "null"), ({"cache__v": 4104}, -1, "aligned"),
    ({"batch__sequences": 1 << 16}, -4, "sequences"), ({"batch__lengths": None}, -1, "null"), ({"batch__page_table": None}, -1, "null"),
    ({"batch__pages_per_sequence": 1 << 26}, -4, "2^31"), ({"batch__rows": 1 << 31}, -4, "2^31"),
]


@pytest.mark.parametrize("changed,status,word", BOTH)
def test_every_entry_point_refuses(lib, changed, status, word):
    cache, batch, _ = arguments(**changed)
    for call in (lib.nf4_cache_append_dev, lib.nf4_cache_read_dev):
        assert call(ctypes.byref(cache), ctypes.byref(batch), 4096, 0, 4096, 0, 0, None) == status
        assert word in lib.nf4_last_error().decode()
    got, message = attention(lib, **changed)
    assert got == status and word in message
    assert lib.nf4_cache_attention_workspace_bytes(ctypes.byref(cache), ctypes.byref(batch), 28, 0) == 0


@pytest.mark.parametrize("call", ["nf4_cache_append_dev", "nf4_cache_read_dev"])
@pytest.mark.parametrize("k,ldk,io,status,word", [(None, 0, 0, -1, "null"), (4104, 0, 0, -1, "aligned"), (4096, 516, 0, -1, "aligned"),
                                                  (4096, 504, 0, -1, "below"), (4096, 0, 7, -1, "io_dtype"), (4096, 1 << 41, 0, -4, "large")])
def test_rows_are_refused(lib, call, k, ldk, io, status, word):
    cache, batch, _ = arguments()
    for args in ((k, ldk, 4096, 0), (4096, 0, k, ldk)):
        assert getattr(lib, call)(ctypes.byref(cache), ctypes.byref(batch), *args, io, None) == status
        assert word in lib.nf4_last_error().decode()


@pytest.mark.parametrize("changed,status,word", [
    ({"args__struct_bytes": 1}, -1, "struct_bytes"), ({"args__q_heads": 0}, -1, "query heads"), ({"args__q_heads": 30}, -1, "query heads"),
    ({"args__q_heads": 1 << 17}, -4, "heads"), ({"args__scale": float("inf")}, -1, "scale"), ({"args__scale": float("nan")}, -1, "scale"),
    ({"args__q": None}, -1, "q is null"), ({"args__out": 4097}, -1, "out"), ({"args__ldo": 64}, -1, "below"), ({"args__io_dtype": 3}, -1, "io_dtype"),
    ({"args__workspace": None}, -1, "workspace"), ({"args__workspace_bytes": 100}, -1, "workspace"), ({"args__workspace": 4112}, -1, "256-byte"),
])
def test_attention_refuses(lib, changed, status, word):
    got, message = attention(lib, **changed)
    assert got == status and word in message, message


def test_nothing_to_do_is_no_error(lib):
    for changed in ({"batch__rows": 0}, {"batch__sequences": 0}):
        cache, batch, args = arguments(**changed)
        args.q = args.out = None if "batch__rows" in changed else 4096
        refs = ctypes.byref(cache), ctypes.byref(batch)
        assert lib.nf4_cache_append_dev(*refs, 4096, 0, 4096, 0, 0, None) == 0
        assert lib.nf4_cache_read_dev(*refs, 4096, 0, 4096, 0, 0, None) == 0
        assert lib.nf4_cache_attention_dev(*refs, ctypes.byref(args), None) == 0


def test_workspace_grows_with_the_call_and_holds_the_flags(lib):
    assert lib.nf4_cache_attention_flag_bytes() % 256 == 0
    sizes = []
    for rows, length in ((1, 64), (2, 4096), (64, 4096)):
        cache, batch, _ = arguments(batch__rows=rows, batch__max_length=length, batch__pages_per_sequence=64)
        for io in (0, 1):
            sizes.append(lib.nf4_cache_attention_workspace_bytes(ctypes.byref(cache), ctypes.byref(batch), 28, io))
    assert all(s >= lib.nf4_cache_attention_flag_bytes() for s in sizes)
    assert max(sizes) < 1 << 30


def test_flags_that_a_call_relies_on(lib):
    """Those of the kernel that streams the cache, which single tokens and short contexts take in bf16; none with f32 tensors."""
    def flags(io, **changed):
        cache, batch, _ = arguments(batch__pages_per_sequence=1024, **changed)
        return lib.nf4_cache_attention_call_flag_bytes(ctypes.byref(cache), ctypes.byref(batch), 28, io)

    most = lib.nf4_cache_attention_flag_bytes()
    assert flags(0, batch__rows=1) == most and flags(0, batch__rows=300, batch__max_length=128) == most
    assert flags(0, batch__rows=4000, batch__max_length=16384) == 0
    assert flags(1, batch__rows=1) == 0
    assert flags(0, batch__rows=1, cache__page_size=24) == most  # (refused by the call itself)


def test_host_tensors_are_refused(lib):
    from unifur_b200 import _lib
    from unifur_b200.kv_cache import CacheBatch, PagedKvCache

    cache = PagedKvCache.new(2, 16, 1, 64, "cpu")
    assert cache.is_quantized() and cache.head_dim() == 64 and cache.page_size() == 16 and cache.heads() == 1 and cache.pages() == 2
    assert cache.resident_bytes() == 2 * 2 * 16 * (32 + 4)
    batch = CacheBatch(torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32), 1)
    x = torch.zeros(1, 64)
    _lib.host()
    for call in (lambda: cache.append(x, x, batch), lambda: cache.read(batch), lambda: cache.attention(x, batch)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
