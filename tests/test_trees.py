"""What the entry points for trees of drafted tokens refuse, looked at without a GPU."""
import ctypes

import pytest

torch = pytest.importorskip("torch")
from test_kv_cache import BOTH, arguments, lib  # noqa: E402,F401


def rotation_of(**changed):
    from unifur_b200 import _lib

    r = _lib.RotationArgs()
    r.struct_bytes = ctypes.sizeof(r)
    r.rotary_dim, r.table_positions, r.table = 128, 100, 4096
    for name, value in changed.items():
        setattr(r, name, value)
    return r


def rotated(lib, cache, batch, rotation, k=4096, ldk=0, v=4096, ldv=0, q=4096, ldq=0, q_heads=28, out=8192, ldo=0, io=0):  # noqa: F811
    return lib.nf4_cache_append_rotated_dev(ctypes.byref(cache), ctypes.byref(batch), ctypes.byref(rotation) if rotation else None, k, ldk, v, ldv, q, ldq,
                                            q_heads, out, ldo, io, None), lib.nf4_last_error().decode()


@pytest.mark.parametrize("changed,status,word", BOTH)
def test_every_entry_point_refuses(lib, changed, status, word):  # noqa: F811
    cache, batch, args = arguments(**changed)
    refs = ctypes.byref(cache), ctypes.byref(batch)
    for call in (lambda: rotated(lib, cache, batch, rotation_of())[0], lambda: lib.nf4_cache_tree_dev(*refs, 4096, 4096, 1, 4096, None),
                 lambda: lib.nf4_cache_keep_dev(*refs, 4096, 4, 4096, 4096, None),
                 lambda: lib.nf4_cache_tree_attention_dev(*refs, 4096, 1, ctypes.byref(args), None)):
        assert call() == status and word in lib.nf4_last_error().decode()
    assert lib.nf4_cache_tree_attention_workspace_bytes(*refs, 28, 0) == 0


@pytest.mark.parametrize("changed,status,word", [
    ({"struct_bytes": 8}, -1, "struct_bytes"), ({"rotary_dim": 0}, -4, "rotary_dim"), ({"rotary_dim": 24}, -4, "rotary_dim"), ({"rotary_dim": 144}, -4, "rotary_dim"),
    ({"table": None}, -1, "table is null"), ({"table": 4104}, -1, "aligned"), ({"table_positions": 1 << 31}, -4, "2^31")])
def test_rotations_are_refused(lib, changed, status, word):  # noqa: F811
    cache, batch, _ = arguments()
    got, message = rotated(lib, cache, batch, rotation_of(**changed))
    assert got == status and word in message
    got, message = rotated(lib, cache, batch, None)
    assert got == -1 and "struct_bytes" in message


@pytest.mark.parametrize("changed,status,word", [
    ({"k": None}, -1, "k is null"), ({"v": 4100}, -1, "aligned"), ({"ldk": 100}, -1, "aligned"), ({"ldv": 504}, -1, "below"), ({"q": None}, -1, "q is null"),
    ({"out": None}, -1, "q_out is null"), ({"ldq": 3576}, -1, "below"), ({"q_heads": 1 << 16}, -4, "query heads"), ({"io": 3}, -1, "io_dtype"),
    ({"out": 4096, "ldo": 4096}, -1, "another row stride")])
def test_rows_to_rotate_are_refused(lib, changed, status, word):  # noqa: F811
    cache, batch, _ = arguments()
    got, message = rotated(lib, cache, batch, rotation_of(), **changed)
    assert got == status and word in message


def test_masks_and_paths_are_refused(lib):  # noqa: F811
    cache, batch, args = arguments()
    refs = ctypes.byref(cache), ctypes.byref(batch)
    assert lib.nf4_cache_tree_dev(*refs, None, 4096, 1, 4096, None) == -1 and b"parents" in lib.nf4_last_error()
    assert lib.nf4_cache_tree_dev(*refs, 4096, 4096, 1 << 27, 4096, None) == -4 and b"words" in lib.nf4_last_error()
    assert lib.nf4_cache_keep_dev(*refs, None, 4, 4096, 4096, None) == -1 and b"kept" in lib.nf4_last_error()
    assert lib.nf4_cache_keep_dev(*refs, 4096, 4, None, 4096, None) == -1 and b"counts" in lib.nf4_last_error()
    assert lib.nf4_cache_keep_dev(*refs, 4096, 1 << 31, 4096, 4096, None) == -4 and b"2^31" in lib.nf4_last_error()
    assert lib.nf4_cache_tree_attention_dev(*refs, None, 1, ctypes.byref(args), None) == -1 and b"masks" in lib.nf4_last_error()
    assert lib.nf4_cache_tree_attention_dev(*refs, 4096, 1 << 27, ctypes.byref(args), None) == -4 and b"words" in lib.nf4_last_error()


@pytest.mark.parametrize("changed,status,word", [
    ({"args__struct_bytes": 1}, -1, "struct_bytes"), ({"args__q_heads": 30}, -1, "query heads"), ({"args__scale": float("nan")}, -1, "scale"),
    ({"args__q": None}, -1, "q is null"), ({"args__ldo": 64}, -1, "below"), ({"args__io_dtype": 3}, -1, "io_dtype"),
    ({"args__workspace": None}, -1, "workspace"), ({"args__workspace_bytes": 100}, -1, "workspace"), ({"args__workspace": 4112}, -1, "256-byte")])
def test_attention_of_trees_refuses(lib, changed, status, word):  # noqa: F811
    cache, batch, args = arguments(**changed)
    assert lib.nf4_cache_tree_attention_dev(ctypes.byref(cache), ctypes.byref(batch), 4096, 1, ctypes.byref(args), None) == status
    assert word in lib.nf4_last_error().decode()


def test_nothing_to_do_is_no_error(lib):  # noqa: F811
    for changed in ({"batch__rows": 0}, {"batch__sequences": 0}):
        cache, batch, args = arguments(**changed)
        refs = ctypes.byref(cache), ctypes.byref(batch)
        assert rotated(lib, cache, batch, rotation_of(), k=None, v=None, q=None, out=None)[0] == 0
        assert lib.nf4_cache_tree_dev(*refs, None, None, 1, None, None) == 0
        assert lib.nf4_cache_tree_attention_dev(*refs, None, 0, ctypes.byref(args), None) == 0
    cache, batch, _ = arguments(batch__sequences=0)
    assert lib.nf4_cache_keep_dev(ctypes.byref(cache), ctypes.byref(batch), None, 0, None, None, None) == 0


def test_workspace_of_trees(lib):  # noqa: F811
    flags = lib.nf4_cache_attention_flag_bytes()
    for rows, length in ((1, 64), (2, 4096), (64, 4096), (512, 65536)):
        cache, batch, _ = arguments(batch__rows=rows, batch__max_length=length, batch__pages_per_sequence=1024)
        refs = ctypes.byref(cache), ctypes.byref(batch)
        for io in (0, 1):
            assert flags <= lib.nf4_cache_tree_attention_workspace_bytes(*refs, 28, io) < 1 << 31
            assert lib.nf4_cache_tree_attention_call_flag_bytes(*refs, 28, io) in ((0, flags) if io == 0 else (0,))


def test_host_tensors_and_unlike_ones_are_refused(lib):  # noqa: F811
    from unifur_b200 import _lib
    from unifur_b200.kv_cache import CacheBatch, PagedKvCache, Rotation

    cache = PagedKvCache.new(2, 16, 1, 64, "cpu")
    batch = CacheBatch(torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32), 1)
    x, words = torch.zeros(1, 64), torch.zeros(1, 1, dtype=torch.int32)
    _lib.host()
    for call in (lambda: cache.append_rotated(x, x, batch, Rotation.new(4, 64, "cpu")), lambda: cache.tree_masks(words[0], batch),
                 lambda: cache.tree_attention(x, words, batch), lambda: cache.keep(words, words[0], batch)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
