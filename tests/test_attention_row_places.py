"""The attention kernel for many rows: where its warps have queries and results in shared memory, by the library's own rule.  A warp writes its
next queries while another may still read its results out, with nothing between them: each warp's bytes have to be its own."""
import ctypes
import os
import re

import pytest

from unifur_b200 import _lib

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "unifur_b200", "csrc", "attention_chunk.cu")


def places(dim, warp, results):
    lib = _lib.load()
    got = [lib.nf4_cache_attention_row_place(dim, 32 * warp + lane, n, results) for lane in range(32) for n in range(dim // 8)]
    assert min(got) >= 0 and all(p % 16 == 0 for p in got) and len(set(got)) == len(got)
    return set(got)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_warps_keep_to_their_own_bytes(dim):
    queries, results = ([places(dim, warp, r) for warp in range(4)] for r in (0, 1))
    assert set().union(*queries) == set(range(0, 128 * dim * 2, 16))  # the whole tile
    for a in range(4):
        assert queries[a] == results[a]
        for b in range(a):
            assert not queries[a] & queries[b]


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_a_row_lies_as_the_mma_reads_it(dim):
    """Boxes of 128 rows of 128 bytes, the chunks of a row exchanged by the row's last three bits."""
    lib = _lib.load()
    for row in (0, 1, 6, 31, 32, 77, 127):
        for x in range(dim // 8):
            assert lib.nf4_cache_attention_row_place(dim, row, x, 1) == x // 8 * 16384 + row * 128 + ((x % 8) ^ (row % 8)) * 16


def test_chunks_come_in_the_order_of_memory():
    """32 neighbouring lanes bring 512 neighbouring bytes of rows of 128 values."""
    lib = _lib.load()
    first = [lib.nf4_cache_attention_row_place(128, 64 + lane, 0, 0) for lane in range(32)]
    assert first == [lib.nf4_cache_attention_row_place(128, 64 + lane // 16, lane % 16, 1) for lane in range(32)]


def test_no_wait_without_a_limit():
    """A warp whose wait ran out leaves its loop; nothing may wait for it there but the barrier of the whole CTA at the kernel's end."""
    with open(SOURCE) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    assert not re.search(r"\bbar\.sync|\bbarrier\.sync|__barrier_sync", text)


def test_refusals():
    lib = _lib.load()
    assert lib.nf4_cache_attention_row_place(96, 0, 0, 0) == -4 and b"head_dim" in ctypes.c_char_p(lib.nf4_last_error()).value
    assert lib.nf4_cache_attention_row_place(64, 128, 0, 0) == -1 and lib.nf4_cache_attention_row_place(64, 0, 8, 0) == -1
