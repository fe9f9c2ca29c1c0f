"""Page tables with room for far more tokens than are there: the kernel for many rows counts its steps in 32 bits, and calls that it could not count
for are the other kernel's."""
import ctypes

import numpy as np
import pytest
import torch

from unifur_b200 import _lib


def arguments(rows, pages_per_sequence, sequences=1, heads=16, dim=128):
    cache, batch = _lib.Cache(), _lib.CacheBatch()
    for s in (cache, batch):
        s.struct_bytes = ctypes.sizeof(s)
    cache.form, cache.num_pages, cache.page_size, cache.heads, cache.head_dim = _lib.CACHE_NF4, 8, 16, heads, dim
    cache.k = cache.v = cache.k_scales = cache.v_scales = 4096  # (never followed)
    batch.sequences, batch.page_table, batch.lengths, batch.row_starts = sequences, 4096, 4096, 4096
    batch.pages_per_sequence, batch.rows = pages_per_sequence, rows
    return cache, batch


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows,pages", [(1000, 1 << 26), (20000, 1 << 26), (1 << 20, 1 << 20), (1 << 23, 1 << 16)])
def test_the_queries_name_the_other_kernel(rows, pages, dim):
    lib = _lib.load()
    cache, batch = arguments(rows, pages, dim=dim)
    refs = ctypes.byref(cache), ctypes.byref(batch)
    flags = lib.nf4_cache_attention_flag_bytes()
    assert lib.nf4_cache_attention_call_flag_bytes(*refs, 128, 0) == flags
    # its workspace is a part of 16 rows to a CTA and twice that, however many rows there are
    assert lib.nf4_cache_attention_workspace_bytes(*refs, 128, 0) == flags + 2 * 148 * 16 * (dim + 2) * 4
    # with a table that is not as wide the rows are enough for the kernel for many
    cache, batch = arguments(1000, 1 << 12, dim=dim)
    assert lib.nf4_cache_attention_call_flag_bytes(ctypes.byref(cache), ctypes.byref(batch), 128, 0) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("quantized", [True, False])
def test_many_rows_and_a_table_of_a_billion_tokens(quantized):
    from cache_util import DEV, batch_of, filled_cache, largest, reference, tolerance

    narrow, pages = batch_of([(700, 600)], 16)
    cache = filled_cache(pages, 16, 16, 64, quantized)
    table = torch.full((1, 1 << 26), -1, dtype=torch.int32, device=DEV)
    table[:, :narrow.page_table.shape[1]] = narrow.page_table
    narrow.page_table, narrow.max_rows, narrow.max_length = table, 0, 0
    q = torch.randn(600, 128, 64, device=DEV).bfloat16()
    out = cache.attention(q, narrow)
    ref, spread, reach = reference(cache, narrow, q, 64 ** -0.5)
    assert (np.abs(out.cpu().double().numpy() - ref) <= tolerance(ref, spread, reach, 64, 700, False, largest(cache))).all()
