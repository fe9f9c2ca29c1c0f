"""Which kernel attention of trees takes."""
import ctypes

from unifur_b200 import _lib


def takes_the_kernel_for_many(cache, batch, q_heads):
    """Whether attention of bf16 nodes is the kernel's for many rows, as the library's question for a call's flags says (which that kernel has none of)."""
    c, b = _lib.Cache(), _lib.CacheBatch()
    for s in (c, b):
        s.struct_bytes = ctypes.sizeof(s)
    c.form, c.num_pages, c.page_size = _lib.CACHE_NF4 if cache.is_quantized() else _lib.CACHE_BF16, cache.pages(), cache.page_size()
    c.heads, c.head_dim = cache.heads(), cache.head_dim()
    c.k, c.v = cache.k.data_ptr(), cache.v.data_ptr()
    if cache.is_quantized():
        c.k_scales, c.v_scales = cache.k_scales.data_ptr(), cache.v_scales.data_ptr()
    b.sequences, b.pages_per_sequence, b.rows = *batch.page_table.shape, batch.rows
    b.page_table, b.lengths, b.row_starts = batch.page_table.data_ptr(), batch.lengths.data_ptr(), batch.row_starts.data_ptr()
    b.max_rows, b.max_length = batch.max_rows, batch.max_length
    return _lib.load().nf4_cache_tree_attention_call_flag_bytes(ctypes.byref(c), ctypes.byref(b), q_heads, 0) == 0
