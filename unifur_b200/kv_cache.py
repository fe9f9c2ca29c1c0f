"""The paged key and value cache of a decoder layer, quantized like the weights beside it, and the attention that reads it.

No counterpart on the reference's NF4 path: these are the operators between the projections that
``linear_forward_grouped`` makes of a layer's input and the one that takes the attention's result.  Every computation is a
call into ``libnf4b200.so``; ``torch`` holds the memory.  They serve: nothing here has a gradient.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import _lib
from .quantize import BLOCK_SIZE


class CacheBatch:
    """The sequences of a call and the rows of its tensors that belong to them.

    Rows ``row_starts[s]`` to ``row_starts[s + 1]`` are the newest tokens of sequence ``s``, which has ``lengths[s]`` tokens in
    the cache with them; token ``t`` is at place ``t % page_size`` of page ``page_table[s][t // page_size]``.  All three are
    int32 tensors on the cache's device (``[sequences, pages]``, ``[sequences]``, ``[sequences + 1]``); their values may change
    between replays of a captured graph.  ``rows``: rows of the call's tensors; those of no sequence are not written.
    ``max_rows``, ``max_length``: the most rows and tokens of a sequence where the program knows them; they choose kernels and
    how work is shared out, and results hold without them.  Sequences may share the pages of a common prefix, but a token that a
    call appends is in a page of its sequence alone."""

    __slots__ = ("page_table", "lengths", "row_starts", "rows", "max_rows", "max_length")

    def __init__(self, page_table: torch.Tensor, lengths: torch.Tensor, row_starts: torch.Tensor, rows: int,
                 max_rows: int = 0, max_length: int = 0):
        self.page_table, self.lengths, self.row_starts = page_table, lengths, row_starts
        self.rows, self.max_rows, self.max_length = rows, max_rows, max_length

    def _args(self) -> tuple:
        return (self.page_table, self.lengths, self.row_starts, self.rows, self.max_rows, self.max_length)


class PagedKvCache:
    """Keys and values in pages of ``page_size`` tokens (a multiple of 16).

    Quantized: ``k``, ``v`` uint8 ``[pages, heads, page_size, head_dim / 2]``, two NF4 codes to a byte, and an f32 scale for
    every 64 values of a row in ``k_scales``, ``v_scales`` ``[pages, heads, page_size, head_dim / 64]``, with the values that
    ``PackedNf4Tensor.quantize`` gives the rows.  Not quantized: bf16 ``[pages, heads, page_size, head_dim]`` without scales.
    ``head_dim`` is 64, 128 or 256."""

    __slots__ = ("k", "v", "k_scales", "v_scales")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scales: Optional[torch.Tensor] = None,
                 v_scales: Optional[torch.Tensor] = None):
        self.k, self.v, self.k_scales, self.v_scales = k, v, k_scales, v_scales

    @staticmethod
    def new(pages: int, page_size: int, heads: int, head_dim: int, device, quantized: bool = True) -> "PagedKvCache":
        def zeros(width, dtype):
            return torch.zeros(pages, heads, page_size, width, dtype=dtype, device=device)

        if not quantized:
            return PagedKvCache(zeros(head_dim, torch.bfloat16), zeros(head_dim, torch.bfloat16))
        return PagedKvCache(zeros(head_dim // 2, torch.uint8), zeros(head_dim // 2, torch.uint8),
                            zeros(head_dim // BLOCK_SIZE, torch.float32), zeros(head_dim // BLOCK_SIZE, torch.float32))

    def is_quantized(self) -> bool:
        return self.k.dtype == torch.uint8

    def pages(self) -> int:
        return self.k.shape[0]

    def heads(self) -> int:
        return self.k.shape[1]

    def page_size(self) -> int:
        return self.k.shape[2]

    def head_dim(self) -> int:
        return self.k.shape[3] * (2 if self.is_quantized() else 1)

    def resident_bytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.k_scales, self.v_scales) if t is not None)

    def _args(self) -> tuple:
        return (self.k, self.v, self.k_scales, self.v_scales)

    def append(self, k: torch.Tensor, v: torch.Tensor, batch: CacheBatch) -> None:
        """Writes the rows' keys and values (``[rows, heads, head_dim]`` or ``[rows, heads * head_dim]``, bf16 or f32, rows at any
        stride) to their places, quantized as they are written.  A row whose token is negative, or in a page that there is
        not, is not written."""
        _lib.host().cache_append(*self._args(), *batch._args(), k, v)

    def read(self, batch: CacheBatch, dtype: torch.dtype = torch.float32,
             out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """The rows' keys and values as the cache has them, ``[rows, heads, head_dim]`` in ``dtype`` (f32 or bf16).  Rows without a
        token in a page that there is are NaNs; rows of no sequence are left as ``out`` has them, and without ``out`` undefined."""
        k, v = out if out is not None else (None, None)
        return _lib.host().cache_read(*self._args(), *batch._args(), dtype, k, v)

    def attention(self, q: torch.Tensor, batch: CacheBatch, scale: Optional[float] = None,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Causal attention of the rows over the cache, which holds their own keys and values already:
        ``softmax(scale * q . k) v`` over each row's token and all before it.  ``q`` is ``[rows, q_heads, head_dim]`` or ``[rows,
        q_heads * head_dim]``, bf16 or f32, rows at any stride; ``q_heads`` is a multiple of the cache's heads, which serve
        neighbouring query heads.  ``scale`` is ``1 / sqrt(head_dim)`` if it is not given.  A row that sees nothing becomes
        zeros, one that sees a token in a page that there is not NaNs (others of its sequence may, too); rows of no sequence are left as ``out``
        has them, and without ``out`` undefined.  ``out`` does not overlap ``q``."""
        if scale is None:
            scale = 1.0 / math.sqrt(self.head_dim())
        return _lib.host().cache_attention(*self._args(), *batch._args(), q, scale, out)
