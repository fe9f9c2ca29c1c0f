"""A paged cache made for a test, and what attention over it is in 64 bits."""
import numpy as np
import torch

from unifur_b200.kv_cache import CacheBatch, PagedKvCache
from unifur_b200.quantize import nf4_levels

DEV = "cuda:0"


def batch_of(specs, page_size, spare_rows=(0, 0), spare_pages=2, width=None, seed=0, hints=True, device=DEV):
    """specs: (tokens in the cache, the call's rows) of each sequence -> (batch, number of pages); the pages lie anywhere in the
    pool, entries behind a sequence's pages name none."""
    rng = np.random.default_rng(seed)
    counts = [-(-length // page_size) for length, _ in specs]
    pages = sum(counts) + spare_pages
    order = rng.permutation(pages).astype(np.int32)
    table = np.full((len(specs), max([1, *counts]) if width is None else width), -1, np.int32)
    at = 0
    for i, n in enumerate(counts):
        table[i, :n] = order[at:at + n]
        at += n
    starts = np.cumsum([spare_rows[0]] + [n for _, n in specs]).astype(np.int32)
    rows = int(starts[-1]) + spare_rows[1]
    to = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(device)  # noqa: E731
    most = dict(max_rows=max(n for _, n in specs), max_length=max(n for n, _ in specs)) if hints else {}
    return CacheBatch(to(table), to(np.array([n for n, _ in specs], np.int32)), to(starts), rows, **most), pages


def filled_cache(pages, page_size, heads, dim, quantized, seed=0, k_std=1.0, v_std=1.0, device=DEV):
    """Every place of the pool holds something finite."""
    g = torch.Generator(device=device).manual_seed(seed)
    if not quantized:
        return PagedKvCache(*((torch.randn(pages, heads, page_size, dim, device=device, generator=g) * std).bfloat16()
                              for std in (k_std, v_std)))
    codes = [torch.randint(0, 256, (pages, heads, page_size, dim // 2), device=device, generator=g, dtype=torch.uint8) for _ in range(2)]
    scales = [(torch.rand(pages, heads, page_size, dim // 64, device=device, generator=g) + 0.5) * 2 * std for std in (k_std, v_std)]
    return PagedKvCache(*codes, *scales)


def spoil_unused(cache, batch):
    """NaNs in every place of the pool that no token of a sequence has (scales of a quantized cache)."""
    used = torch.zeros(cache.pages(), cache.page_size(), dtype=torch.bool)
    table, lengths = batch.page_table.cpu(), batch.lengths.cpu()
    for s in range(len(lengths)):
        for t in range(int(lengths[s])):
            used[int(table[s, t // cache.page_size()]), t % cache.page_size()] = True
    free = ~used.to(cache.k.device)[:, None, :, None]
    for t in (cache.k_scales, cache.v_scales) if cache.is_quantized() else (cache.k, cache.v):
        t.masked_fill_(free, float("nan"))


def stored(cache, name):
    """The pool's values in 64 bits, [pages, heads, page_size, dim] (numpy)."""
    pool = getattr(cache, name)
    if not cache.is_quantized():
        return pool.cpu().double().numpy()
    p = pool.cpu().numpy()
    codes = np.stack((p & 15, p >> 4), -1).reshape(*p.shape[:3], -1)
    scales = getattr(cache, name + "_scales").cpu().numpy()
    return nf4_levels().numpy().astype(np.float64)[codes] * np.repeat(scales.astype(np.float64), 64, -1)


def largest(cache):
    t = cache.v_scales if cache.is_quantized() else cache.v
    return float(torch.nan_to_num(t.float()).abs().max())


def tokens_of(values, batch, page_size, s):
    """A sequence's tokens [tokens, heads, dim] out of stored()."""
    length = int(batch.lengths[s])
    t = np.arange(length)
    page = batch.page_table[s].cpu().numpy()[t // page_size]
    return values[page, :, t % page_size]


def reference(cache, batch, q, scale):
    """out, sum of weights * |value| and the largest sum of |q * k| * scale of each row, in 64 bits; rows of no sequence: NaNs."""
    k_all, v_all = stored(cache, "k"), stored(cache, "v")
    q = q.cpu().double().numpy()
    out, spread, reach = (np.full(q.shape[:n], np.nan) for n in (3, 3, 2))
    starts = batch.row_starts.cpu().numpy()
    group = q.shape[1] // cache.heads()
    for s in range(len(starts) - 1):
        n, length = int(starts[s + 1] - starts[s]), int(batch.lengths[s])
        k, v = tokens_of(k_all, batch, cache.page_size(), s), tokens_of(v_all, batch, cache.page_size(), s)
        if n == 0:
            continue
        rows, see = slice(int(starts[s]), int(starts[s + 1])), length - n + np.arange(n) + 1
        hidden = np.arange(length) >= see[:, None]
        for h in range(q.shape[1]):
            kk, vv, qq = k[:, h // group], v[:, h // group], q[rows, h]
            x = np.where(hidden, -np.inf, scale * (qq @ kk.T))
            w = np.exp(x - np.maximum(x.max(1, initial=-np.inf, keepdims=True), -1e300))
            w /= np.maximum(w.sum(1, keepdims=True), 1e-300)
            out[rows, h], spread[rows, h] = w @ vv, w @ np.abs(vv)
            reach[rows, h] = np.where(hidden, 0, abs(scale) * (np.abs(qq) @ np.abs(kk).T)).max(1, initial=0)
    return out, spread, reach


def tolerance(out, spread, reach, dim, length, f32, high):
    """How far a result may be off.  Relative errors of the weights: twice the scores' errors (e^x), their own rounding, and the
    sums'; they move a result by as much of sum(weight * |value|); then the result is rounded.
    f32: sums of dim and length products, 2^-24 each.  bf16: keys and values enter as f16 (2^-11) or as they are, a query as it is, the
    weights as bf16 (2^-8) or f16; f32 sums beside that.  f16 is off by up to 2^-25 where a number is below 2^-14, which counts beside
    `high`, the largest scale (or value) of the cache: weights are kept 2^7 above their size in units of at most 2 high, so that a token
    is off by 2^-25 2^-7 2 high at most; values are in units of at most 2 high, off by 2^-25 of that."""
    out, reach = np.abs(out), reach[..., None]
    sums = 2.0 ** -24 * (2 * (dim + 4) * reach + 2 * length + 64)
    if f32:
        return 2.0 ** -24 * out + sums * spread
    return 2.0 ** -8 * out + (2 * 2 * 2.0 ** -11 * reach + 2.0 ** -8 + 2.0 ** -11 + sums) * spread * (1 + 2.0 ** -8) + \
        (length * 2.0 ** -31 + 2.0 ** -24) * high
