"""Lengths beyond the page table, row starts beyond the call's rows and numbers below zero are cut to what there is: every operator gives what it gives for the cut
values, and writes nothing else.  (All of them go by one function that cuts, ahead of any address.)  And batches of unlike rows."""
import numpy as np
import pytest
import torch

from cache_util import DEV, batch_of, filled_cache, reference
from test_gpu_cache_sums import most_off, worst
from unifur_b200 import _lib
from unifur_b200.kv_cache import CacheBatch

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
MOST = 2 ** 31 - 1


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def both(rows_of_last):
    """A batch with values that have to be cut, and the same with the cut ones: a sequence longer than its table, one of no tokens whose length is below zero, one
    whose rows go on behind the tensor's last."""
    n = 3 + 2 + rows_of_last
    table = torch.randperm(3 * 4, device=DEV).to(torch.int32).view(3, 4)
    given = CacheBatch(table, ints(MOST, -7, 60), ints(-4, 3, 5, MOST), n, 64, 64)
    cut = CacheBatch(table, ints(64, 0, 60), ints(0, 3, 5, n), n, 64, 64)
    return given, cut


# attention of few rows, of many rows (a wide table without hints), of f32
@pytest.mark.parametrize("rows,dtype,wide", [(4, BF16, False), (50, BF16, True), (50, F32, False)])
@pytest.mark.parametrize("quantized", [True, False])
def test_what_is_cut(rows, dtype, wide, quantized):
    heads, group, dim = 2, 4, 128
    given, cut = both(rows)
    if wide:
        for b in (given, cut):
            table = torch.full((3, 4096), -1, dtype=torch.int32, device=DEV)
            table[:, :4] = b.page_table
            b.page_table, b.max_rows, b.max_length = table, 0, 0
        given.lengths, cut.lengths = ints(64, -7, 60), ints(64, 0, 60)  # (the table has room for 65536 tokens that it names no pages of)
    cache = filled_cache(12, 16, heads, dim, quantized)
    g = torch.Generator(device=DEV).manual_seed(3)
    q = torch.randn(cut.rows, heads * group, dim, device=DEV, generator=g).to(dtype)
    outs = []
    for b in (given, cut):
        whole = torch.full((cut.rows + 4, heads * group, dim), 7.0, device=DEV, dtype=dtype)
        before = _lib.launch_count()
        cache.attention(q, b, out=whole[2:-2])
        assert not wide or _lib.launch_count() - before >= 2
        assert (whole[:2] == 7).all() and (whole[-2:] == 7).all()
        outs.append(whole)
    assert torch.equal(*outs) and torch.isfinite(outs[0]).all()
    assert (outs[0][2 + 3:2 + 5] == 0).all()  # the rows of the sequence without tokens
    ref, _, _ = reference(cache, cut, q, dim ** -0.5)
    real = np.r_[0:3, 5:cut.rows]
    got = outs[0][2:-2].cpu().double().numpy()
    assert worst(got[real], ref[real]) <= most_off(cache, cut, q, dim ** -0.5, dim, 64, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("quantized", [True, False])
def test_append_and_read(dtype, quantized):
    given, cut = both(9)
    k, v = (torch.randn(cut.rows, 2, 64, device=DEV).to(dtype) for _ in range(2))
    caches, reads = [], []
    for b in (given, cut):
        cache = filled_cache(12, 16, 2, 64, quantized)
        cache.append(k, v, b)
        wholes = [torch.full((cut.rows + 4, 2, 64), 7.0, device=DEV, dtype=dtype) for _ in range(2)]
        cache.read(b, dtype, out=tuple(w[2:-2] for w in wholes))
        assert all((w[:2] == 7).all() and (w[-2:] == 7).all() for w in wholes)
        caches.append(cache)
        reads.append(wholes)
    for name in ("k", "v", "k_scales", "v_scales"):
        a, b = (getattr(c, name) for c in caches)
        assert a is None or torch.equal(a, b)
    for a, b in zip(*reads):
        assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(5.0), b.nan_to_num(5.0))
        assert torch.isnan(a[2 + 3:2 + 5]).all() and not torch.isnan(a[2:5]).any() and not torch.isnan(a[7:]).any()


# A prompt's chunk, or drafted tokens, beside many single tokens in one call.
@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("specs,dtype,launches", [
    ([(300 + 41 * i, 1) for i in range(31)] + [(2048, 2048)] + [(3000 - 90 * i, 1) for i in range(32)], BF16, 2),
    ([(40 + 100 * i, 1) for i in range(20)] + [(1500, 24), (90, 7)] + [(17 * i, 1) for i in range(20)], BF16, 1),
    ([(300 + 41 * i, 1) for i in range(20)] + [(700, 300)] + [(5, 5)], F32, None)])
def test_unlike_rows(specs, dtype, launches, quantized):
    batch, pages = batch_of(specs, 32)
    cache = filled_cache(pages, 32, 2, 128, quantized)
    g = torch.Generator(device=DEV).manual_seed(3)
    q = torch.randn(batch.rows, 8, 128, device=DEV, generator=g).to(dtype)
    before = _lib.launch_count()
    got = cache.attention(q, batch)
    taken = _lib.launch_count() - before
    assert launches is None or (taken == 1 if launches == 1 else taken >= 2)  # which kernel
    ref, _, _ = reference(cache, batch, q, 128 ** -0.5)
    some = np.linalg.norm(ref, axis=-1) > 0  # (a sequence of no tokens: zeros)
    got = got.cpu().double().numpy()
    assert (got[~some] == 0).all()
    assert worst(got[some], ref[some]) <= most_off(cache, batch, q, 128 ** -0.5, 128, 3000, dtype)
