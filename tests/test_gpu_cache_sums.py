"""Attention over long sequences, every token counted once: limits on whole rows, which a unit of sixteen or 32 tokens left out or taken twice
exceeds, and values that say which tokens they are of."""
import numpy as np
import pytest
import torch

from cache_util import batch_of, filled_cache, reference, stored, tokens_of

F32, BF16 = torch.float32, torch.bfloat16


def most_off(cache, batch, q, scale, dim, length, dtype):
    """How far a row may be off in norm, relative to its own.  bf16: the result's rounding, 2^-8, and as much for the weights', which are independent from
    token to token, so that their parts add up as the tokens' own do (random values: to the row's norm).  A score is off by half steps of 2^-11 of its
    products (three of a key), independent too: 2^-11 sqrt(3) of the root of the sum of their squares in the mean, twice that for numerator
    and denominator, and twice that for the spread.  f32: sums of dim products and of length weights, half steps of 2^-24."""
    if dtype == F32:
        return 2.0 ** -24 * (dim + 4 * length ** 0.5 + 32)
    q, k = q.cpu().double().numpy(), cache.k
    size = float(cache.k_scales.float().nan_to_num().square().mean()) ** 0.5 if cache.is_quantized() else float(k.float().nan_to_num().square().mean()) ** 0.5
    return 2 * 2.0 ** -8 + 4 * 3 ** 0.5 * 2.0 ** -11 * abs(scale) * size * float(np.sqrt((q ** 2).sum(-1)).max())


def inputs(specs, heads, group, dim, quantized, dtype, q_std, device, page_size=64, wide=False):
    batch, pages = batch_of(specs, page_size, device=device, **(dict(width=65536 // page_size, hints=False) if wide else {}))
    cache = filled_cache(pages, page_size, heads, dim, quantized, device=device)
    g = torch.Generator(device=device).manual_seed(11)
    q = (torch.randn(batch.rows, heads * group, dim, device=device, generator=g) * q_std).to(dtype)
    return cache, batch, q


def worst(got, ref):
    """The largest error of a row in norm, relative to the row's."""
    return float((np.linalg.norm(got - ref, axis=-1) / np.linalg.norm(ref, axis=-1)).max())


# ---- on the CPU: what the limit sees --------------------------------------------------------------


@pytest.mark.parametrize("length,lost,q_std", [(2100, 32, 1.0), (5000, 128, 1.0), (3000, 16, 30.0), (4000, 32, 1.0)])
def test_the_limit_sees_a_unit_left_out(length, lost, q_std):
    """Mistakes planted in the 64-bit side: tokens left out, tokens taken twice, a part joined by a wrong factor."""
    cache, batch, q = inputs([(length, 1)], 2, 4, 128, True, BF16, q_std, "cpu")
    scale = 128 ** -0.5
    ref, _, _ = reference(cache, batch, q, scale)
    limit = most_off(cache, batch, q, scale, 128, length, BF16)
    k, v = (tokens_of(stored(cache, name), batch, 64, 0) for name in ("k", "v"))
    x = np.einsum("hgd,thd->hgt", q[0].double().numpy().reshape(2, 4, 128), k) * scale

    def off(weights):  # with tokens that count as much as this, the rows' largest error
        w = np.exp(x - x.max(-1, keepdims=True)) * weights
        return worst((np.einsum("hgt,thd->hgd", w, v) / w.sum(-1, keepdims=True)).reshape(1, 8, 128), ref)

    one = np.ones(length)
    assert off(one) < 1e-12
    first = int(x[0, 0].argmax()) // lost * lost if q_std > 1 else 32  # (sharp scores: the unit that has the largest)
    planted = []
    for factor in (0.0, 2.0) if q_std == 1 else (0.0,):  # (twice what has all the weight is the same)
        planted.append(one.copy())
        planted[-1][first:first + lost] = factor
    if q_std == 1:
        planted.append(np.where(np.arange(length) < length // 2, 1.0, 1.5))
    for weights in planted:
        assert off(weights) > limit, (off(weights), limit)
    assert worst(0.6 * ref, ref) > limit


# ---- on the GPU -------------------------------------------------------------------------------------

CASES = [
    ([(2100, 1), (50, 1)], BF16, 1.0, False), ([(5000, 1)], BF16, 1.0, False), ([(16000, 1), (7000, 1), (1, 1)], BF16, 1.0, False),
    ([(3000, 1)], BF16, 30.0, False), ([(900, 5), (4000, 4)], BF16, 1.0, False), ([(100, 1)] * 40 + [(9000, 1)], BF16, 1.0, False),
    ([(700, 300), (3000, 64)], BF16, 1.0, True), ([(2100, 600)], BF16, 1.0, True), ([(3000, 90)], BF16, 30.0, True),
    ([(2100, 1), (300, 20)], F32, 1.0, False), ([(3000, 70)], F32, 1.0, False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("specs,dtype,q_std,wide", CASES)
def test_rows_in_norm(specs, dtype, q_std, wide, dim, quantized):
    cache, batch, q = inputs(specs, 2, 4, dim, quantized, dtype, q_std, "cuda:0", wide=wide)
    scale = dim ** -0.5
    got = cache.attention(q, batch)
    ref, _, _ = reference(cache, batch, q, scale)
    off, limit = worst(got.cpu().double().numpy(), ref), most_off(cache, batch, q, scale, dim, max(n for n, _ in specs), dtype)
    assert off <= limit, (off, limit)


@pytest.mark.gpu
@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("dim,page_size", [(64, 16), (128, 48), (128, 64), (256, 16)])
@pytest.mark.parametrize("specs,dtype,wide", [
    ([(5000, 1)], BF16, False), ([(9000, 1), (17, 1), (16, 1), (33, 1), (4000, 1)], BF16, False), ([(1, 1)] * 63 + [(12000, 1)], BF16, False),
    ([(1 + 11 * i, 1) for i in range(64)], BF16, False), ([(4000, 5), (40, 3), (2000, 7)], BF16, False), ([(1, 1)] * 300 + [(3000, 1)] * 3, BF16, False),
    ([(3000, 257), (513, 513)], BF16, True), ([(1500, 40)] * 4 + [(100, 100)] * 9, BF16, True), ([(2000, 1), (700, 100)], F32, False)])
def test_every_token_counts_once(specs, dtype, wide, dim, page_size, quantized):
    """Scores all alike, and values that are ones in one place, which moves on every sixteen tokens: a result is how many of the tokens that a
    row sees have it there, of all that it sees.  Sixteen tokens more or less are 16 / (16 * ceil(length / 16 / dim)) of a place or
    more: of 12000 tokens with 64 places 1/12, where half a step of bf16 is 2^-8."""
    batch, pages = batch_of(specs, page_size, **(dict(width=65536 // page_size, hints=False) if wide else {}))
    heads, group = 2, 2
    cache = filled_cache(pages, page_size, heads, dim, quantized)
    starts, table = batch.row_starts.tolist(), batch.page_table.cpu()
    places = torch.full((pages, page_size), -1, dtype=torch.long)
    ref = np.zeros((batch.rows, dim))
    for s, (length, n) in enumerate(specs):
        t = np.arange(length)
        places[table[s, t // page_size].long(), t % page_size] = torch.from_numpy(t // 16 % dim)
        for i in range(n):
            sees = length - n + i + 1
            ref[starts[s] + i] = np.bincount(t[:sees] // 16 % dim, minlength=dim) / sees
    ones = (places[..., None] == torch.arange(dim)).to("cuda:0")[:, None].expand(pages, heads, page_size, dim)
    if quantized:  # the levels 1 (code 15) and 0 (code 7)
        codes = torch.where(ones, 15, 7).to(torch.uint8)
        cache.v.copy_(codes[..., 0::2] | codes[..., 1::2] << 4)
        cache.v_scales.fill_(1.0)
    else:
        cache.v.copy_(ones)
    g = torch.Generator(device="cuda:0").manual_seed(11)
    q = torch.randn(batch.rows, heads * group, dim, device="cuda:0", generator=g).to(dtype)
    out = cache.attention(q, batch, 0.0).cpu().double().numpy()
    # half steps: the result's, the weights' (none: they are powers of two), and with NF4 the level's in f16; sums of up to 12000 in f32
    may = 2.0 ** -24 * 12000 + (2.0 ** -8 + 2.0 ** -11 if dtype == BF16 else 0)
    assert (np.abs(out - ref[:, None]) <= may * ref[:, None]).all(), float((np.abs(out - ref[:, None]) / np.maximum(ref[:, None], 1e-9)).max())
