"""Attention of single tokens over sequences of unlike length takes about what its parts take, whichever sequence is the long one."""
import pytest
import torch

from cache_util import DEV, batch_of, filled_cache

pytestmark = pytest.mark.gpu


def shortest(specs, quantized):
    """Microseconds a call, the least of ten runs of twenty calls."""
    batch, pages = batch_of(specs, 64)
    cache = filled_cache(pages, 64, 4, 128, quantized)
    q = torch.randn(batch.rows, 28, 128, device=DEV).bfloat16()
    for _ in range(5):
        cache.attention(q, batch)
    best = float("inf")
    for _ in range(10):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        for _ in range(20):
            cache.attention(q, batch)
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b) / 20 * 1e3)
    return best


@pytest.mark.parametrize("quantized", [True, False])
@pytest.mark.parametrize("short,long", [(63, 120000), (200, 40000)])
@pytest.mark.parametrize("last", [True, False])
def test_a_long_sequence_among_short_ones(last, short, long, quantized):
    """Ten times and more where the CTAs that have the short ones are last; 0.9 to 1.1 measured."""
    mixed = [(1, 1)] * short + [(long, 1)] if last else [(long, 1)] + [(1, 1)] * short
    assert shortest(mixed, quantized) < 2.5 * (shortest([(1, 1)] * short, quantized) + shortest([(long, 1)], quantized))


@pytest.mark.parametrize("quantized", [True, False])
def test_lengths_that_grow(quantized):
    """64 sequences of 1 to 700 tokens: no more than 64 of 700 and half as much again."""
    assert shortest([(1 + 11 * i, 1) for i in range(64)], quantized) < 1.5 * shortest([(700, 1)] * 64, quantized)
