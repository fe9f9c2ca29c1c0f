"""How wide the masks of trees are: what the batch says of its most rows, or what the caller brings; whatever is hinted, masks of the caller's width are the same."""
import numpy as np
import pytest
import torch

from cache_util import DEV, batch_of, filled_cache
from tree_util import ancestors, packed, random_parents

pytestmark = pytest.mark.gpu

SPECS = [(90, 70), (3, 3), (64, 40)]


def full(parents, words):
    starts, rows = np.cumsum([0] + [n for _, n in SPECS]), []
    for s, (_, n) in enumerate(SPECS):
        rows.append(packed(ancestors(parents, int(starts[s]), n)[0], words))
    return np.concatenate(rows)


@pytest.mark.parametrize("hint,words", [(0, 4), (70, 3), (64, 2), (3, 1), (1000, 32)])
def test_width(hint, words):
    batch, pages = batch_of(SPECS, 16)
    batch.max_rows = hint
    cache = filled_cache(pages, 16, 1, 64, True)
    parents = random_parents(SPECS, (0, 0), np.random.default_rng(1))
    up = torch.from_numpy(parents).to(DEV)
    masks, positions = cache.tree_masks(up, batch)
    assert masks.shape == (batch.rows, words) and (masks.cpu().numpy() == full(parents, words)).all()
    # the caller's width, and with it the results
    own = (torch.empty(batch.rows, 3, dtype=torch.int32, device=DEV), torch.empty(batch.rows, dtype=torch.int32, device=DEV))
    cache.tree_masks(up, batch, out=own)
    assert (own[0].cpu().numpy() == full(parents, 3)).all() and torch.equal(own[1], positions)
    q = torch.randn(batch.rows, 4, 64, device=DEV, generator=torch.Generator(device=DEV).manual_seed(2))
    batch.max_rows = 70
    right = cache.tree_attention(q, own[0], batch)
    if hint in (0, 70, 1000):
        assert torch.equal(cache.tree_attention(q, masks, batch), right)
    else:  # nodes behind the words are seen by none
        seen = torch.cat([torch.arange(n) for _, n in SPECS]) < 32 * words
        out = cache.tree_attention(q, masks, batch)
        assert torch.equal(out[seen], right[seen]) and not torch.equal(out[~seen], right[~seen])
