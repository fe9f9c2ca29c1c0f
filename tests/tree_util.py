"""Trees of drafted tokens made for a test, and what attention over them is in 64 bits."""
import numpy as np
import torch

from cache_util import DEV, stored, tokens_of


def random_parents(specs, spare_rows, rng, roots=0.1):
    """A parent to each row: an earlier node, or -1; rows of no sequence have 0."""
    got = [0] * spare_rows[0]
    for _, n in specs:
        got += [-1 if i == 0 or rng.random() < roots else int(rng.integers(0, i)) for i in range(n)]
    return np.array(got + [0] * spare_rows[1], np.int32)


def ancestors(parents, first, n):
    """[n, n]: which nodes each node of a sequence sees, and each node's depth."""
    seen, depth = np.zeros((n, n), bool), np.zeros(n, np.int64)
    for i in range(n):
        p = int(parents[first + i])
        if 0 <= p < i:
            seen[i], depth[i] = seen[p], depth[p] + 1
        seen[i, i] = True
    return seen, depth


def packed(bits, words):
    """[rows, n] truth values to [rows, words] of int32; what does not fit is dropped."""
    wide = np.zeros((bits.shape[0], 32 * words), np.uint64)
    n = min(bits.shape[1], 32 * words)
    wide[:, :n] = bits[:, :n]
    return (wide.reshape(-1, words, 32) << np.arange(32, dtype=np.uint64)).sum(-1).astype(np.uint32).view(np.int32)


def unpacked(masks):
    """[rows, words] of int32 to [rows, 32 * words] truth values."""
    return (masks.view(np.uint32)[..., None] >> np.arange(32, dtype=np.uint32) & 1).astype(bool).reshape(len(masks), -1)


def masks_of(kind, specs, batch, rng):
    """Masks of a call's rows: tree (ancestors), any (whatever bits), none, all."""
    starts, most = batch.row_starts.cpu().numpy(), max(n for _, n in specs)
    words = max(1, -(-most // 32)) + (1 if kind == "any" else 0)
    bits = np.zeros((batch.rows, 32 * words), bool)
    if kind == "any":
        bits = rng.random(bits.shape) < 0.3
    elif kind == "all":
        bits[:] = True
    elif kind == "tree":
        parents = random_parents(specs, (int(starts[0]), batch.rows - int(starts[-1])), rng)
        for s, (_, n) in enumerate(specs):
            bits[starts[s]:starts[s + 1], :n] = ancestors(parents, int(starts[s]), n)[0]
    return torch.from_numpy(packed(bits, words)).to(DEV)


def tree_reference(cache, batch, q, masks, scale):
    """out, sum of weights * |value| and the largest sum of |q * k| * scale of each row, in 64 bits; rows of no sequence: NaNs."""
    k_all, v_all = stored(cache, "k"), stored(cache, "v")
    q, bits = q.cpu().double().numpy(), unpacked(masks.cpu().numpy())
    out, spread, reach = (np.full(q.shape[:n], np.nan) for n in (3, 3, 2))
    starts, group = batch.row_starts.cpu().numpy(), q.shape[1] // cache.heads()
    for s in range(len(starts) - 1):
        n, length = int(starts[s + 1] - starts[s]), int(batch.lengths[s])
        if n == 0:
            continue
        k, v = tokens_of(k_all, batch, cache.page_size(), s), tokens_of(v_all, batch, cache.page_size(), s)
        rows, context = slice(int(starts[s]), int(starts[s + 1])), length - n
        hidden = np.zeros((n, length), bool)
        for t in range(max(context, 0), length):
            j = t - context
            hidden[:, t] = ~bits[rows, j] if j < bits.shape[1] else True
        hidden[:max(-context, 0)] = True  # rows whose own token is negative
        for h in range(q.shape[1]):
            kk, vv, qq = k[:, h // group], v[:, h // group], q[rows, h]
            x = np.where(hidden, -np.inf, scale * (qq @ kk.T))
            w = np.exp(x - np.maximum(x.max(1, initial=-np.inf, keepdims=True), -1e300))
            w /= np.maximum(w.sum(1, keepdims=True), 1e-300)
            out[rows, h], spread[rows, h] = w @ vv, w @ np.abs(vv)
            reach[rows, h] = np.where(hidden, 0, abs(scale) * (np.abs(qq) @ np.abs(kk).T)).max(1, initial=0)
    return out, spread, reach
