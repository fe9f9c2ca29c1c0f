"""Trees of drafted tokens over the key and value cache as cases: what a decoder layer does to verify many continuations at once.

  tree    the masks (which of a sequence's drafted tokens a token descends from) and the positions of trees given by their parents
  rotate  a call's new keys, turned by the angles of their positions, and values into the pages of their sequences, its queries
          turned by the same; a pass reads back what it wrote, so that the cache's new state is among its outputs
  attend  each drafted token over all that is cached of its sequence ahead of the tree, and over its own ancestors in the tree
  keep    the tokens of the accepted paths to the places behind the context; a pass appends the drafted tokens first, so that it
          can be repeated, and reads back what was kept

``own`` says which side a pass takes: the plain form (elementary torch operations, f32) or the package's operators.
"""
import math
import random

import torch

own = False

BLOCK = 64  # values that share a scale
# the sixteen NF4 levels
LEVELS = (-1.0, -0.6961928009986877, -0.5250730514526367, -0.39491748809814453, -0.28444138169288635, -0.18477343022823334,
          -0.09105003625154495, 0.0, 0.07958029955625534, 0.16093020141124725, 0.24611230194568634, 0.33791524171829224,
          0.44070982933044434, 0.5626170039176941, 0.7229568362236023, 1.0)
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _case(op, form, dtype, sequences, new, context, heads=4, group=7, dim=128, page=64, ragged=0, rotary=0, pairs=False, tree=True):
    """`sequences` of up to `context` tokens in the cache, the newest `new` of them the call's rows, which are trees of drafted
    tokens or, without `tree`, follow one another; `ragged`: 0, all alike, or the seed of their sizes.  `heads` of keys and values,
    `group` query heads to each.  `rotary` of a head's values are turned (0: all), neighbours or (without `pairs`) halves."""
    return {"op": op, "form": form, "dtype": dtype, "sequences": sequences, "new": new, "context": context, "heads": heads,
            "group": group, "dim": dim, "page": page, "ragged": ragged, "rotary": rotary or dim, "pairs": pairs, "tree": tree}


def listed():
    return [
        # a draft model's trees of one step of a server: sixteen sequences, 64 nodes
        dict(_case("tree", "nf4", "bf16", 16, 64, 4096), name="tree_step"),
        # one long tree: several drafts laid one behind the other
        dict(_case("tree", "nf4", "bf16", 1, 500, 9000, page=48), name="tree_long"),
        # the drafted tokens of eight sequences (heads of the Qwen2-7B-shaped block: 28 over 4 of 128), cache quantized
        dict(_case("rotate", "nf4", "bf16", 8, 16, 4096), name="rotate_step"),
        # prompts of several users, no multiple of a page
        dict(_case("rotate", "nf4", "bf16", 3, 2731, 2731, page=48, ragged=5, tree=False), name="rotate_prompts"),
        # the reference's tensor type, neighbours turned, half of a head's values, cache not quantized
        dict(_case("rotate", "bf16", "f32", 2, 900, 1200, heads=8, group=4, page=16, rotary=64, pairs=True, ragged=8, tree=False),
             name="rotate_part"),
        # the smallest: one young sequence's few drafted tokens
        dict(_case("attend", "bf16", "bf16", 1, 4, 200), name="attend_few"),
        # the block's trees of 64 nodes: eight sequences
        dict(_case("attend", "nf4", "bf16", 8, 64, 4096), name="attend_block"),
        # a server's batch of uneven sequences and trees
        dict(_case("attend", "nf4", "bf16", 16, 16, 8192, heads=8, group=4, page=32, ragged=11), name="attend_server"),
        # the same with a cache that is not quantized, small pages and larger trees
        dict(_case("attend", "bf16", "bf16", 18, 20, 8192, heads=8, group=4, page=16, ragged=7), name="attend_wide"),
        # the reference's tensor type
        dict(_case("attend", "nf4", "f32", 3, 21, 700, heads=2, group=4, dim=64, page=48, ragged=9), name="attend_f32"),
        # the end of a step of one sequence and of a server's
        dict(_case("keep", "nf4", "bf16", 1, 8, 1000), name="keep_one"),
        dict(_case("keep", "bf16", "bf16", 48, 40, 2048, heads=8, group=4, page=16, ragged=4), name="keep_server"),
    ]


def _spread(rng, low, high):
    """A size of [low, high], even over its logarithm."""
    return min(max(int(round(math.exp(rng.uniform(math.log(low), math.log(high))))), low), high)


def draw(rng):
    op = rng.choice(("tree", "rotate", "rotate", "attend", "attend", "attend", "attend", "keep"))
    heads, group = rng.choice(((4, 7), (8, 4), (2, 7), (2, 4), (1, 8), (4, 1), (16, 1), (2, 16), (1, 5)))
    dim, page = rng.choice((64, 128, 128, 128, 256)), rng.choice((16, 32, 48, 64, 64, 128, 256))
    form, ragged = rng.choice(("nf4", "nf4", "bf16")), rng.randrange(1, 1000) if rng.random() < 0.6 else 0
    dtype = "f32" if rng.random() < 0.15 else "bf16"
    row = heads * dim
    if op == "tree":
        sequences = _spread(rng, 1, 64)
        new = _spread(rng, 1, 512)
        return _case(op, form, dtype, sequences, new, _spread(rng, new, 16384), heads, group, dim, page, ragged)
    if op == "keep":
        sequences = _spread(rng, 1, 64)
        new = _spread(rng, 1, max(1, min(64, (1 << 20) // (sequences * row))))
        return _case(op, form, dtype, sequences, new, _spread(rng, max(new, 16), max(new, 16, min(4096, (1 << 24) // (sequences * row)))),
                     heads, group, dim, page, ragged)
    if op == "rotate":
        tree = rng.random() < 0.4
        rotary, pairs = rng.choice((dim, dim, dim // 2, 16 * rng.randint(1, dim // 16))), rng.random() < 0.3
        sequences = _spread(rng, 1, 64 if tree else 8)
        most = max(1, (1 << 23) // (sequences * row * group))
        new = _spread(rng, 1, min(64, most)) if tree else _spread(rng, 1, min(8192, most))
        context = _spread(rng, new, max(new, min(32768, (1 << 25) // (sequences * row))))
        return _case(op, form, dtype, sequences, new, context, heads, group, dim, page, ragged, rotary, pairs, tree)
    sequences = _spread(rng, 1, 32)
    # bounded by the largest listed cases' work
    products = (7 << 30) // (sequences * row * group)
    new = _spread(rng, 1, min(128 if dtype == "f32" else 512, products // 64, math.isqrt(products)))
    most = min(65536, (1 << 26) // (sequences * row), products // new)
    if dtype == "f32":
        most = min(most, 4096)
    return _case(op, form, dtype, sequences, new, _spread(rng, max(new, 64), max(new, 64, most)), heads, group, dim, page, ragged)


# ---- sizes and inputs ---------------------------------------------------------------------------


def _sizes(case):
    """[(tokens in the cache, newest ones that are the call's rows)] of the case's sequences."""
    c = case
    if not c["ragged"]:
        return [(c["context"], c["new"])] * c["sequences"]
    rng, got = random.Random(c["ragged"]), []
    for i in range(c["sequences"]):
        new = c["new"] if i == 0 else rng.randint(max(1, c["new"] // 3), c["new"])
        length = c["context"] if i == 0 else rng.randint(max(1, c["context"] // 8), c["context"])
        got.append((max(new, length), new))
    return got


def _levels(dtype):
    return torch.tensor(LEVELS, dtype=torch.float32, device="cuda").to(dtype)


def _quantized(x):
    """f32 values [..., dim] to packed codes [..., dim / 2] and the scales of their blocks [..., dim / 64]; for inputs, where a
    value next to a border may go either way."""
    levels = _levels(torch.float32)
    blocks = x.unflatten(-1, (-1, BLOCK))
    scales = blocks.abs().amax(-1)
    codes = torch.bucketize((blocks / scales[..., None]).flatten(-2), (levels[1:] + levels[:-1]) / 2).to(torch.uint8)
    return codes[..., 0::2] | codes[..., 1::2] << 4, scales


def _rows(s):
    """Every row's sequence and its number in it."""
    at = torch.arange(s["rows"], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["starts"][1:], at, right=True)
    return seq, (at - s["starts"][seq]).long()


def _plain_tree(s):
    """Masks [rows, words] and positions [rows] of the trees: who is reached from a node in 1, 2, 4, ... steps to its parent."""
    seq, i = _rows(s)
    n = s["most_rows"]
    reach = torch.zeros(len(s["lengths"]), n, n, device="cuda")
    reach[seq, i, i] = 1.0
    up = s["parents"].long()
    has = (up >= 0).float()
    reach[seq, i, up.clamp(min=0)] += has
    for _ in range(max(1, (n - 1).bit_length())):
        reach = (reach @ reach).clamp(max=1.0)
    seen = reach[seq, i]  # [rows, n]
    position = (s["lengths"] - (s["starts"][1:] - s["starts"][:-1]))[seq] + (seen.sum(-1) - 1).to(torch.int32)
    words = s["words"]
    bits = torch.nn.functional.pad(seen, (0, 32 * words - n)).long().unflatten(-1, (words, 32))
    return [(bits << torch.arange(32, device="cuda")).sum(-1).to(torch.int32), position]


def prepare(case, seed):
    c, sizes = case, _sizes(case)
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, device="cuda", generator=gen) * std

    heads, dim, page, op = c["heads"], c["dim"], c["page"], c["op"]
    counts = [-(-length // page) for length, _ in sizes]
    width, pages = max(counts), sum(counts) + 3
    # every sequence's pages somewhere in the pool; an entry that no token needs names no page
    order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
    filled = torch.tensor(counts, device="cuda")[:, None] > torch.arange(width, device="cuda")
    table = torch.full((len(sizes), width), -1, dtype=torch.int32, device="cuda")
    table[filled] = order[:sum(counts)]
    starts, rows = [0], 0
    for _, new in sizes:
        rows += new
        starts.append(rows)
    most_rows = max(n for _, n in sizes)
    s = {"op": op, "form": c["form"], "dtype": DTYPES[c["dtype"]], "rows": rows, "most_rows": most_rows, "heads": heads, "dim": dim,
         "held": torch.float32 if c["form"] == "nf4" else torch.bfloat16,
         "most_tokens": max(n for n, _ in sizes), "table": table, "page": page, "scale": dim ** -0.5, "words": -(-most_rows // 32),
         "lengths": torch.tensor([n for n, _ in sizes], dtype=torch.int32, device="cuda"),
         "starts": torch.tensor(starts, dtype=torch.int32, device="cuda"), "positions": None}
    if c["tree"]:
        # a node's parent is any node before it; one in twenty is a further root
        _, i = _rows(s)
        up = (torch.rand(rows, device="cuda", generator=gen) * i).long().clamp(max=(i - 1).clamp(min=0))
        root = (torch.rand(rows, device="cuda", generator=gen) < 0.05) | (i == 0)
        s["parents"] = torch.where(root, -1, up).to(torch.int32)
        if op in ("rotate", "attend"):
            s["masks"], s["positions"] = _plain_tree(s)
    # keys have channels of unlike size, values are smaller
    channels = torch.exp(normal(heads, 1, dim, std=0.5))
    for name, std in (("k", channels), ("v", 0.3)):
        if op == "attend":
            if c["form"] == "nf4":
                s[name + "_pool"], s[name + "_scales"] = _quantized(normal(pages, heads, page, dim) * std)
            else:
                s[name + "_pool"] = (normal(pages, heads, page, dim) * std).to(torch.bfloat16)
            continue
        if c["form"] == "nf4":
            s[name + "_pool"] = torch.zeros(pages, heads, page, dim // 2, dtype=torch.uint8, device="cuda")
            s[name + "_scales"] = torch.zeros(pages, heads, page, dim // BLOCK, device="cuda")
        else:
            s[name + "_pool"] = torch.zeros(pages, heads, page, dim, dtype=torch.bfloat16, device="cuda")
        if op != "tree":  # rows as the projections leave them
            s[name] = (normal(rows, heads, dim) * (channels[:, 0] if name == "k" else std)).to(s["dtype"])
    if op in ("attend", "rotate"):
        s["q"] = normal(rows, heads * c["group"], dim).to(s["dtype"])
    if op == "rotate":
        s["pairs"], s["rotary"] = c["pairs"], c["rotary"]
        steps = torch.arange(c["rotary"] // 2, device="cuda", dtype=torch.float64)
        angles = torch.arange(s["most_tokens"], device="cuda", dtype=torch.float64)[:, None] * 1e6 ** (-2 * steps / c["rotary"])
        s["turns"] = torch.cat((angles.cos(), angles.sin()), 1).float()  # [positions, rotary], as a program keeps it
    if op == "keep":
        # a path begins at the first node, and has eight nodes at most; how many is the case's, which ones the seed's
        many, rng = random.Random(c["ragged"]), random.Random(seed)
        paths = [[0, *sorted(rng.sample(range(1, new), many.randint(0, min(7, new - 1))))] for _, new in sizes]
        kept = torch.zeros(len(sizes), max(len(p) for p in paths), dtype=torch.int32)
        for row, path in zip(kept, paths):
            row[:len(path)] = torch.tensor(path, dtype=torch.int32)
        s["kept"], counts = kept.cuda(), [len(p) for p in paths]
        s["counts"] = torch.tensor(counts, dtype=torch.int32, device="cuda")
        s["kept_rows"], s["most_kept"] = sum(counts), max(counts)
        s["kept_starts"] = torch.tensor([0, *counts], dtype=torch.int32).cumsum(0).to(torch.int32).cuda()
    return s


# ---- a pass -------------------------------------------------------------------------------------


def _own(s):
    from unifur_b200.kv_cache import CacheBatch, PagedKvCache, Rotation

    cache = PagedKvCache(s["k_pool"], s["v_pool"], s.get("k_scales"), s.get("v_scales"))
    batch = CacheBatch(s["table"], s["lengths"], s["starts"], s["rows"], max_rows=s["most_rows"], max_length=s["most_tokens"])
    if s["op"] == "tree":
        return list(cache.tree_masks(s["parents"], batch))
    if s["op"] == "attend":
        return cache.tree_attention(s["q"], s["masks"], batch, s["scale"])
    if s["op"] == "rotate":
        q = cache.append_rotated(s["k"], s["v"], batch, Rotation(s["turns"], pairs=s["pairs"]), s["positions"], s["q"])
        return [q, *cache.read(batch, s["held"])]
    cache.append(s["k"], s["v"], batch)
    lengths = cache.keep(s["kept"], s["counts"], batch)
    after = CacheBatch(s["table"], lengths, s["kept_starts"], s["kept_rows"], max_rows=s["most_kept"], max_length=s["most_tokens"])
    return [lengths, *cache.read(after, s["held"])]


def _places(s, seq, token):
    """The page and the place in it of sequences' tokens."""
    return s["table"][seq, token // s["page"]].long(), (token % s["page"]).long()


def _tokens(s):
    seq, i = _rows(s)
    return seq, (s["lengths"] - (s["starts"][1:] - s["starts"][:-1]))[seq] + i.to(torch.int32)


def _values(s, name, page, place):
    """The cache's values at (page, place) in f32: [..., heads, dim]."""
    if s["form"] == "bf16":
        return s[name + "_pool"][page, :, place].float()
    packed = s[name + "_pool"][page, :, place]
    codes = torch.stack((packed & 15, packed >> 4), -1).flatten(-2)
    values = _levels(torch.float32)[codes.long()].unflatten(-1, (-1, BLOCK))
    return (values * s[name + "_scales"][page, :, place][..., None]).flatten(-2)


def _store(s, name, values, page, place):
    """f32 values [rows, heads, dim] into the cache."""
    if s["form"] == "bf16":
        s[name + "_pool"][page, :, place] = values.to(torch.bfloat16)
        return
    blocks = values.unflatten(-1, (-1, BLOCK))
    scales = blocks.abs().amax(-1)
    quotients = (blocks / scales[..., None]).nan_to_num(0.0)  # a block of zeros has the level 0
    codes = (quotients[..., None] - _levels(torch.float32)).abs().argmin(-1).flatten(-2).to(torch.uint8)
    s[name + "_pool"][page, :, place] = codes[..., 0::2] | codes[..., 1::2] << 4
    s[name + "_scales"][page, :, place] = scales


def _turned(s, x, position):
    """Rows [rows, heads, dim] turned, in f32."""
    x, half = x.float(), s["rotary"] // 2
    turn = s["turns"][position.long()][:, None]
    cos, sin = turn[..., :half], turn[..., half:]
    out = x.clone()
    first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if s["pairs"] else (slice(0, half), slice(half, 2 * half))
    a, b = x[..., first], x[..., second]
    out[..., first] = a * cos - b * sin
    out[..., second] = b * cos + a * sin
    return out


def _plain_attention(s):
    starts, lengths = s["starts"].long(), s["lengths"].long()
    counts = starts[1:] - starts[:-1]
    tokens = torch.arange(s["most_tokens"], device="cuda")
    page = s["table"][:, tokens // s["page"]].long().clamp(min=0)
    place = (tokens % s["page"]).expand_as(page)
    k, v = (_values(s, name, page, place).transpose(1, 2) for name in ("k", "v"))  # [sequences, heads, tokens, dim]
    # queries padded to the largest tree: [sequences, rows, heads, group, dim] -> [sequences, heads, rows * group, dim]
    i = torch.arange(s["most_rows"], device="cuda")
    row = (starts[:-1, None] + i).clamp(max=s["rows"] - 1)
    heads = k.shape[1]
    q = s["q"].float().unflatten(1, (heads, -1))[row].permute(0, 2, 1, 3, 4)
    group = q.shape[3]
    scores = (q.flatten(2, 3) @ k.transpose(2, 3)) * s["scale"]
    node = tokens - (lengths - counts)[:, None]  # [sequences, tokens]: the token's number in the tree
    bit = node.clamp(0, 32 * s["words"] - 1)
    word = s["masks"][row].gather(2, (bit // 32)[:, None].expand(-1, len(i), -1))  # [sequences, rows, tokens]
    in_tree = ((word >> (bit % 32)[:, None]) & 1) != 0
    seen = ((node < 0)[:, None] | in_tree) & (tokens < lengths[:, None])[:, None]
    seen = seen[:, None, :, None].expand(-1, heads, -1, group, -1).flatten(2, 3)
    scores = scores.masked_fill_(~seen, -math.inf)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = (weights @ v) / weights.sum(-1, keepdim=True)
    out = out.unflatten(2, (-1, group)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    return out[i < counts[:, None]].to(s["dtype"])


def run(state):
    s = state
    if own:
        return _own(s)
    if s["op"] == "tree":
        return _plain_tree(s)
    if s["op"] == "attend":
        return _plain_attention(s)
    seq, token = _tokens(s)
    page, place = _places(s, seq, token)
    if s["op"] == "rotate":
        position = token if s["positions"] is None else s["positions"]
        _store(s, "k", _turned(s, s["k"], position), page, place)
        _store(s, "v", s["v"].float(), page, place)
        return [_turned(s, s["q"], position).to(s["dtype"]), *(_values(s, name, page, place).to(s["held"]) for name in ("k", "v"))]
    for name in ("k", "v"):
        _store(s, name, s[name].float(), page, place)
    context = s["lengths"] - (s["starts"][1:] - s["starts"][:-1])
    at = torch.arange(s["kept_rows"], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["kept_starts"][1:], at, right=True)
    j = at - s["kept_starts"][seq]
    old, new = _places(s, seq, context[seq] + s["kept"][seq, j.long()]), _places(s, seq, context[seq] + j)
    for name in ("k_pool", "v_pool", *(("k_scales", "v_scales") if s["form"] == "nf4" else ())):
        s[name][new[0], :, new[1]] = s[name][old[0], :, old[1]]
    return [context + s["counts"], *(_values(s, name, *new).to(s["held"]) for name in ("k", "v"))]


# ---- the definition in 64 bits ------------------------------------------------------------------


def _exact_tokens(s, name, seq, first, last):
    """The cache's tokens [first, last) of a sequence: [tokens, heads, dim]."""
    pool, scales, size = s[name + "_pool"], s.get(name + "_scales"), s["page"]
    ids = s["table"][seq].tolist()[first // size:-(-last // size)]
    skip = first % size
    whole = pool[ids].transpose(1, 2).flatten(0, 1)[skip:skip + last - first]
    if scales is None:
        return whole.double()
    factors = scales[ids].transpose(1, 2).flatten(0, 1)[skip:skip + last - first].double()
    levels = torch.tensor(LEVELS, dtype=torch.float64, device="cuda")
    values = torch.empty(*whole.shape[:2], 2 * whole.shape[2], dtype=torch.float64, device="cuda")
    values[..., 0::2] = levels[(whole & 15).int()]
    values[..., 1::2] = levels[(whole >> 4).int()]
    return values * factors.repeat_interleave(BLOCK, -1)


def _exact_stored(x, form):
    """What the cache holds for values x, ahead of a rounding to bf16."""
    x = x.double()
    if form == "bf16":
        return x
    levels = torch.tensor(LEVELS, dtype=torch.float64, device="cuda")
    out = torch.empty_like(x)
    for b in range(0, x.shape[-1], BLOCK):
        part = x[..., b:b + BLOCK]
        scale = part.abs().amax(-1, keepdim=True)
        unit = torch.where(scale > 0, part / scale, torch.zeros_like(part))
        best, off = torch.zeros_like(unit), torch.full_like(unit, math.inf)
        for level in levels:
            d = (unit - level).abs()
            best, off = torch.where(d < off, level, best), torch.minimum(d, off)
        out[..., b:b + BLOCK] = best * scale
    return out


def _exact_turned(x, position, turns, pairs):
    """Each value by its partner's place: turned by (cos, sin), a rotation of the plane that the two span."""
    x, rotary = x.double(), turns.shape[1]
    half, d = rotary // 2, torch.arange(rotary, device="cuda")
    first = d % 2 == 0 if pairs else d < half
    partner = (d ^ 1) if pairs else (d + half) % rotary
    which = d // 2 if pairs else d % half
    turn = turns.double()[position.long()]
    cos, sin = turn[:, which][:, None], turn[:, half + which][:, None]
    out = x.clone()
    out[..., :rotary] = x[..., :rotary] * cos + x[..., partner] * torch.where(first, -sin, sin)
    return out


def exact(case, seed):
    s, sizes = prepare(case, seed), _sizes(case)
    starts = s["starts"].tolist()
    if s["op"] == "tree":
        parents = s["parents"].tolist()
        masks, positions = torch.zeros(s["rows"], s["words"], dtype=torch.int64), []
        for i, (length, new) in enumerate(sizes):
            above, depth = [], []
            for j in range(new):
                p = parents[starts[i] + j]
                above.append((above[p] if p >= 0 else 0) | 1 << j)
                depth.append(depth[p] + 1 if p >= 0 else 0)
            for j in range(new):
                masks[starts[i] + j] = torch.tensor([above[j] >> 32 * w & 0xffffffff for w in range(s["words"])])
                positions.append(length - new + depth[j])
        return [torch.where(masks >= 1 << 31, masks - (1 << 32), masks).to(torch.int32).cuda(),
                torch.tensor(positions, dtype=torch.int32, device="cuda")]
    if s["op"] == "rotate":
        position = s["positions"]
        if position is None:
            position = torch.cat([torch.arange(length - new, length) for length, new in sizes]).cuda()
        # a quotient next to a border goes by its rounding to f32, which 64 bits do not say
        turned = _exact_turned(s["k"], position, s["turns"], s["pairs"])
        return [_exact_turned(s["q"], position, s["turns"], s["pairs"]), None if s["form"] == "nf4" else turned,
                None if s["form"] == "nf4" and s["dtype"] == torch.float32 else _exact_stored(s["v"], s["form"])]
    if s["op"] == "keep":
        lengths = torch.tensor([length - new for length, new in sizes], dtype=torch.int32, device="cuda") + s["counts"]
        if s["form"] == "nf4" and s["dtype"] == torch.float32:
            return [lengths, None, None]
        at = torch.cat([starts[i] + s["kept"][i, :int(n)] for i, n in enumerate(s["counts"])]).long()
        return [lengths, _exact_stored(s["k"][at], s["form"]), _exact_stored(s["v"][at], s["form"])]
    parts = []
    for i, (length, new) in enumerate(sizes):
        k, v = _exact_tokens(s, "k", i, 0, length), _exact_tokens(s, "v", i, 0, length)
        rows = slice(starts[i], starts[i + 1])
        q, words = s["q"][rows].double(), s["masks"][rows]
        group = q.shape[1] // k.shape[1]
        hidden = torch.zeros(new, length, dtype=torch.bool, device="cuda")
        for j in range(new):
            hidden[:, length - new + j] = (words[:, j // 32] >> j % 32) & 1 == 0
        heads = []
        for h in range(q.shape[1]):
            scores = torch.mm(q[:, h], k[:, h // group].t()) * s["scale"]
            heads.append(torch.mm(torch.softmax(scores.masked_fill(hidden, -math.inf), -1), v[:, h // group]))
        parts.append(torch.stack(heads, 1))
    return torch.cat(parts)


# ---- what a pass cannot do without --------------------------------------------------------------


def work(case):
    c, sizes = case, _sizes(case)
    esize = 4 if c["dtype"] == "f32" else 2
    rows, tokens = sum(n for _, n in sizes), sum(n for n, _ in sizes)
    row = c["heads"] * c["dim"]  # values of a key or value row
    stored = row // 2 + 4 * row // BLOCK if c["form"] == "nf4" else 2 * row
    back = 4 * row if c["form"] == "nf4" else 2 * row  # and as it is read
    words = -(-max(n for _, n in sizes) // 32)
    if c["op"] == "tree":
        return {"bytes": rows * (8 + 4 * words), "flops": rows}
    if c["op"] == "keep":  # rows in, their storage out; the paths' storage read, and written as it is and dense
        paths = sum(min(4, n) for _, n in sizes)
        return {"bytes": 2 * rows * (esize * row + stored) + 2 * paths * (2 * stored + back), "flops": 0}
    if c["op"] == "rotate":  # rows in, storage and queries out; what is stored is read back
        turns = 4 * c["rotary"] * rows
        return {"bytes": 2 * rows * (esize * row + stored + back) + 2 * esize * rows * row * c["group"] + turns,
                "flops": 3 * rows * c["heads"] * (c["group"] + 1) * c["rotary"]}
    # of a tree of n nodes a row sees some 1 + log n; the products are counted as dense, which tensor cores take them as
    pairs = sum(new * length for length, new in sizes)
    return {"bytes": 2 * tokens * stored + 2 * esize * rows * row * c["group"] + 4 * words * rows, "flops": 4 * pairs * row * c["group"]}
