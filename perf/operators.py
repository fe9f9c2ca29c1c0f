"""The key and value cache's operators as cases: what a decoder layer does between its quantized projections.

  append     a call's new keys and values into the pages of their sequences, quantized to NF4 as they are written or kept in
             bf16; a pass reads back what it wrote, so that the cache's new state is among its outputs
  read       rows of the cache back as dense tensors
  attention  each sequence's newest rows over all that its pages hold, causally: single tokens, drafted tokens, chunks of a
             prompt, whole prompts

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


def _case(op, form, dtype, sequences, new, context, heads=4, group=7, dim=128, page=64, ragged=0):
    """`sequences` of up to `context` tokens in the cache, the newest `new` of them the call's rows; `ragged`: 0, all alike, or
    the seed of their lengths.  `heads` of keys and values, `group` query heads to each."""
    return {"op": op, "form": form, "dtype": dtype, "sequences": sequences, "new": new, "context": context, "heads": heads,
            "group": group, "dim": dim, "page": page, "ragged": ragged}


def listed():
    return [
        # a decode step of eight sequences: one token each into the cache (heads of the Qwen2-7B-shaped block: 28 over 4 of 128)
        dict(_case("append", "nf4", "bf16", 8, 1, 4096), name="append_step"),
        # prompts of several users, no multiple of a page
        dict(_case("append", "nf4", "bf16", 3, 2731, 2731, page=48, ragged=5), name="append_prompts"),
        # the whole context of eight sequences back in bf16, as for moving it or for a check of what quantization cost
        dict(_case("read", "nf4", "bf16", 8, 4096, 4096, ragged=3), name="read_context"),
        # a short shared prefix back in the reference's type
        dict(_case("read", "nf4", "f32", 1, 333, 333, heads=2, dim=64, page=16), name="read_prefix"),
        # the smallest call: one token of one young sequence
        dict(_case("attention", "bf16", "bf16", 1, 1, 200), name="decode_one"),
        # the block's decode step: eight sequences
        dict(_case("attention", "nf4", "bf16", 8, 1, 4096), name="decode_block"),
        # a server's batch of uneven sequences, cache not quantized
        dict(_case("attention", "bf16", "bf16", 64, 1, 8192, ragged=7), name="decode_many"),
        # one token over a long context
        dict(_case("attention", "nf4", "bf16", 1, 1, 131072, page=128), name="decode_long"),
        # drafted tokens of sixteen sequences, to be verified at once
        dict(_case("attention", "nf4", "bf16", 16, 5, 8192, heads=8, group=4, page=32, ragged=11), name="chunk_draft"),
        # the block's prompt of 4096 tokens
        dict(_case("attention", "nf4", "bf16", 1, 4096, 4096), name="chunk_prompt"),
        # chunks of three prompts over what is cached of them
        dict(_case("attention", "bf16", "bf16", 3, 1024, 12288, page=16, ragged=2), name="chunk_context"),
        # the reference's tensor type
        dict(_case("attention", "nf4", "f32", 3, 100, 700, heads=2, group=4, dim=64, page=48, ragged=9), name="chunk_f32"),
    ]


def _spread(rng, low, high):
    """A size of [low, high], even over its logarithm."""
    return min(max(int(round(math.exp(rng.uniform(math.log(low), math.log(high))))), low), high)


def draw(rng):
    op = rng.choice(("append", "read", "attention", "attention", "attention", "attention"))
    heads, group = rng.choice(((4, 7), (8, 4), (2, 7), (2, 4), (1, 8), (4, 1), (16, 1), (2, 16), (1, 5)))
    dim, page = rng.choice((64, 128, 128, 128, 256)), rng.choice((16, 32, 48, 64, 64, 128, 256))
    form, ragged = rng.choice(("nf4", "nf4", "bf16")), rng.randrange(1, 1000) if rng.random() < 0.6 else 0
    dtype = "f32" if rng.random() < 0.15 else "bf16"
    if op != "attention":
        sequences = _spread(rng, 1, 64)
        new = _spread(rng, 1, max(1, min(8192, (1 << 24) // (sequences * heads * dim))))
        context = new if op == "read" else _spread(rng, new, max(new, min(16384, (1 << 25) // (sequences * heads * dim))))
        return _case(op, form, dtype, sequences, new, context, heads, group, dim, page, ragged)
    kind = rng.choice(("decode", "decode", "draft", "chunk", "chunk"))
    sequences = _spread(rng, 1, 64 if kind == "decode" else 16 if kind == "draft" else 4)
    new = 1 if kind == "decode" else rng.randint(2, 8) if kind == "draft" else _spread(rng, 9, 256 if dtype == "f32" else 2048)
    # bounded by what a plain pass holds: keys and values in f32, and the scores
    most = min(131072, (1 << 27) // (sequences * heads * dim), (1 << 35) // (sequences * heads * group * new * dim))
    if dtype == "f32":
        most = min(most, 4096)
    context = _spread(rng, max(new, 64), max(new, 64, most))
    return _case(op, form, dtype, sequences, new, context, heads, group, dim, page, ragged)


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
        got.append((new, new) if c["op"] == "read" else (max(new, length), new))
    return got


def _levels(device, dtype):
    return torch.tensor(LEVELS, dtype=torch.float32, device=device).to(dtype)


def _quantized(x):
    """f32 values [..., dim] to packed codes [..., dim / 2] and the scales of their blocks [..., dim / 64]; for inputs, where a
    value next to a border may go either way."""
    levels = _levels(x.device, torch.float32)
    blocks = x.unflatten(-1, (-1, BLOCK))
    scales = blocks.abs().amax(-1)
    codes = torch.bucketize((blocks / scales[..., None]).flatten(-2), (levels[1:] + levels[:-1]) / 2).to(torch.uint8)
    return codes[..., 0::2] | codes[..., 1::2] << 4, scales


def prepare(case, seed):
    c, sizes = case, _sizes(case)
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, device="cuda", generator=gen) * std

    heads, dim, page = c["heads"], c["dim"], c["page"]
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
    s = {"op": c["op"], "form": c["form"], "dtype": DTYPES[c["dtype"]], "rows": rows, "most_rows": max(n for _, n in sizes),
         "most_tokens": max(n for n, _ in sizes), "table": table, "page": page, "scale": dim ** -0.5,
         "lengths": torch.tensor([n for n, _ in sizes], dtype=torch.int32, device="cuda"),
         "starts": torch.tensor(starts, dtype=torch.int32, device="cuda")}
    # keys have channels of unlike size, values are smaller
    channels = torch.exp(normal(heads, 1, dim, std=0.5))
    for name, std in (("k", channels), ("v", 0.3)):
        if c["op"] == "append":
            if c["form"] == "nf4":
                s[name + "_pool"] = torch.zeros(pages, heads, page, dim // 2, dtype=torch.uint8, device="cuda")
                s[name + "_scales"] = torch.zeros(pages, heads, page, dim // BLOCK, device="cuda")
            else:
                s[name + "_pool"] = torch.zeros(pages, heads, page, dim, dtype=torch.bfloat16, device="cuda")
            # rows as the projections leave them
            s[name] = (normal(rows, heads, dim) * (channels[:, 0] if name == "k" else std)).to(s["dtype"])
        elif c["form"] == "nf4":
            s[name + "_pool"], s[name + "_scales"] = _quantized(normal(pages, heads, page, dim) * std)
        else:
            s[name + "_pool"] = (normal(pages, heads, page, dim) * std).to(torch.bfloat16)
    if c["op"] == "attention":
        s["q"] = normal(rows, heads * c["group"], dim).to(s["dtype"])
    return s


# ---- a pass -------------------------------------------------------------------------------------


def _own(s):
    from unifur_b200.kv_cache import CacheBatch, PagedKvCache

    cache = PagedKvCache(s["k_pool"], s["v_pool"], s.get("k_scales"), s.get("v_scales"))
    batch = CacheBatch(s["table"], s["lengths"], s["starts"], s["rows"], max_rows=s["most_rows"], max_length=s["most_tokens"])
    if s["op"] == "attention":
        return cache.attention(s["q"], batch, s["scale"])
    if s["op"] == "read":
        return list(cache.read(batch, s["dtype"]))
    cache.append(s["k"], s["v"], batch)
    return list(cache.read(batch, torch.float32))


def _places(s):
    """The page and the place in it of every row's token."""
    at = torch.arange(s["rows"], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["starts"][1:], at, right=True)
    token = (s["lengths"] - s["starts"][1:])[seq] + at
    return s["table"][seq, token // s["page"]].long(), (token % s["page"]).long()


def _values(s, name, page, place):
    """The cache's values at (page, place) in f32: [..., heads, dim]."""
    if s["form"] == "bf16":
        return s[name + "_pool"][page, :, place].float()
    packed = s[name + "_pool"][page, :, place]
    codes = torch.stack((packed & 15, packed >> 4), -1).flatten(-2)
    values = _levels("cuda", torch.float32)[codes.long()].unflatten(-1, (-1, BLOCK))
    return (values * s[name + "_scales"][page, :, place][..., None]).flatten(-2)


def _plain_append(s, name, page, place):
    if s["form"] == "bf16":
        s[name + "_pool"][page, :, place] = s[name].to(torch.bfloat16)
        return
    blocks = s[name].float().unflatten(-1, (-1, BLOCK))
    scales = blocks.abs().amax(-1)
    quotients = (blocks / scales[..., None]).nan_to_num(0.0)  # a block of zeros has the level 0
    codes = (quotients[..., None] - _levels("cuda", torch.float32)).abs().argmin(-1).flatten(-2).to(torch.uint8)
    s[name + "_pool"][page, :, place] = codes[..., 0::2] | codes[..., 1::2] << 4
    s[name + "_scales"][page, :, place] = scales


def _plain_attention(s):
    starts, lengths = s["starts"].long(), s["lengths"].long()
    counts = starts[1:] - starts[:-1]
    tokens = torch.arange(s["most_tokens"], device="cuda")
    page = s["table"][:, tokens // s["page"]].long().clamp(min=0)
    place = (tokens % s["page"]).expand_as(page)
    k, v = (_values(s, name, page, place).transpose(1, 2) for name in ("k", "v"))  # [sequences, heads, tokens, dim]
    # queries padded to the longest chunk: [sequences, rows, heads, group, dim] -> [sequences, heads, rows * group, dim]
    i = torch.arange(s["most_rows"], device="cuda")
    row = (starts[:-1, None] + i).clamp(max=s["rows"] - 1)
    heads = k.shape[1]
    q = s["q"].float().unflatten(1, (heads, -1))[row].permute(0, 2, 1, 3, 4)
    group = q.shape[3]
    scores = (q.flatten(2, 3) @ k.transpose(2, 3)) * s["scale"]
    last = (lengths - counts)[:, None] + i  # the newest token that a row sees
    seen = (tokens <= last[..., None])[:, None, :, None].expand(-1, heads, -1, group, -1).flatten(2, 3)
    scores = scores.masked_fill_(~seen, -math.inf)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = (weights @ v) / weights.sum(-1, keepdim=True)
    out = out.unflatten(2, (-1, group)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    return out[i < counts[:, None]].to(s["dtype"])


def run(state):
    s = state
    if own:
        return _own(s)
    if s["op"] == "attention":
        return _plain_attention(s)
    page, place = _places(s)
    if s["op"] == "append":
        _plain_append(s, "k", page, place)
        _plain_append(s, "v", page, place)
        return [_values(s, "k", page, place), _values(s, "v", page, place)]
    return [_values(s, "k", page, place).to(s["dtype"]), _values(s, "v", page, place).to(s["dtype"])]


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
    """What the cache holds for values x."""
    if form == "bf16":
        return x.to(torch.bfloat16).double()
    x = x.double()
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


def exact(case, seed):
    s, sizes = prepare(case, seed), _sizes(case)
    if s["op"] == "append":
        # f32 inputs: a quotient next to a border goes by its rounding to f32, which 64 bits do not say
        if s["form"] == "nf4" and s["dtype"] == torch.float32:
            return [None, None]
        return [_exact_stored(s["k"], s["form"]), _exact_stored(s["v"], s["form"])]
    if s["op"] == "read":
        return [torch.cat([_exact_tokens(s, name, i, length - new, length) for i, (length, new) in enumerate(sizes)])
                for name in ("k", "v")]
    parts = []
    for i, (length, new) in enumerate(sizes):
        k, v = _exact_tokens(s, "k", i, 0, length), _exact_tokens(s, "v", i, 0, length)
        at = int(s["starts"][i])
        q = s["q"][at:at + new].double()
        group = q.shape[1] // k.shape[1]
        hidden = torch.ones(new, length, dtype=torch.bool, device="cuda").triu(length - new + 1)
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
    if c["op"] == "append":  # rows in, their storage out; that is read back as f32
        return {"bytes": 2 * rows * (esize * row + stored + 4 * row), "flops": 0}
    if c["op"] == "read":
        return {"bytes": 2 * rows * (stored + esize * row), "flops": 0}
    pairs = sum(new * (length - new) + new * (new + 1) // 2 for length, new in sizes)
    return {"bytes": 2 * tokens * stored + 2 * esize * rows * row * c["group"], "flops": 4 * pairs * row * c["group"]}
