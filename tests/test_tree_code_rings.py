"""The kernel for attention of trees over a quantized cache, modelled as far as its barriers go, with the depths that its source has: warps that copy codes, groups of warps that
expand them, the warp that issues products, the softmax warps; and beside the rings of tiles the short ones that say which power of two a step's scales were divided by and whether a
page was missing.  Every wait is for a barrier's parity, as the hardware has it.  Whoever passes must find what it waited for."""
import os
import random
import re

import pytest

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "unifur_b200", "csrc", "attention_tree.cu")


def number(pattern):
    with open(SOURCE) as f:
        found = re.findall(pattern, f.read())
    assert len(found) == 1, pattern
    return int(found[0])


LOADERS = number(r"kLoaders = (\d+);")
EXPANDERS = number(r"kExpandWarps = (\d+)")   # of a group
GROUPS = (number(r"kCopyWarp = (\d+)") - number(r"kExpandWarp = (\d+)")) // EXPANDERS
POWERS = number(r"float2 s_powers\[(\d+)\]")
BAD = number(r"s_bad\[(\d+)\], s_first")
SOFTMAX = 3  # (warps of unlike speed; the kernel has eight, or four)


class Barrier:
    def __init__(self, count):
        self.count, self.left, self.phase = count, count, 0

    def arrive(self):
        self.left -= 1
        if self.left == 0:
            self.left, self.phase = self.count, self.phase + 1

    def passes(self, parity):
        return (self.phase & 1) != parity


def turns(pieces):
    """The tiles in their order: (piece, step of all, is it values?): K 0, K 1, V 0, K 2, V 1, ..., the last V, piece after piece."""
    first = 0
    for piece, steps in enumerate(pieces):
        order = [(0, 0)]
        for j in range(steps):
            order += [(j + 1, 0)] * (j + 1 < steps) + [(j, 1)]
        assert sorted(order) == [(j, v) for j in range(steps) for v in (0, 1)]
        for j, values in order:
            yield piece, first + j, values
        first += steps


def run(slots, pieces, seed, ahead=False, lost=(), powers=POWERS, bad=BAD, barriers_of_slot=2, early=False):
    """`ahead`: one warp copies tiles as they are; `lost`: pieces with a page that there is not; `early`: an expander gives codes back before it has them."""
    rng = random.Random(seed)
    tiles = list(turns(pieces))
    raw_full = [[Barrier(1) for _ in range(barriers_of_slot)] for _ in range(LOADERS)]
    raw_empty = [Barrier(EXPANDERS) for _ in range(LOADERS)]
    writers = 1 if ahead else EXPANDERS
    full, empty = [Barrier(writers) for _ in range(slots)], [Barrier(1) for _ in range(slots)]
    s_full, p_ready = [Barrier(1) for _ in range(2)], [Barrier(SOFTMAX) for _ in range(2)]
    q_ready, o_done = Barrier(SOFTMAX), Barrier(1)
    raw, taken, ring = [None] * LOADERS, [EXPANDERS] * LOADERS, [[(None, True)] * writers for _ in range(slots)]
    s_powers, s_bad = [None] * powers, [0] * bad

    def loader(own):
        for n, tile in enumerate(range(own, len(tiles), LOADERS)):
            piece, step, values = tiles[tile]
            if piece in lost:
                s_bad[piece % bad] = piece + 1
            if n:
                yield lambda: raw_empty[own].passes((n + 1) & 1)
            assert taken[own] == EXPANDERS, "codes written over before all had them"
            raw[own], taken[own] = None, 0
            yield lambda: True  # (the copies are under way)
            raw[own] = tile
            if not values:
                s_powers[step % powers] = step
            raw_full[own][tile % barriers_of_slot].arrive()

    def expander(group, warp):
        for tile in range(group, len(tiles), GROUPS):
            of, slot = tile % LOADERS, tile % slots
            yield lambda: raw_full[of][tile % barriers_of_slot].passes(tile // (LOADERS * barriers_of_slot) & 1)
            assert raw[of] == tile, f"codes of tile {raw[of]} for {tile}"
            if early:
                taken[of] += 1
                raw_empty[of].arrive()
            if tile >= slots:
                yield lambda: empty[slot].passes((tile // slots + 1) & 1)
            assert ring[slot][warp][1], "a tile written over before its products"
            yield lambda: True  # (looked up and written, from codes that are read till the end)
            assert raw[of] == tile, "codes written over while they are read"
            ring[slot][warp] = (tile, False)
            full[slot].arrive()
            if not early:
                taken[of] += 1
                raw_empty[of].arrive()

    def copier():
        for tile, (piece, step, values) in enumerate(tiles):
            slot = tile % slots
            if not values:
                if piece in lost:
                    s_bad[piece % bad] = piece + 1
                s_powers[step % powers] = step
            if tile >= slots:
                yield lambda: empty[slot].passes((tile // slots + 1) & 1)
            assert ring[slot][0][1], "a tile written over before its products"
            yield lambda: True
            ring[slot][0] = (tile, False)
            full[slot].arrive()

    def products():
        waits_q = used = 0
        for tile, (piece, step, values) in enumerate(tiles):
            slot = tile % slots
            yield lambda: full[slot].passes(tile // slots & 1)
            if not values and (tile == 0 or tiles[tile - 1][0] != piece):
                yield lambda: q_ready.passes(waits_q & 1)
                waits_q += 1
            if values:
                yield lambda: p_ready[used & 1].passes(used // 2 & 1)
                used += 1
            assert all(t == tile for t, _ in ring[slot]), "products of a tile that is not there"
            yield lambda: True
            assert all(t == tile for t, _ in ring[slot])
            ring[slot] = [(t, True) for t, _ in ring[slot]]
            if not values:
                s_full[step & 1].arrive()
            elif tile + 1 == len(tiles) or tiles[tile + 1][0] != piece:
                o_done.arrive()
            empty[slot].arrive()

    def softmax():
        step = 0
        for piece, steps in enumerate(pieces):
            yield lambda: True
            q_ready.arrive()
            for step in range(step, step + steps):
                yield lambda: s_full[step & 1].passes(step // 2 & 1)
                yield lambda: True
                assert s_powers[step % powers] == step, "another step's power of two"
                yield lambda: True
                p_ready[step & 1].arrive()
            step += 1
            yield lambda: o_done.passes(piece & 1)
            yield lambda: True
            assert (s_bad[piece % bad] == piece + 1) == (piece in lost), "a missing page of another piece, or one that was forgotten"

    agents = [products()] + [softmax() for _ in range(SOFTMAX)]
    agents += [copier()] if ahead else [loader(i) for i in range(LOADERS)] + [expander(g, w) for g in range(GROUPS) for w in range(EXPANDERS)]
    waits = {a: next(a, None) for a in agents}
    slow = {a: rng.random() ** 3 + 0.01 for a in agents}
    idle = 0
    while waits:
        a = rng.choices(list(waits), [slow[a] for a in waits])[0]
        if rng.random() < 0.01:
            slow[a] = rng.random() ** 3 + 0.01
        if waits[a] is None:
            del waits[a]
        elif waits[a]():
            idle = 0
            waits[a] = next(a, None)
        else:
            idle += 1
            assert idle < 20000, "nobody gets on"


PIECES = [[1] * 30, [30], [7, 1, 2, 1, 9, 1, 1, 5], [3, 4, 3, 1, 1, 12], [2] * 15]
LOST = [(), (0, 3, 4, 8, 9, 10, 17)]


def test_the_source_is_what_is_modelled():
    assert (LOADERS, GROUPS, EXPANDERS) == (3, 2, 4) and POWERS == BAD == 8
    with open(SOURCE) as f:
        text = f.read()
    assert f"s_powers[t.info & {POWERS - 1}u] = powers" in text and f"s_powers[(step + j) & {POWERS - 1}u] = powers" in text
    assert f"s_powers + ((step + j) & {POWERS - 1}u)" in text
    # marks of missing pages: of the codes' loaders, of small pages, of tiles that come as they are, and where they are looked at
    assert text.count(f"& {BAD - 1}u] = ") - text.count("s_powers[t.info") - text.count("s_powers[(step + j)") == 4
    assert f"s_bad[piece & {BAD - 1}u] == piece + 1" in text


@pytest.mark.parametrize("lost", LOST)
@pytest.mark.parametrize("pieces", PIECES)
@pytest.mark.parametrize("slots", [3, 6])
def test_whoever_passes_finds_what_it_waited_for(slots, pieces, lost):
    for seed in range(12):
        run(slots, pieces, seed, lost=lost)


@pytest.mark.parametrize("lost", LOST)
@pytest.mark.parametrize("pieces", PIECES)
@pytest.mark.parametrize("slots", [4, 7])
def test_a_cache_that_is_expanded_ahead(slots, pieces, lost):
    for seed in range(12):
        run(slots, pieces, seed, ahead=True, lost=lost)


@pytest.mark.parametrize("slots,changed,word", [
    (4, {"barriers_of_slot": 1}, "codes of tile"), (4, {"early": True}, "written over while they are read"), (6, {"powers": 4}, "another step's power"),
    (6, {"bad": 6}, "of another piece"), (7, {"ahead": True, "powers": 4}, "another step's power"), (7, {"ahead": True, "bad": 4}, "of another piece")])
def test_the_model_sees_what_is_too_little(slots, changed, word):
    pieces = [1] * 40 if "bad" in changed else [20, 20]
    with pytest.raises(AssertionError, match=word):
        for seed in range(400):
            run(slots, pieces, seed, lost=range(0, 40, 2) if "bad" in changed else (), **changed)
