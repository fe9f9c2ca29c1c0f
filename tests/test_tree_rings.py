"""The rings of the kernel for attention of trees over a quantized cache, modelled: three warps copy codes in turn, each to a slot of its own, two groups expand every second
tile to a ring, and the products take the tiles in their order, each at whatever speed.  A wait is for a barrier's parity, as the hardware has it: it passes where the phase
that is under way has the other one, so that a barrier which two waiters come to in turn can let one pass a round early.  Whoever passes must find what it waited for."""
import random

import pytest

LOADERS, GROUPS, WARPS = 3, 2, 4  # warps: of a group


class Barrier:
    def __init__(self, count):
        self.count, self.left, self.phase = count, count, 0

    def arrive(self):
        self.left -= 1
        if self.left == 0:
            self.left, self.phase = self.count, self.phase + 1

    def passes(self, parity):
        return (self.phase & 1) != parity


def run(slots, tiles, seed, barriers_of_slot=2):
    rng = random.Random(seed)
    raw_full = [[Barrier(1) for _ in range(barriers_of_slot)] for _ in range(LOADERS)]
    raw_empty = [Barrier(WARPS) for _ in range(LOADERS)]
    full, empty = [Barrier(WARPS) for _ in range(slots)], [Barrier(1) for _ in range(slots)]
    raw, ring = [None] * LOADERS, [[None] * WARPS for _ in range(slots)]
    reading = [0] * LOADERS  # warps that have taken what is in the slot

    def loader(own):
        for n, tile in enumerate(range(own, tiles, LOADERS)):
            if n:
                yield lambda: raw_empty[own].passes((n + 1) & 1)
            assert raw[own] is None or reading[own] == WARPS, "codes written over before all had them"
            raw[own], reading[own] = None, 0
            yield lambda: True  # (the copies are under way)
            raw[own] = tile
            raw_full[own][tile % barriers_of_slot].arrive()

    def expander(group, warp):
        for tile in range(group, tiles, GROUPS):
            of = tile % LOADERS
            yield lambda: raw_full[of][tile % barriers_of_slot].passes(tile // (LOADERS * barriers_of_slot) & 1)
            assert raw[of] == tile, f"codes of tile {raw[of]} for {tile}"
            yield lambda: True
            assert raw[of] == tile
            reading[of] += 1
            raw_empty[of].arrive()
            slot = tile % slots
            if tile >= slots:
                yield lambda: empty[slot].passes((tile // slots + 1) & 1)
            assert ring[slot][warp] is None or ring[slot][warp][1], "a tile written over before its products"
            yield lambda: True
            ring[slot][warp] = [tile, False]
            full[slot].arrive()

    def products():
        for tile in range(tiles):
            slot = tile % slots
            yield lambda: full[slot].passes(tile // slots & 1)
            assert all(r[0] == tile for r in ring[slot]), "products of a tile that is not there"
            yield lambda: True
            assert all(r[0] == tile for r in ring[slot])
            for r in ring[slot]:
                r[1] = True
            empty[slot].arrive()

    agents = [loader(i) for i in range(LOADERS)] + [expander(g, w) for g in range(GROUPS) for w in range(WARPS)] + [products()]
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
            assert idle < 100000, "nobody gets on"


@pytest.mark.parametrize("slots", [3, 4, 5, 6, 7])
def test_whoever_passes_finds_what_it_waited_for(slots):
    for seed in range(40):
        run(slots, 60, seed)


def test_one_barrier_to_a_slot_would_not_do():
    """With one, a group passes on the round before: the model shows it."""
    with pytest.raises(AssertionError):
        for seed in range(200):
            run(4, 60, seed, barriers_of_slot=1)


def run_small_pages(slots, pieces, seed, holds_back=True):
    """The loaders of a bf16 cache with small pages: four warps to K's tiles and four to V's, which hold a tile back until the next one's copies are under way."""
    rng = random.Random(seed)
    values = []  # of each tile of the ring: is it V's?  K 0, K 1, V 0, K 2, V 1, ..., the last V, piece after piece
    for steps in pieces:
        values += [turn + 1 == 2 * steps or (turn > 0 and turn % 2 == 0) for turn in range(2 * steps)]
    assert all(sum(values[a:b]) == (b - a) // 2 for a, b in [(sum(pieces[:i]) * 2, sum(pieces[:i + 1]) * 2) for i in range(len(pieces))])
    full, empty = [Barrier(4) for _ in range(slots)], [Barrier(1) for _ in range(slots)]
    ring = [[None] * 4 for _ in range(slots)]

    def loader(own, warp):
        pending = None
        for tile, v in enumerate(values):
            if v != own:
                continue
            slot = tile % slots
            if tile >= slots and not empty[slot].passes((tile // slots + 1) & 1):
                if pending is not None and holds_back:
                    yield lambda: True
                    full[pending].arrive()
                    pending = None
                yield lambda: empty[slot].passes((tile // slots + 1) & 1)
            assert ring[slot][warp] is None or ring[slot][warp][1], "a tile written over before its products"
            yield lambda: True
            ring[slot][warp] = [tile, False]
            if pending is not None:
                full[pending].arrive()
            pending = slot
        yield lambda: True
        if pending is not None:
            full[pending].arrive()

    def products():
        for tile in range(len(values)):
            slot = tile % slots
            yield lambda: full[slot].passes(tile // slots & 1)
            assert all(r is not None and r[0] == tile for r in ring[slot]), "products of a tile that is not there"
            yield lambda: True
            for r in ring[slot]:
                r[1] = True
            empty[slot].arrive()

    agents = [loader(own, warp) for own in (False, True) for warp in range(4)] + [products()]
    waits = {a: next(a, None) for a in agents}
    idle = 0
    while waits:
        a = rng.choice(list(waits))
        if waits[a] is None:
            del waits[a]
        elif waits[a]():
            idle = 0
            waits[a] = next(a, None)
        else:
            idle += 1
            assert idle < 5000, "nobody gets on"


PIECES = [[1], [1, 1, 1, 1, 1], [7, 1, 2, 1, 9], [30], [3, 4, 3, 1, 1, 12]]


@pytest.mark.parametrize("slots", [5, 6, 7])
@pytest.mark.parametrize("pieces", PIECES)
def test_small_pages_get_on_and_come_in_order(slots, pieces):
    for seed in range(20):
        run_small_pages(slots, pieces, seed)


def test_a_tile_held_back_over_a_wait_would_stop_all():
    """In a ring of two places (of one the parities would say nothing): the loader would wait for products of the tile that it has not given yet."""
    with pytest.raises(AssertionError, match="nobody gets on"):
        run_small_pages(2, [1, 1, 1], 0, holds_back=False)
