"""The decode kernel's division of tiles into runs, in Python: whatever the
lengths, the pieces that the joining CTA counts and reads are those that the runs
leave, each in a slot of its own."""
import random

import pytest

TILE, JOIN = 64, 16   # (the tile is 128 with head_dim 64; the rule is the same)


def run_start(total, c, g):
    return total * c // g


def run_of(total, x, g):
    return ((x + 1) * g - 1) // total


def pieces_of(total, begin, tiles, g):
    return tiles if total < g else run_of(total, begin + tiles - 1, g) - run_of(total, begin, g) + 1


def piece_slot(total, begin, i, g):
    r = run_of(total, begin + i, g) if total < g else run_of(total, begin, g) + i
    return 2 * r + (i == 0)


@pytest.mark.parametrize("seed", range(40))
def test_pieces_are_those_the_runs_leave(seed):
    rng = random.Random(seed)
    g = rng.choice([1, 2, 7, 148, 296])
    per_seq = rng.choice([1, 2, 8])
    lens = [rng.choice([0, 1, 63, 64, 65, rng.randrange(1, 5000), rng.randrange(1, 200)]) for _ in range(rng.randrange(1, 90))]
    if seed % 4 == 0:
        lens[rng.randrange(len(lens))] = 131072
    units = [max(1, -(-x // TILE)) for x in lens for _ in range(per_seq)]
    total = sum(units)
    begins = [sum(units[:i]) for i in range(len(units))]
    left = {}          # unit -> slots its pieces are left in, in order
    used = set()
    for c in range(g):
        t, t1 = run_start(total, c, g), run_start(total, c + 1, g)
        while t < t1:
            u = max(i for i, b in enumerate(begins) if b <= t)
            tile0, tile1 = t - begins[u], min(units[u], t1 - begins[u])
            if not (tile0 == 0 and tile1 == units[u]):
                slot = 2 * c + (tile0 == 0)
                assert slot not in used
                used.add(slot)
                mine = tile0 if total < g else c - run_of(total, begins[u], g)
                assert mine == len(left.setdefault(u, []))
                left[u].append(slot)
            t += tile1 - tile0
    for u, slots in left.items():
        n = pieces_of(total, begins[u], units[u], g)
        assert slots == [piece_slot(total, begins[u], i, g) for i in range(n)]
        groups = -(-n // JOIN)
        assert groups <= 32
        # the slots that a group's count and joined partial live in are the group's own
        firsts = [slots[i] for i in range(0, n, JOIN)]
        assert len(set(firsts)) == groups


def test_run_of_is_the_run_that_holds_a_tile():
    for total in (1, 2, 5, 147, 148, 149, 1000, 12345):
        for g in (1, 3, 148, 296):
            for x in range(0, total, max(1, total // 97)):
                c = run_of(total, x, g)
                assert run_start(total, c, g) <= x < run_start(total, c + 1, g)
