"""How the paged kernels divide their work, from the kernels' own arithmetic
(paged_split.h through the library's qwen_paged_* hooks; no GPU): every tile is taken
once, pieces have slots of their own, and the joins read the slots that were written."""
import ctypes
import random

import pytest

from qweninferenceengine_b200 import _lib

L = ctypes.CDLL(_lib.LIB_PATH)
L.qwen_paged_run_start.restype = ctypes.c_uint
U, I = ctypes.c_uint, ctypes.c_int
TILE, JOIN = 64, 16


def run_start(total, c, g):
    return L.qwen_paged_run_start(U(total), U(c), U(g))


def run_of(total, x, g):
    return L.qwen_paged_run_of(U(total), U(x), U(g))


def cut_piece(total, begin, tiles, tile0, c, g):
    piece, slots = I(), (I * 512)()
    n = L.qwen_paged_cut_piece(U(total), U(begin), U(tiles), U(tile0), I(c), U(g), ctypes.byref(piece), slots, I(512))
    assert n <= 512
    return piece.value, list(slots[:n])


# ---------------------------------------------------------- k_paged_decode ---
@pytest.mark.parametrize("g", [1, 2, 7, 59, 118, 148, 296])
def test_runs_near_the_largest_number_of_tiles(g):
    rng = random.Random(g)
    for total in [0, 1, g - 1, g, g + 1, 2 ** 31 - 1, 2 ** 31 - g] + [rng.randrange(2 ** 31) for _ in range(50)]:
        starts = [run_start(total, c, g) for c in range(g + 1)]
        assert starts == [total * c // g for c in range(g + 1)]
        for x in {0, total - 1, total // 2, *starts, *[s - 1 for s in starts]}:
            if 0 <= x < total:
                c = run_of(total, x, g)
                assert starts[c] <= x < starts[c + 1]


def walk(units, g):
    """The kernel's walk: (run, unit, tile0, tile1) of every piece."""
    begins, at = [], 0
    for tiles in units:
        begins.append(at)
        at += tiles
    for c in range(g):
        t, t1, u = run_start(at, c, g), run_start(at, c + 1, g), 0
        while t < t1:
            while t >= begins[u] + units[u]:
                u += 1
            tile0, tile1 = t - begins[u], min(units[u], t1 - begins[u])
            yield c, u, begins[u], tile0, tile1
            t += tile1 - tile0


@pytest.mark.parametrize("seed", range(60))
def test_pieces_and_their_slots(seed):
    rng = random.Random(seed)
    g = rng.choice([1, 2, 7, 118, 148, 296])
    per_seq = rng.choice([1, 2, 8, 64])
    lens = [rng.choice([0, 1, 63, 64, 65, rng.randrange(1, 5000), rng.randrange(1, 200)])
            for _ in range(rng.choice([1, 2, 9, 90, 400]))]
    if seed % 4 == 0:
        lens[rng.randrange(len(lens))] = 131072
    units = [max(1, -(-x // TILE)) for x in lens for _ in range(per_seq)]
    total, taken, left, says, used = sum(units), [0] * len(units), {}, {}, set()
    for c, u, begin, tile0, tile1 in walk(units, g):
        assert taken[u] == tile0
        taken[u] = tile1
        if tile0 == 0 and tile1 == units[u]:
            continue
        slot = 2 * c + (tile0 == 0)
        piece, slots = cut_piece(total, begin, units[u], tile0, c, g)
        assert slot not in used and 0 <= slot < 2 * g
        used.add(slot)
        assert piece == len(left.setdefault(u, []))
        left[u].append(slot)
        assert says.setdefault(u, slots) == slots   # all of a unit's runs count alike
    assert taken == units
    for u, slots in left.items():
        assert slots == says[u]
        groups = -(-len(slots) // JOIN)
        assert groups <= 32
        assert len({slots[i] for i in range(0, len(slots), JOIN)}) == groups


# ---------------------------------------------------------------- k_prefix ---
def prefix(kv_heads, n_seq, n_heads, length, sms=148):
    plan, n, cap = (I * 5)(), I(), 1 << 17
    rows = (I * (7 * cap))()
    args = (I(kv_heads), I(n_seq), I(n_heads), U(length), I(sms))
    g = L.qwen_paged_prefix_pieces(*args, plan, rows, I(cap), ctypes.byref(n))
    assert n.value <= cap
    pieces = [tuple(rows[7 * i:7 * i + 7]) for i in range(n.value)]
    tiles = plan[0]
    slots, joins = (I * 4096)(), {}
    for h in range(kv_heads):
        for tile in range(tiles):
            m = L.qwen_paged_prefix_partials(*args, I(h), I(tile), slots, I(4096))
            assert m <= 4096
            joins[h, tile] = list(slots[:m])
    return g, list(plan), pieces, joins


def check_prefix(kv_heads, n_seq, n_heads, length, sms=148):
    g, (tiles, pairs, steps, share2, share1), pieces, joins = prefix(kv_heads, n_seq, n_heads, length, sms)
    assert 1 <= g <= sms and tiles == -(-n_seq * (n_heads // kv_heads) // 128) and steps == -(-length // 128)
    taken, wrote = {}, {}
    for c, h, pair, w, i0, i1, piece_id in pieces:
        assert 0 <= c < g and 0 <= h < kv_heads and 0 <= pair < pairs and 0 <= i0 < i1 <= steps
        assert w == (2 if 2 * pair + 1 < tiles else 1)
        assert taken.get((h, pair), 0) == i0   # a unit's steps, each once, in the order of its pieces
        taken[h, pair] = i1
        assert 0 <= piece_id < kv_heads * pairs + g   # the workspace's slots
        for stream in range(2):
            tile = 2 * pair + stream if w == 2 else 2 * pair
            wrote.setdefault((h, tile), []).append(2 * piece_id + stream)
    assert set(taken) == {(h, pair) for h in range(kv_heads) for pair in range(pairs)}
    assert all(x == steps for x in taken.values())
    every = [x for v in wrote.values() for x in v]
    assert len(set(every)) == len(every)
    assert wrote == joins
    return g, share2, pieces


# Units with CTAs of their own, and (the later ones) more units than the prefix's SMs.
SIZES = [(2, 1, 12, 5000), (2, 8, 12, 1000), (8, 64, 32, 8704), (2, 256, 12, 32768), (1, 1, 1, 1), (2, 65, 128, 3333),
         (8, 256, 64, 1000), (8, 400, 32, 1000), (8, 517, 32, 129), (2, 1024, 12, 4096), (2, 1100, 12, 77),
         (8, 1300, 16, 700), (2, 2048, 14, 300), (64, 160, 64, 515), (128, 100, 128, 2049), (1024, 1, 1024, 1),
         (1024, 129, 1024, 1000), (1, 65535, 1, 1 << 14), (3, 700, 96, 1 << 17)]


@pytest.mark.parametrize("size", SIZES)
def test_prefix_steps_and_partials(size):
    check_prefix(*size)


def test_both_divisions_are_among_them():
    shares, spanning = set(), 0
    for size in SIZES:
        g, share2, pieces = check_prefix(*size)
        shares.add(share2 > 0)
        spanning += len({p[0] for p in pieces}) < len(pieces)   # a CTA with more than one piece
    assert shares == {True, False} and spanning > 5


@pytest.mark.parametrize("seed", range(40))
def test_prefix_of_any_size(seed):
    rng = random.Random(seed)
    kv_heads = rng.choice([1, 2, 3, 8, 40, 128])
    group = rng.choice([1, 2, 6, 7, 64])
    n_seq = max(1, int(2 ** rng.uniform(0, 11)) // max(1, kv_heads * group // 64))
    check_prefix(kv_heads, n_seq, kv_heads * group, int(2 ** rng.uniform(0, 17)), rng.choice([148, 132, 20]))
