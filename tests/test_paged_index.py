"""The split of a paged attention's keys into work items, restated on the CPU
(plugins_amd/csrc/paged_ops.hip: split_of, find_work): every key of every tile
is in one item, items and split tiles stay within what the host sized the launch
and the scratch for, whatever the lengths -- in the kernel's own 32-bit sums."""
import random

import numpy as np
import pytest

F = np.float32
CUS = 256


def split_of(kv, group, rows, seqs, max_rows):
    pairs = max_rows * group
    tile = 4 if pairs <= 16 else 5 if pairs <= 32 else 7
    n = (2 * CUS + kv - 1) // kv
    few = n // 2 if pairs <= 32 else 3 * n // 8
    most = 4 * n if pairs <= 32 else n + n // 2
    tiles = ((rows * group) >> tile) + seqs
    return dict(group=group, tile=tile, least=2 if pairs <= 32 else 4, round=n, few=few, most=most,
                whole=F(F(0.9 if pairs <= 32 else 1.4) / F(n)), more=F(4.5 if pairs <= 32 else 8),
                items=n if tiles <= few else tiles + most,
                split=min(tiles, n if tiles <= few else most))


def butterfly(lanes):
    v = lanes.copy()
    for m in (1, 2, 4, 8, 16, 32):
        v = (v + v[np.arange(64) ^ m]).astype(F)
    assert (v == v[0]).all()
    return v[0]


def items_of(sl, counts, lens):
    """[(sequence, tile, k0, k1)], split tiles."""
    units, tiles = np.zeros(64, F), np.zeros(64, F)
    nt = [(n * sl["group"] + (1 << sl["tile"]) - 1) >> sl["tile"] for n in counts]
    un = [(n + c + 63) >> 6 for n, c in zip(counts, lens)]
    for s, (t, u) in enumerate(zip(nt, un)):
        units[s % 64] = F(units[s % 64] + F(F(t) * F(u)))
        tiles[s % 64] = F(tiles[s % 64] + F(t))
    units, tiles = butterfly(units), butterfly(tiles)
    few = tiles <= F(sl["few"])
    target = F(sl["round"]) - tiles if few else F(sl["most"])
    assert target > 0
    longest = max([u for t, u in zip(nt, un) if t > 0], default=0)
    spare = F(np.floor(F(0.5) * F(sl["round"])) - tiles)
    out = []
    # reciprocals are right to one unit in the last place either way: both ends
    for to in (F(0), F(np.inf)):
        r, rs = (np.nextafter(F(1) / x if x else F(np.inf), to) for x in (max(tiles, F(1)), spare))
        half = np.ceil(F(units * rs)) if spare > 0 else F(0)
        least = max(F(sl["least"] if few else 4),
                    half if spare > 0 and half <= 16 else
                    min(F(8), np.floor(F(F(units * F(0.0625)) * r))))
        whole = F(longest) <= F(F(sl["whole"] * units) + sl["more"])
        chunk = int(min(max(F(1 << 25) if whole else
                            np.ceil(F(F(units * F(1 + 2.0 ** -12)) / target)), least), F(1 << 25)))
        items, split = [], 0
        for s, (t, u) in enumerate(zip(nt, un)):
            if t == 0:
                continue
            ns = (u + chunk - 1) // chunk
            each = (u + ns - 1) // ns
            split += t if ns > 1 else 0
            end = counts[s] + lens[s]
            for x in range(t * ns):
                j, i = divmod(x, t)
                items.append((s, t - 1 - i, min(j * each * 64, end), min((j + 1) * each * 64, end)))
        out.append((items, split))
    return out


def check(kv, group, counts, lens):
    sl = split_of(kv, group, sum(counts), len(counts), max(counts))
    for items, split in items_of(sl, counts, lens):
        assert len(items) <= sl["items"] and split <= sl["split"], (len(items), split, sl)
        at = {}
        for s, tile, k0, k1 in items:
            assert at.get((s, tile), 0) == k0 <= k1 and k0 % 64 in (0, k0 if k0 == k1 else 0)
            at[s, tile] = k1
        for (s, tile), end in at.items():
            assert end == counts[s] + lens[s]
        assert len(at) == sum((n * group + (1 << sl["tile"]) - 1) >> sl["tile"] for n in counts)


@pytest.mark.parametrize("seed", range(60))
def test_items_cover_every_key_once_within_their_bounds(seed):
    rng = random.Random(seed)
    seqs = rng.choice([1, 1, 2, 5, 17, 63, 64, 65, 130, 500])
    most = rng.choice([1, 1, 2, 4, 8, 33, 64, 300, 2000])
    ctx = rng.choice([0, 1, 63, 100, 5000, 200000, 3000000])
    counts = [rng.randint(0, most) for _ in range(seqs)]
    counts[rng.randrange(seqs)] = most
    lens = [rng.randint(0, ctx) if rng.random() < 0.8 else 0 for _ in range(seqs)]
    check(rng.choice([1, 2, 3, 8, 16, 200, 600]), rng.choice([1, 2, 3, 4, 5, 8, 16]), counts, lens)


def test_items_of_the_largest_batches():
    check(8, 4, [1] * 60000, [7] * 60000)
    check(1, 1, [1], [(1 << 30) - 1])
    check(2, 4, [1 << 20], [(1 << 30) - (1 << 20)])
    check(1, 8, [1] * 63 + [1024], [1 << 24] * 64)


def test_sequences_that_share_rows_pass_the_bounds():
    """Why a step whose cu goes back is not begun: 300 rows taken 20 times over
    are more items than the launch has, and the joins of the last ones are never
    filled in."""
    sl = split_of(8, 4, 300, 40, 300)
    for items, split in items_of(sl, [300, 0] * 20, [0] * 38 + [60000, 0]):
        at = [i for i, x in enumerate(items) if x[0] == 38]
        assert split > 0 and len(at) > 1 and at[0] >= sl["items"]


def parts_of(sl):
    """Items of split tiles that the scratch has places for, of a kv head."""
    few = sl["items"] == sl["round"]
    return sl["round"] if few else sl["most"] + sl["split"]


def check_parts(kv, group, counts, lens):
    sl = split_of(kv, group, sum(counts), len(counts), max(counts))
    for items, split in items_of(sl, counts, lens):
        of = {}
        for s, tile, _, _ in items:
            of[s, tile] = of.get((s, tile), 0) + 1
        assert sum(n for n in of.values() if n > 1) <= parts_of(sl)
        assert sum(n > 1 for n in of.values()) == split


@pytest.mark.parametrize("seed", range(60))
def test_parts_of_split_tiles_fit_the_scratch(seed):
    rng = random.Random(1000 + seed)
    seqs = rng.choice([1, 1, 2, 5, 17, 63, 64, 65, 130, 500])
    most = rng.choice([1, 1, 2, 4, 8, 33, 64, 300, 2000])
    ctx = rng.choice([0, 100, 5000, 200000, 3000000])
    counts = [rng.randint(0, most) for _ in range(seqs)]
    counts[rng.randrange(seqs)] = most
    lens = [rng.randint(0, ctx) if rng.random() < 0.8 else 0 for _ in range(seqs)]
    check_parts(rng.choice([1, 2, 3, 8, 16, 200, 600]), rng.choice([1, 2, 3, 4, 5, 8, 16]), counts, lens)


def test_parts_of_the_largest_batches():
    check_parts(8, 4, [1] * 60000, [7] * 60000)
    check_parts(1, 1, [1], [(1 << 30) - 1])
    check_parts(2, 4, [1 << 20], [(1 << 30) - (1 << 20)])
    check_parts(1, 8, [1] * 63 + [1024], [1 << 24] * 64)
    check_parts(8, 4, [2000] * 20, [0] * 19 + [3000000])


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kv,group", [(1, 8), (8, 4), (64, 1)])
def test_scratch_does_not_grow_with_the_rows(kv, group, dim):
    """Whole tiles leave nothing behind: a prompt of any length, or any number of
    sequences, takes what split tiles can."""
    import ctypes

    from plugins_amd import exl3 as X
    from plugins_amd import paged as P
    c = P.CacheDesc(ctypes.sizeof(P.CacheDesc), X.DT_F16, 4096, 8192, 1, 1 << 20, kv, 16, dim, 60000,
                    1 << 20, 64)

    def need(seqs, rows, most):
        r = P.RowsDesc(ctypes.sizeof(P.RowsDesc), seqs, rows, most, 64, 64)
        return P.paged_lib().exl3p_attend_scratch_bytes(ctypes.byref(c), ctypes.byref(r), kv * group)

    for seqs, rows, most in ((1, 7, 7), (1, 300, 300), (1, 131072, 131072), (4, 8000, 2000),
                             (64, 64, 1), (60000, 60000, 1), (1, 1 << 24, 1 << 24), (500, 4000, 8)):
        sl = split_of(kv, group, rows, seqs, most)
        assert need(seqs, rows, most) == 32 * (1 + sl["split"]) + \
            parts_of(sl) * kv * (1 << sl["tile"]) * (dim + 2) * 4
        assert need(seqs, rows, most) < 128 << 20
