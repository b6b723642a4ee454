"""Weights of keys: a row's weights add up to one however large its scores are, whichever
path its pairs take; deals of several tiles and more items than a launch has workgroups;
what a row that saw a bad key leaves alone."""
import math

import pytest

torch = pytest.importorskip("torch")

from plugins_amd import paged as P  # noqa: E402
from tests import _budget as B  # noqa: E402
from tests import _paged as R  # noqa: E402
from tests.test_gpu_budget import scores, weighed  # noqa: E402
from tests.test_gpu_paged import batch  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("dtype,size", [(F16, 8), (F16, 64), (F16, 96), (F16, 512), (BF16, 32), (BF16, 128)])
@pytest.mark.parametrize("n,group,window", [(1, 4, 0), (8, 4, 0), (9, 4, 0), (40, 1, 0), (129, 3, 0), (200, 2, 33)])
def test_weights_of_large_scores_add_up(n, group, window, dtype, size):
    """Scores of 63 * 64 size (2^19 for 128) and a few more, whole numbers that 32 bits hold:
    what differs between a row's keys is those few (at most 10), so a weight is as exact
    as one of small scores: powers and the sum of `keys` terms (keys + 64) 2^-23, the
    scale's own rounding 10 * 2^-24 log2(e).  Scores of 2^20 powers of two and more are
    rounded when they are scaled, and those of up to 32 pairs are always: there all keys of
    a row are alike, and their scores too."""
    counts, lens, page = [n, 3], [300, 70], 16
    g, k, v, table, cu, _ = batch(counts, lens, dtype, 2, group, 64, page, 3)
    pairs = (window or n) * group
    alike = pairs <= 32 or 63 * 64 * size * 1.4427 * 2 >= 2 ** 20
    k = torch.full_like(k, size)
    q = torch.full((sum(counts), 2 * group, 64), 64.0).to(dtype)
    k[..., 0] = 0 if alike else torch.randint(0, 6, k.shape[:-1], generator=g).to(dtype)
    q[..., 0] = torch.randint(0, 3, q.shape[:-1], generator=g).to(dtype)
    seen = [[list(range(i + 1)) for i in range(m)] for m in counts]
    had = torch.zeros(2, 2, 600)
    want, _ = B.weights(q, k, table, cu, lens, seen, page, group, 1.0, had, 1.0, window)
    got = weighed(k, table, counts, lens, q, had, scale=1.0, window=window).double()
    off = (got - want).abs() - want * ((300 + n + 64) * 2.0 ** -23 + 10 * 1.5 * 2.0 ** -24 + (pairs + 4) * 2.0 ** -24)
    assert float(off.max()) <= 2.0 ** -100
    total = got[0].sum(-1)
    assert ((total / pairs - 1).abs() < 1e-4).all()


def close(got, want, tol):
    off = (got.double() - want).abs() - tol
    assert not torch.isnan(got).any() and float(off.max()) <= 0, float(off.max())


@pytest.mark.parametrize("room", [900, 2_200_000, 5_000_000])
def test_deals_of_several_tiles(room):
    """256 rows of 4 heads a kv head are 8 tiles of 128 pairs; the sums of as many deals over
    the larger rooms would take more than 2^28 bytes, so a deal has two tiles, or four."""
    counts, lens = [256, 130], [300, 64 * 9 + 5]
    g, k, v, table, cu, q = batch(counts, lens, BF16, 2, 4, 64, 32, 5)
    seen = [[list(range(i + 1)) for i in range(n)] for n in counts]
    had = scores(2, 2, 900, g)
    want, tol = B.weights(q, k, table, cu, lens, seen, 32, 4, 0.125, had, 0.9)
    full = torch.full((2, 2, room), 5.0)
    full[..., :900] = had
    got = weighed(k, table, counts, lens, q, full, decay=0.9)
    close(got[..., :900], want, tol)
    assert (got[..., 900:] == 5.0).all()
    # masks: rows that see nothing of some tiles' keys
    free = [[[j for j in range(n) if torch.rand(1, generator=g) < 0.2] for _ in range(n)] for n in counts]
    mask = R.masks([js for s in free for js in s], 4)
    want, tol = B.weights(q, k, table, cu, lens, free, 32, 4, 0.125, had, 0.9)
    close(weighed(k, table, counts, lens, q, full, mask, decay=0.9)[..., :900], want, tol)


@pytest.mark.parametrize("ctx,room", [(21000, 21300), (100000, 270000)])
def test_more_items_than_workgroups(ctx, room):
    """Over 256 CUs, 64 kv heads leave each 32 workgroups and one for each of at most 9 tiles; 8
    deals of 333 units of 64 keys in parts of 64 at most are 48 items, so workgroups come
    round again, and so they do for 2 deals of four tiles and 1567 units, 50 items."""
    n, kv, group, dim, page = 256, 64, 4, 64, 256
    g = torch.Generator(device=DEV).manual_seed(3)
    pages = -(-(ctx + n) // page)
    k = torch.randn(1, pages + 1, kv, page, dim, generator=g, device=DEV).to(F16)
    table = torch.randperm(pages + 1, generator=g, device=DEV)[None, :pages].int()
    q = torch.randn(n, kv * group * dim, generator=g, device=DEV).to(F16)
    score = torch.zeros(1, kv, room, device=DEV)
    P.weigh(P.PagedCache.over(k, torch.empty_like(k), table.contiguous()), 0, P.Rows.of([n], [ctx], DEV), q, score)
    at = torch.arange(ctx + n, device=DEV)
    hide = at[None] > ctx + torch.arange(n, device=DEV)[:, None]
    for h in (0, 1, 37, 63):
        keys = k[0, table[0, at // page].long(), h, at % page].double()
        total, tol = torch.zeros(ctx + n, dtype=torch.float64, device=DEV), 0.0
        for x in range(h * group, (h + 1) * group):
            mine = q[:, x * dim:(x + 1) * dim].double()
            s = (mine @ keys.T * 0.125).masked_fill(hide, -math.inf)
            w = torch.softmax(s, -1)
            es = (mine.abs() @ keys.abs().T).amax(-1) * 0.125 * (dim + 4) * 2.0 ** -24
            total += w.sum(0)
            tol = tol + (w * (2.4 * es + (ctx + n + 64) * 2.0 ** -23)[:, None]).sum(0)
        tol = tol + (n * group + 4) * 2.0 ** -24 * total + n * group * 2.0 ** -120
        off = (score[0, h, :ctx + n].double() - total).abs() - tol
        assert float(off.max()) <= 0, h
    assert not score[..., ctx + n:].any()


@pytest.mark.parametrize("what", [math.nan, math.inf])
@pytest.mark.parametrize("n,group", [(3, 4), (8, 4), (11, 4), (40, 4), (64, 3)])
def test_what_a_row_with_a_bad_key_touches(what, n, group):
    """Two branches, one under a row whose key is NaN or infinite: a key's weight is NaN
    exactly where a row that sees it also sees that one; every other key's is the formula's,
    its rows' alone."""
    counts, lens, page = [n], [20], 16
    g, k, v, table, cu, q = batch(counts, lens, BF16, 2, group, 128, page, 6)
    parents = [-1] + [max(0, i - 2) for i in range(1, n)]
    parents[2:] = [-1 if i == 2 else p for i, p in enumerate(parents)][2:]  # row 2 begins a tree of its own
    seen = [R.ancestors(parents)]
    mask = R.masks(seen[0], 1)
    pg, row = R.slots(table, 0, page, 20 + n)
    k[0, pg[21], :, row[21]] = what
    had = scores(1, 2, 100, g)
    got = weighed(k, table, counts, lens, q, had, mask)
    bad = [i for i in range(n) if 1 in seen[0][i]]
    hit = {20 + j for i in bad for j in seen[0][i]} | set(range(20))
    clean = k.clone()
    clean[0, pg[21], :, row[21]] = 0
    want, tol = B.weights(q, clean, table, cu, lens, seen, page, group, 1 / math.sqrt(128), had)
    for x in range(20 + n):
        if x in hit:
            assert torch.isnan(got[0, :, x]).all(), x
        else:
            assert ((got[0, :, x].double() - want[0, :, x]).abs() <= tol[0, :, x]).all(), x
    assert set(range(20 + n)) - hit or n < 3
