"""The operators over a paged KV cache on the GPU, against their formulas in 64
bits (tests/_paged.py derives the bounds)."""
import math

import pytest

torch = pytest.importorskip("torch")

from plugins_amd import exl3 as X  # noqa: E402
from plugins_amd import paged as P  # noqa: E402
from tests import _paged as R  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def batch(counts, lens, dtype, kv, group, dim, page, seed, extra=3, layers=1, max_pages=None):
    """Host tensors of a step: pools of random values, NaN wherever no sequence
    has a key, a random table, cu, q."""
    g = torch.Generator().manual_seed(seed)
    table, pages = R.random_table(counts, lens, page, extra, g, max_pages)
    shape = (layers, pages, kv, page, dim)
    k, v = torch.randn(shape, generator=g).to(dtype), torch.randn(shape, generator=g).to(dtype)
    mine = torch.zeros(pages, page, dtype=torch.bool)
    for s, (n, c) in enumerate(zip(counts, lens)):
        pg, row = R.slots(table, s, page, n + c)
        mine[pg, row] = True
    hole = ~mine[None, :, None, :, None]
    k, v = k.masked_fill(hole, math.nan), v.masked_fill(hole, math.nan)
    cu = [0]
    for n in counts:
        cu.append(cu[-1] + n)
    q = torch.randn(cu[-1], kv * group, dim, generator=g).to(dtype)
    return g, k, v, table, cu, q


def attended(k, v, table, counts, lens, q, mask, rows=None, **kw):
    cache = P.PagedCache.over(k.to(DEV), v.to(DEV), table.to(DEV))
    rows = rows or P.Rows.of(counts, lens, DEV)
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device=DEV)
    got = P.attend(cache, kw.pop("layer", 0), rows, q.to(DEV), out,
                   mask=None if mask is None else mask.to(DEV), **kw)
    torch.cuda.synchronize()
    assert got is out
    return out.cpu()


def near(got, want, tol, what):
    off = (got.double() - want).abs()
    assert not torch.isnan(off).any(), what
    worst = float((off - tol).max())
    assert worst <= 0, (what, worst, float((off / tol.clamp(min=1e-300)).max()))


CASES = [
    # counts, lens, kv, group, dim, page
    ([1], [0], 1, 1, 64, 16),
    ([1], [1], 2, 4, 128, 16),
    ([1], [2047], 2, 4, 128, 64),
    ([1, 1, 1], [15, 16, 17], 2, 3, 64, 16),
    ([5, 0, 3, 1], [31, 200, 0, 64], 2, 4, 128, 32),
    ([17, 64, 2], [100, 3, 1000], 1, 8, 128, 16),
    ([70, 1, 33], [0, 513, 250], 2, 5, 64, 64),
    ([129], [300], 1, 2, 128, 256),
    ([40], [90], 1, 7, 64, 128),
    ([7, 8, 0, 2], [0, 777, 5, 90], 2, 4, 128, 64),
    ([9, 4], [63, 1500], 3, 3, 64, 16),
    ([20, 9, 16], [130, 0, 2500], 2, 4, 128, 32),
    ([33], [64], 5, 2, 64, 64),
    ([60], [5000], 1, 4, 128, 64),
    ([1, 1], [4095, 4096], 8, 1, 128, 256),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("counts,lens,kv,group,dim,page", CASES)
@pytest.mark.parametrize("tree", [False, True])
def test_attend(counts, lens, kv, group, dim, page, dtype, tree):
    g, k, v, table, cu, q = batch(counts, lens, dtype, kv, group, dim, page, 11 + sum(counts))
    parents = [R.random_tree(n, g) if n else [] for n in counts]
    seen = [R.ancestors(p) if tree else [list(range(i + 1)) for i in range(len(p))] for p in parents]
    mask = R.masks([js for s in seen for js in s], -(-max(counts) // 64)) if tree else None
    scale = 1 / math.sqrt(dim)
    want, tol = R.attention(q, k, v, table, cu, lens, seen, page, group, scale)
    got = attended(k, v, table, counts, lens, q, mask)
    near(got, want, tol, "attend")
    # again, bit for bit
    assert torch.equal(got, attended(k, v, table, counts, lens, q, mask))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attend_free_masks_and_empty_rows(dtype):
    """Masks that are no tree's: rows that see none of the rows, not even
    themselves; behind an empty context such a row is zeros."""
    counts, lens = [6, 70, 4], [0, 40, 0]
    g, k, v, table, cu, q = batch(counts, lens, dtype, 2, 4, 128, 16, 5)
    seen = [[[j for j in range(n) if torch.rand(1, generator=g) < 0.4] for _ in range(n)]
            for n in counts]
    seen[0][2], seen[2] = [], [[] for _ in range(4)]
    mask = R.masks([js for s in seen for js in s], 3)  # a word more than is needed
    want, tol = R.attention(q, k, v, table, cu, lens, seen, 16, 4, 0.3)
    got = attended(k, v, table, counts, lens, q, mask, scale=0.3)
    near(got, want, tol, "free masks")
    assert not got[2].any() and not got[cu[2]:].any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("n,group", [(3, 4), (40, 4)])
def test_attend_keeps_what_is_masked_out(dtype, what, n, group):
    """A drafted row whose key and value overflowed: the rows that see it are
    NaN or infinite, the others as if it were not there."""
    counts, lens, page = [n, 2], [37, 50], 16
    g, k, v, table, cu, q = batch(counts, lens, dtype, 2, group, 128, page, 6)
    parents = [[-1] + [max(0, i - 2) for i in range(1, n)], [-1, 0]]
    seen = [R.ancestors(p) for p in parents]
    mask = R.masks([js for s in seen for js in s], 1)
    pg, row = R.slots(table, 0, page, 37 + n)
    for pool in (k, v):
        pool[0, pg[37 + 1], :, row[37 + 1]] = what
    bad = [i for i in range(n) if 1 in seen[0][i]]
    want, tol = R.attention(q, k, v, table, cu, lens, seen, page, group, 1 / math.sqrt(128))
    got = attended(k, v, table, counts, lens, q, mask)
    fine = [t for t in range(n + 2) if t not in bad]
    near(got[fine], want[fine], tol[fine], "masked out")
    assert not torch.isfinite(got[bad].float()).all(-1).any()
    # without a mask: the rows before it
    seen = [[list(range(i + 1)) for i in range(m)] for m in counts]
    want, tol = R.attention(q, k, v, table, cu, lens, seen, page, group, 1 / math.sqrt(128))
    got = attended(k, v, table, counts, lens, q, None)
    fine = [0, n, n + 1]
    near(got[fine], want[fine], tol[fine], "masked out, in a line")
    assert not torch.isfinite(got[1:n].float()).all(-1).any()


def test_attend_large_scores_and_an_infinite_key():
    """Scores of thousands (f32 exponents far apart), and a context whose one
    key is -inf against positive queries: weight 0."""
    counts, lens = [2], [100]
    g, k, v, table, cu, q = batch(counts, lens, torch.float16, 1, 4, 64, 16, 7)
    q = q.abs() * 30
    k = k * 30
    pg, row = R.slots(table, 0, 16, 102)
    k[0, pg[5], :, row[5]] = -math.inf
    seen = [[[0], [0, 1]]]
    k2 = k.clone()
    k2[0, pg[5], :, row[5]] = -60.0
    want, tol = R.attention(q, k2, v, table, cu, lens, seen, 16, 4, 0.125)
    got = attended(k, v, table, counts, lens, q, None, scale=0.125)
    # es of these scores: the bound's own, from |q k|
    assert torch.isfinite(got.float()).all()
    near(got, want, tol, "large scores")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,gap", [(1, 14.5), (1, 18.5), (40, 14.5), (40, 18.5)])
def test_attend_many_small_weights(dtype, rows, gap):
    """One key far above 20000 others whose weights only count together: each is
    about 2^-21 of the largest, where f16 alone would hold a few bits of it, or
    2^-27, where the kernel's weights are f16's subnormal numbers."""
    n_ctx = 20000
    counts, lens = [rows], [n_ctx]
    g, k, v, table, cu, q = batch(counts, lens, dtype, 1, 1, 64, 256, 8)
    v = v.abs()
    q = torch.ones_like(q)
    k = torch.zeros_like(k)
    pg, row = R.slots(table, 0, 256, n_ctx + rows)
    k[0, pg[123], :, row[123]] = gap / 64
    v[0, pg[123], :, row[123]] = 0
    seen = [[list(range(i + 1)) for i in range(rows)]]
    want, tol = R.attention(q, k, v, table, cu, lens, seen, 256, 1, 1.0)
    near(attended(k, v, table, counts, lens, q, None, scale=1.0), want, tol, "small weights")


def test_attend_strides_and_rows_behind():
    """q inside a fused q+k+v matrix, an output with wider rows, and rows of the
    tensors behind the last sequence: left as they were."""
    counts, lens, kv, group, dim, page = [3, 9], [40, 7], 2, 4, 128, 16
    g, k, v, table, cu, q = batch(counts, lens, torch.float16, kv, group, dim, page, 9)
    total, extra = 12, 5
    width = kv * group * dim
    fused = torch.randn(total + extra, width + 2 * kv * dim, generator=g).half()
    fused[:total, :width] = q.view(total, width)
    rows = P.Rows(torch.tensor(cu, dtype=torch.int32, device=DEV),
                  torch.tensor(lens, dtype=torch.int32, device=DEV), total + extra, 9)
    out = torch.full((total + extra, width + 64), 5.0, dtype=torch.float16, device=DEV)
    cache = P.PagedCache.over(k.to(DEV), v.to(DEV), table.to(DEV))
    P.attend(cache, 0, rows, fused.to(DEV)[:, :width], out[:, :width])
    seen = [[list(range(i + 1)) for i in range(n)] for n in counts]
    want, tol = R.attention(q, k, v, table, cu, lens, seen, page, group, 1 / math.sqrt(dim))
    near(out[:total, :width].cpu().view(total, -1, dim), want, tol, "strides")
    assert bool((out[:, width:] == 5.0).all()) and bool((out[total:] == 5.0).all())


def test_attend_bad_pages_and_lengths_are_nan():
    """A sequence whose table names no page, whose length is negative or does not
    fit its table is NaN; the others are what they are alone."""
    counts, lens = [2, 2, 2, 2, 2], [30, 30, 30, 30, 30]
    g, k, v, table, cu, q = batch(counts, lens, torch.float16, 1, 4, 64, 16, 10)
    seen = [[[0], [0, 1]]] * 5
    want, tol = R.attention(q, k, v, table, cu, lens, seen, 16, 4, 0.125)
    bad = table.clone()
    bad[1, 1] = -1
    bad[2, 0] = k.shape[1]
    rows = P.Rows.of(counts, [30, 30, 30, -1, 100], DEV)
    got = attended(k, v, bad, counts, lens, q, None, rows=rows)
    assert torch.isnan(got[2:]).all()
    near(got[:2], want[:2], tol[:2], "beside bad ones")


def test_attend_beyond_32_bits():
    """Pages whose bytes and elements lie past 2^32 of a layer."""
    kv, page, dim, group = 8, 256, 128, 1
    per = kv * page * dim
    pages = (1 << 32) // per + 9
    free = torch.cuda.mem_get_info()[0]
    if free < 4 * 2 * per * pages:
        pytest.skip("not enough memory")
    k = torch.empty(2, pages, kv, page, dim, dtype=torch.float16, device=DEV)
    v = torch.empty_like(k)
    g = torch.Generator().manual_seed(12)
    small_k = torch.randn(2, 3, kv, page, dim, generator=g).half()
    small_v = torch.randn(2, 3, kv, page, dim, generator=g).half()
    at = [pages - 1, pages - 5, pages - 3]
    for x, p in enumerate(at):
        k[:, p], v[:, p] = small_k[:, x].to(DEV), small_v[:, x].to(DEV)
    cache = P.PagedCache.over(k, v, torch.tensor([at], dtype=torch.int32, device=DEV))
    counts, lens = [2], [600]
    q = torch.randn(2, kv, dim, generator=g).half()
    rows = P.Rows.of(counts, lens, DEV)
    got = P.attend(cache, 1, rows, q.to(DEV)).cpu().view(2, kv, dim)
    tab = torch.tensor([[0, 1, 2]], dtype=torch.int32)
    want, tol = R.attention(q, small_k, small_v, tab, [0, 2], lens, [[[0], [0, 1]]], page, 1,
                            1 / math.sqrt(dim), layer=1)
    near(got, want, tol, "far pages")
    # append, commit and copies there
    pos, slot, mask = P.plan(cache, rows, torch.tensor([-1, 0], dtype=torch.int32, device=DEV))
    assert slot.tolist() == [at[2] * page + 88, at[2] * page + 89]
    new = torch.randn(2, kv * dim, generator=g).half().to(DEV)
    P.qkv_append(cache, 1, q.to(DEV), new, new, None, None, torch.zeros_like(pos), slot,
                 q.to(DEV))
    torch.cuda.synchronize()
    assert torch.equal(v[1, at[2], :, 88:90], new.view(2, kv, dim).transpose(0, 1))
    assert torch.equal(k[1, at[2], :, 88:90], new.view(2, kv, dim).transpose(0, 1))
    P.copy_pages(cache, [at[2]], [pages - 8])
    torch.cuda.synchronize()
    assert torch.equal(v[:, pages - 8], v[:, at[2]])


def test_attend_other_stream_and_graph():
    """A call on another stream than the current one; captured, with lengths,
    table and q changed between the replays; two graphs over the same rows."""
    counts, lens = [3, 20], [500, 70]
    g, k, v, table, cu, q = batch(counts, lens, torch.bfloat16, 2, 4, 128, 32, 13, max_pages=40)
    want0 = attended(k, v, table, counts, lens, q, None)
    cache = P.PagedCache.over(k.to(DEV), v.to(DEV), table.to(DEV))
    rows = P.Rows.of(counts, lens, DEV)
    qd = q.to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out = P.attend(cache, 0, rows, qd, stream=side)
    side.synchronize()
    assert torch.equal(out.cpu().view(q.shape), want0)
    outs, graphs = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=side, capture_error_mode="thread_local"):
            outs.append(P.attend(cache, 0, rows, qd))
        graphs.append(gr)
    for turn in range(3):
        new = [500 - 100 * turn, 70 - 30 * turn]
        rows.len.copy_(torch.tensor(new, dtype=torch.int32))
        qd.copy_((q * (1 + turn)).to(DEV))
        want = attended(k, v, table, counts, new, q * (1 + turn), None)
        for gr, out in zip(graphs, outs):
            out.fill_(3.0)
            gr.replay()
        eager = P.attend(cache, 0, rows, qd)
        torch.cuda.synchronize()
        for out in (*outs, eager):
            assert torch.equal(out.cpu().view(q.shape), want), turn


@pytest.mark.parametrize("n,group", [(1, 4), (6, 5)])
def test_attend_split_calls_repeat(n, group):
    """Split tiles of few pairs, joined from the scratch: two hundred calls in a
    row on scratch that holds garbage or an earlier call's, and replays of one
    captured call, all bit for bit."""
    counts, lens = [n, 1, n], [3000, 700, 9000]
    g, k, v, table, cu, q = batch(counts, lens, torch.float16, 2, group, 64, 64, 19)
    seen = [[list(range(i + 1)) for i in range(m)] for m in counts]
    want, tol = R.attention(q, k, v, table, cu, lens, seen, 64, group, 0.125)
    cache = P.PagedCache.over(k.to(DEV), v.to(DEV), table.to(DEV))
    rows, qd = P.Rows.of(counts, lens, DEV), q.to(DEV)
    first = P.attend(cache, 0, rows, qd).clone()
    near(first.cpu().view(q.shape), want, tol, "split")
    scratch = torch.full((P.attend_scratch_bytes(cache, rows, 2 * group),), 255, dtype=torch.uint8,
                         device=DEV)
    out = torch.empty_like(first)
    wrong = torch.zeros((), dtype=torch.int64, device=DEV)
    for i in range(200):
        out.fill_(3.0)
        P.attend(cache, 0, rows, qd, out, scratch=scratch)
        wrong += (out != first).sum()
        if i % 50 == 0:
            scratch.random_(0, 256)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=side, capture_error_mode="thread_local"):
        P.attend(cache, 0, rows, qd, out, scratch=scratch)
    for i in range(200):
        out.fill_(3.0)
        gr.replay()
        wrong += (out != first).sum()
    assert wrong.item() == 0


@pytest.mark.parametrize("heads", [1, 5])
def test_attend_many_sequences(heads):
    """More sequences than a wave has lanes, most without rows; the context's
    keys differ widely."""
    g = torch.Generator().manual_seed(14)
    counts = [int(torch.randint(0, 3, (1,), generator=g)) for _ in range(150)]
    lens = [int(torch.randint(0, 90, (1,), generator=g)) for _ in range(150)]
    lens[70], counts[70], counts[149] = 3000, 2, 2
    g, k, v, table, cu, q = batch(counts, lens, torch.float16, 1, heads, 64, 16, 15)
    seen = [[list(range(i + 1)) for i in range(n)] for n in counts]
    want, tol = R.attention(q, k, v, table, cu, lens, seen, 16, heads, 0.125)
    near(attended(k, v, table, counts, lens, q, None), want, tol, "many sequences")


# ------------------------------------------------------------------ tree plan

@pytest.mark.parametrize("counts,lens,page", [
    ([1], [0], 16), ([60], [2048], 64), ([64, 65, 0, 1, 130], [0, 5, 9, 300, 31], 16),
    ([1024], [100], 256), ([3] * 200, list(range(200)), 16)])
def test_tree_plan(counts, lens, page):
    g = torch.Generator().manual_seed(sum(counts))
    table, pages = R.random_table(counts, lens, page, 2, g)
    k = torch.empty(1, pages, 1, page, 64, dtype=torch.float16, device=DEV)
    cache = P.PagedCache.over(k, k.clone(), table.to(DEV))
    rows = P.Rows.of(counts, lens, DEV)
    trees = [R.random_tree(n, g) if n else [] for n in counts]
    if counts[0] >= 60:  # a line, several roots, parents that are no parents
        trees[0] = [-1] + list(range(counts[0] - 1))
        trees[-1] = [-1 if i % 3 == 0 else i - 1 for i in range(counts[-1])]
        trees[0][7], trees[0][9], trees[0][11] = 7, 1000000, -5
    flat = [p for t in trees for p in t]
    anc = [a for t in trees for a in R.ancestors(t)]
    for words in (-(-max(counts) // 64), -(-max(counts) // 64) + 2):
        pos = torch.full((len(flat),), -9, dtype=torch.int32, device=DEV)
        slot, mask = pos.clone(), torch.full((len(flat), words), -9, dtype=torch.int64, device=DEV)
        P.tree_plan(cache, rows, torch.tensor(flat, dtype=torch.int32, device=DEV), pos, slot, mask)
        torch.cuda.synchronize()
        assert torch.equal(mask.cpu(), R.masks(anc, words))
        t = 0
        for s, n in enumerate(counts):
            for i in range(n):
                assert pos[t].item() == lens[s] + len(anc[t]) - 1 if t < 300 else True
                t += 1
        want = torch.cat([(R.slots(table, s, page, lens[s] + n)[0] * page
                           + R.slots(table, s, page, lens[s] + n)[1])[lens[s]:]
                          for s, n in enumerate(counts)])
        assert torch.equal(slot.cpu().long(), want)
        depth = torch.tensor([len(a) - 1 for a in anc])
        base = torch.cat([torch.full((n,), c) for n, c in zip(counts, lens)])
        assert torch.equal(pos.cpu().long(), base + depth)
    # rows in a line: no parent
    pos, slot, mask = P.plan(cache, rows)
    assert mask is None and torch.equal(slot.cpu().long(), want)
    line = torch.cat([torch.arange(c, c + n) for n, c in zip(counts, lens)])
    assert torch.equal(pos.cpu().long(), line)
    mask = torch.empty(len(flat), words, dtype=torch.int64, device=DEV)
    P.tree_plan(cache, rows, None, pos, slot, mask)
    torch.cuda.synchronize()
    assert torch.equal(mask.cpu(), R.masks([list(range(i + 1)) for n in counts for i in range(n)],
                                           words))


def test_tree_plan_of_a_first_sequence_that_starts_late():
    """Rows before cu[0] are no sequence's."""
    k = torch.empty(1, 2, 1, 16, 64, dtype=torch.float16, device=DEV)
    cache = P.PagedCache.over(k, k.clone(), torch.tensor([[1]], dtype=torch.int32, device=DEV))
    rows = P.Rows(torch.tensor([2, 4], dtype=torch.int32, device=DEV),
                  torch.tensor([3], dtype=torch.int32, device=DEV), 5, 2)
    pos, slot, mask = P.plan(cache, rows, torch.tensor([7, 7, -1, 0, 7], dtype=torch.int32, device=DEV))
    assert slot.tolist() == [-1, -1, 19, 20, -1] and pos[2:4].tolist() == [3, 4]
    assert mask[:, 0].tolist() == [0, 0, 1, 3, 0]


def test_tree_plan_of_rows_and_keys_that_do_not_fit():
    """Rows behind the last sequence, rows past max_rows, a length that does not
    fit its table, a page that is none: slot -1."""
    page, k = 16, torch.empty(1, 6, 1, 16, 64, dtype=torch.float16, device=DEV)
    table = torch.tensor([[0, 1], [2, -1], [3, 9], [4, 5]], dtype=torch.int32, device=DEV)
    cache = P.PagedCache.over(k, k.clone(), table)
    cu = torch.tensor([0, 4, 7, 9, 11], dtype=torch.int32, device=DEV)
    lens = torch.tensor([5, 14, 15, 31], dtype=torch.int32, device=DEV)
    rows = P.Rows(cu, lens, 13, 3)
    pos, slot, mask = P.plan(cache, rows, torch.full((13,), -1, dtype=torch.int32, device=DEV))
    assert slot.tolist() == [5, 6, 7, -1, 46, 47, -1, 63, -1, -1, -1, -1, -1]
    assert pos[:3].tolist() == [5, 5, 5] and pos[4:7].tolist() == [14, 14, 14]
    assert mask[:, 0].tolist() == [1, 2, 4, 0, 1, 2, 4, 1, 2, 1, 2, 0, 0]


# --------------------------------------------------- norms, rotation and append

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,kv,group,dim,page,norms", [
    (1, 8, 4, 128, 64, True), (7, 1, 1, 64, 16, True), (37, 2, 5, 64, 32, False),
    (130, 2, 4, 128, 256, True), (600, 1, 3, 128, 16, True)])
def test_qkv_append(rows, kv, group, dim, page, norms, dtype):
    g = torch.Generator().manual_seed(rows)
    pages = -(-rows // page) + 3
    fused = (3 * torch.randn(rows, (group + 2) * kv * dim, generator=g)).to(dtype)
    wq, wk = group * kv * dim, kv * dim
    qn = (1 + 0.1 * torch.randn(dim, generator=g)).to(dtype) if norms else None
    kn = (1 + 0.1 * torch.randn(dim, generator=g)).to(dtype) if norms else None
    # positions from the first to the far end of the type
    pos = torch.randint(0, 1 << 20, (rows,), generator=g, dtype=torch.int32)
    pos[0] = 0
    pos[-1] = 2 ** 31 - 1 if rows > 1 else 12345
    slot = torch.randperm(pages * page, generator=g)[:rows].int()
    dead = rows // 3 if rows > 2 else None
    if dead is not None:
        slot[dead] = -1
    old = torch.randn(2, pages, kv, page, dim, generator=g).to(dtype)
    k, v = old.to(DEV), (old + 1).to(DEV)
    cache = P.PagedCache.over(k, v, torch.zeros(1, 1, dtype=torch.int32, device=DEV))
    fd = fused.to(DEV)
    out = torch.full((rows, wq), 9.0, dtype=dtype, device=DEV)
    dv = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    P.qkv_append(cache, 1, fd[:, :wq], fd[:, wq:wq + wk], fd[:, wq + wk:], dv(qn), dv(kn), pos.to(DEV),
                 slot.to(DEV), out, 1e-6, 1e6)
    torch.cuda.synchronize()
    live = [t for t in range(rows) if t != dead]
    want, tol = R.rotated(fused[:, :wq].reshape(rows, -1, dim), qn, pos, 1e-6, 1e6)
    near(out.cpu().view(rows, -1, dim)[live], want[live], tol[live], "q")
    if dead is not None:
        assert bool((out[dead] == 9.0).all())
    want, tol = R.rotated(fused[:, wq:wq + wk].reshape(rows, kv, dim), kn, pos, 1e-6, 1e6)
    kc, vc = k.cpu(), v.cpu()
    at = slot.long()[live]
    near(kc[1, at // page, :, at % page], want[live], tol[live], "k")
    assert torch.equal(vc[1, at // page, :, at % page],
                       fused[:, wq + wk:].reshape(rows, kv, dim)[live])
    # every other key and value, and the other layer, as they were
    keep = torch.ones(pages, page, dtype=torch.bool)
    keep[at // page, at % page] = False
    for pool, was in ((kc, old), (vc, (old + 1).to(dtype))):
        assert torch.equal(pool[0], was[0])
        assert torch.equal(pool[1].transpose(1, 2)[keep], was[1].transpose(1, 2)[keep])
    # in place, the same bits
    P.qkv_append(cache, 1, fd[:, :wq], fd[:, wq:wq + wk], fd[:, wq + wk:], dv(qn), dv(kn), pos.to(DEV),
                 slot.to(DEV), fd[:, :wq], 1e-6, 1e6)
    torch.cuda.synchronize()
    assert torch.equal(fd[:, :wq][live], out[live])
    if dead is not None:
        assert torch.equal(fd[dead, :wq].cpu(), fused[dead, :wq])


# --------------------------------------------------------------------- commit

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("counts,lens,kv,dim,page,layers,most", [
    ([1], [0], 1, 64, 16, 1, 1), ([8], [13], 2, 128, 16, 3, 8), ([24, 0, 1, 64], [7, 5, 30, 100], 8, 128, 64, 2, 64),
    ([130, 40], [60, 15], 3, 64, 16, 2, 40), ([300], [5], 8, 128, 32, 1, 300)])
def test_commit(counts, lens, kv, dim, page, layers, most, dtype):
    g = torch.Generator().manual_seed(sum(counts))
    table, pages = R.random_table(counts, lens, page, 2, g)
    shape = (layers, pages, kv, page, dim)
    k, v = torch.randn(shape, generator=g).to(dtype), torch.randn(shape, generator=g).to(dtype)
    trees, ids, target = [], [], []
    for n in counts:
        t = R.random_tree(n, g) if n else []
        if n > 100:  # deep: most rows follow the one before or the one before that
            t = [-1] + [max(0, i - 1 - int(torch.randint(0, 2, (1,), generator=g)))
                        for i in range(1, n)]
        trees.append(t)
        # few tokens: siblings of one token and long accepted paths are common
        ids.append([int(x) for x in torch.randint(0, 2, (n,), generator=g)])
        target.append([int(x) for x in torch.randint(0, 2, (n,), generator=g)])
        for j in range(1, n):
            if torch.rand(1, generator=g) < 0.6:
                target[-1][t[j]] = ids[-1][j]
    cu = [0]
    for n in counts:
        cu.append(cu[-1] + n)
    flat = lambda x: torch.tensor([y for z in x for y in z], dtype=torch.int32, device=DEV)  # noqa: E731
    kd, vd = k.to(DEV), v.to(DEV)
    cache = P.PagedCache.over(kd, vd, table.to(DEV))
    rows = P.Rows.of(counts, lens, DEV)
    S = len(counts)
    path = torch.full((S, most), -7, dtype=torch.int32, device=DEV)
    count, nxt, new = (torch.full((S,), -7, dtype=torch.int32, device=DEV) for _ in range(3))
    P.commit(cache, rows, flat(trees), flat(ids), flat(target), path, count, nxt, new)
    torch.cuda.synchronize()
    longest = 0
    for s, n in enumerate(counts):
        way, after = R.walk(trees[s], ids[s], target[s], most)
        longest = max(longest, len(way))
        assert path[s].tolist() == way + [-1] * (most - len(way))
        assert (count[s].item(), nxt[s].item(), new[s].item()) == (len(way), after, lens[s] + len(way))
        pg, row = R.slots(table, s, page, lens[s] + n)
        src = [lens[s] + i for i in way]
        dst = list(range(lens[s], lens[s] + len(way)))
        for pool in (k, v):
            pool[:, pg[dst], :, row[dst]] = pool[:, pg[src], :, row[src]].clone()
    assert longest > 1 or max(counts) <= 8
    assert torch.equal(kd.cpu(), k) and torch.equal(vd.cpu(), v)


def test_commit_of_lines_and_bad_sequences():
    """Without parents the rows are a line; a sequence that does not fit its
    table accepts nothing; a page that is none moves nothing."""
    page = 16
    g = torch.Generator().manual_seed(3)
    k = torch.randn(1, 4, 1, page, 64, generator=g).half()
    table = torch.tensor([[0, 1], [2, -1], [3, -1]], dtype=torch.int32, device=DEV)
    kd = k.to(DEV)
    cache = P.PagedCache.over(kd, kd.clone(), table)
    rows = P.Rows.of([4, 4, 4], [10, 30, 14], DEV)
    ids = torch.tensor([5, 6, 7, 8] * 3, dtype=torch.int32, device=DEV)
    target = torch.tensor([6, 7, 0, 0, 6, 7, 8, 9, 6, 7, 8, 9], dtype=torch.int32, device=DEV)
    path = torch.empty(3, 3, dtype=torch.int32, device=DEV)
    count, nxt, new = (torch.empty(3, dtype=torch.int32, device=DEV) for _ in range(3))
    P.commit(cache, rows, None, ids, target, path, count, nxt, new)
    torch.cuda.synchronize()
    assert path.tolist() == [[0, 1, 2], [-1, -1, -1], [0, 1, 2]]
    assert count.tolist() == [3, 0, 3] and nxt.tolist() == [0, -1, 8] and new.tolist() == [13, 30, 17]
    assert torch.equal(kd.cpu(), k)


# ----------------------------------------------------------------------- pages

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("count,pages,layers,kv,page,dim", [
    (1, 3, 2, 1, 16, 64), (5, 20, 3, 3, 16, 128), (300, 700, 1, 2, 16, 64), (2, 6, 4, 8, 64, 128)])
def test_copy_pages(count, pages, layers, kv, page, dim, dtype):
    g = torch.Generator().manual_seed(count)
    k, v = (torch.randn(layers, pages, kv, page, dim, generator=g).to(dtype) for _ in range(2))
    order = torch.randperm(pages, generator=g).tolist()
    dst, rest = order[:count], order[count:]
    src = [rest[i % len(rest)] for i in range(count)]  # a page may be read twice
    kd, vd = k.to(DEV), v.to(DEV)
    cache = P.PagedCache.over(kd, vd, torch.zeros(1, 1, dtype=torch.int32, device=DEV))
    P.copy_pages(cache, src, dst)
    torch.cuda.synchronize()
    for pool, got in ((k, kd), (v, vd)):
        pool[:, dst] = pool[:, src]
        assert torch.equal(got.cpu(), pool)


def test_forks_and_compaction_keep_every_sequence():
    """Sequences that fork, write, roll back and go: each reads its own keys
    throughout, and after the pool is compacted."""
    cache = P.PagedCache(layers=2, pages=24, kv_heads=2, seqs=4, max_pages=8, page=16, head_dim=64,
                         device=DEV)
    g = torch.Generator().manual_seed(1)
    text = {}  # what each sequence holds: values [keys, layers, kv, dim]

    def write(seq, start, n):
        cache.reserve(seq, start, start + n)
        rows = P.Rows.of([n], [start], DEV)
        at = P.Rows.of([0] * seq + [n], [0] * seq + [start], DEV)
        pos, slot, _ = P.plan(cache, at)
        new = torch.randn(n, 2, 2, 64, generator=g).half()
        for layer in range(2):
            x = new[:, layer].reshape(n, 128).to(DEV)
            P.qkv_append(cache, layer, x, x, x, None, None, pos, slot, x.clone())
        text[seq] = torch.cat([text.get(seq, new[:0])[:start], new])
        assert rows.rows == n

    def check():
        torch.cuda.synchronize()
        table = cache.table.cpu()
        assert torch.equal(table, torch.from_numpy(cache.book.table()))
        for seq, want in text.items():
            pg, row = R.slots(table, seq, 16, len(want))
            got = cache.v.cpu()[:, pg, :, row].view(len(want), 2, 2, 64)
            assert torch.equal(got, want), seq

    write(0, 0, 40)
    for a, b, keys in ((0, 1, 40), (0, 2, 17)):
        cache.fork(a, b, keys)
        text[b] = text[a][:keys]
    check()
    write(1, 40, 3)   # into a page that 0 holds too: copied first
    write(2, 17, 30)
    check()
    write(0, 35, 20)  # rolled back and written again
    check()
    cache.fork(1, 3, 43)
    text[3] = text[1]
    cache.trim(1, 20)
    text[1] = text[1][:20]
    write(1, 20, 9)
    check()
    cache.trim(0, 0)
    del text[0]
    assert cache.compact() > 0
    check()
    used = {int(p) for p in cache.table.flatten() if p >= 0}
    assert used == set(range(len(used)))
    assert cache.compact() == 0
    write(0, 0, 33)
    check()


# ------------------------------------------------- calls that take no usual form

def test_steps_without_sequences():
    """No sequence, with and without rows: padding gets slot -1, the others write
    nothing."""
    k = torch.zeros(1, 2, 1, 16, 64, dtype=torch.float16, device=DEV)
    cache = P.PagedCache.over(k, k.clone(), torch.zeros(2, 1, dtype=torch.int32, device=DEV))
    i32 = {"dtype": torch.int32, "device": DEV}
    rows = P.Rows.of([], [], DEV)
    pos, slot, mask = P.plan(cache, rows, torch.empty(0, **i32))
    assert pos.numel() == slot.numel() == mask.numel() == 0
    empty = torch.empty(0, **i32)
    P.commit(cache, rows, None, empty, empty, torch.empty(0, 3, **i32), empty, empty, empty)
    padded = P.Rows(torch.zeros(1, **i32), empty, 3, 0)
    pos, slot, _ = P.plan(cache, padded)
    assert pos.tolist() == [0] * 3 and slot.tolist() == [-1] * 3
    q = torch.ones(3, 128, dtype=torch.float16, device=DEV)
    out = torch.full_like(q, 7.0)
    P.attend(cache, 0, padded, q, out)
    P.qkv_append(cache, 0, q, q[:, :64], q[:, 64:], None, None, pos, slot, out)
    torch.cuda.synchronize()
    assert bool((out == 7.0).all()) and not k.any()


def test_arguments_that_would_pass_for_others_are_refused():
    """A mask without words is none, `next` does not overwrite the tree's ids, a
    page number past 32 bits is not its low bits."""
    k = torch.zeros(1, 2, 1, 16, 64, dtype=torch.float16, device=DEV)
    cache = P.PagedCache.over(k, k.clone(), torch.zeros(2, 1, dtype=torch.int32, device=DEV))
    rows = P.Rows.of([2, 2], [0, 3], DEV)
    i32 = {"dtype": torch.int32, "device": DEV}
    none = torch.empty(4, 0, dtype=torch.int64, device=DEV)
    q = torch.ones(4, 64, dtype=torch.float16, device=DEV)
    with pytest.raises(ValueError, match="mask"):
        P.attend(cache, 0, rows, q, mask=none)
    with pytest.raises(ValueError, match="mask"):
        P.tree_plan(cache, rows, None, torch.empty(4, **i32), torch.empty(4, **i32), none)
    ids = torch.ones(4, **i32)
    path, (a, b, c) = torch.empty(2, 2, **i32), (torch.empty(2, **i32) for _ in range(3))
    for kw in ((a, ids[:2], c), (ids[2:], b, c), (a, b, rows.cu[1:])):
        with pytest.raises(X.Exl3Error, match="over an input"):
            P.commit(cache, rows, None, ids, ids.clone(), path, *kw)
    with pytest.raises(OverflowError):
        P.copy_pages(cache, [1 << 32], [1])


@pytest.mark.parametrize("counts,lens,kv,splits", [
    ([300, 1], [6000, 40], 1, 10),       # ten tiles, several items each, of unlike ends
    ([200, 90, 31, 1, 160], [0, 70, 500, 3, 0], 8, 0),   # whole tiles, several a sequence
    ([2] * 300, [40] * 299 + [700], 8, 1)])  # one of 300 is split
def test_attend_items_of_several_tiles(counts, lens, kv, splits):
    """Items of a sequence go by keys first, then tiles; their sums lie in the
    scratch by tiles."""
    from tests import test_paged_index as I
    group = 4
    sl = I.split_of(kv, group, sum(counts), len(counts), max(counts))
    assert all(n == splits for _, n in I.items_of(sl, counts, lens))
    g, k, v, table, cu, q = batch(counts, lens, torch.float16, kv, group, 64, 64, 23)
    seen = [[list(range(i + 1)) for i in range(n)] for n in counts]
    want, tol = R.attention(q, k, v, table, cu, lens, seen, 64, group, 0.125)
    near(attended(k, v, table, counts, lens, q, None), want, tol, "items")


@pytest.mark.parametrize("counts,lens,group", [
    ([1, 1], [40, 3000], 4), ([6], [3000], 4), ([40, 3], [0, 20], 4), ([33, 7], [4000, 9], 8)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attend_in_place(counts, lens, group, dtype):
    """out in place of q: tiles of few pairs and of many, whole and split, the bits
    of a call with an output of its own; so with q a slice of a wider matrix."""
    g, k, v, table, cu, q = batch(counts, lens, dtype, 2, group, 128, 64, 31)
    want = attended(k, v, table, counts, lens, q, None)
    cache = P.PagedCache.over(k.to(DEV), v.to(DEV), table.to(DEV))
    rows, width = P.Rows.of(counts, lens, DEV), 2 * group * 128
    wide = torch.full((cu[-1], width + 128), 3.0, dtype=dtype, device=DEV)
    wide[:, :width] = q.view(cu[-1], -1).to(DEV)
    for x in (q.to(DEV), wide[:, :width]):
        assert P.attend(cache, 0, rows, x, x) is x
        assert torch.equal(x.cpu().view(q.shape), want)
    assert bool((wide[:, width:] == 3.0).all())


def test_operators_refuse_what_would_race():
    """Through the mirror: an output over an input, unless it is q itself."""
    k = torch.zeros(1, 8, 2, 16, 64, dtype=torch.float16, device=DEV)
    cache = P.PagedCache.over(k, k.clone(), torch.arange(4, dtype=torch.int32, device=DEV).view(2, 2))
    i32 = {"dtype": torch.int32, "device": DEV}
    numbers = torch.tensor([0, 2, 4, 0, 3, 0], **i32)  # cu, len and more
    rows = P.Rows(numbers[:3], numbers[3:5], 4, 2)
    fused = torch.ones(5, 512, dtype=torch.float16, device=DEV)
    q, kk, vv = fused[:4, :256], fused[:4, 256:384], fused[:4, 384:]
    parent = torch.tensor([-1, 0, -1, 0], **i32)
    pos, slot, _ = P.plan(cache, rows)
    for out in (fused[1:, :256], fused[:4, 128:384], fused[:4, 256:]):
        with pytest.raises(X.Exl3Error, match="PagedOverlap"):
            P.qkv_append(cache, 0, q, kk, vv, None, None, pos, slot, out)
    for out in (fused[1:, :256], fused[:4, 128:384]):
        with pytest.raises(X.Exl3Error, match="PagedOverlap"):
            P.attend(cache, 0, rows, q, out)
    for p, s in ((parent, slot), (pos, pos), (numbers[2:], slot), (pos, numbers[:4])):
        with pytest.raises(X.Exl3Error, match="PagedOverlap"):
            P.tree_plan(cache, rows, parent, p, s)
    one, two = torch.empty(2, 2, **i32), torch.empty(2, **i32)
    with pytest.raises(X.Exl3Error, match="PagedOverlap"):
        P.commit(cache, rows, parent, pos, slot, one, two, two, torch.empty(2, **i32))
    # rows beside each other in one matrix are apart
    P.qkv_append(cache, 0, q, kk, vv, None, None, pos, slot, q)
    P.attend(cache, 0, rows, q, fused[:4, 256:])
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("scale", [2.0 ** 17, 3e7, 1e9, -1e9, 1e30, -1e30])
@pytest.mark.parametrize("rows,ctx", [(1, 50), (1, 5000), (40, 50), (40, 5000)])
def test_attend_scales_that_make_scores_huge(rows, ctx, scale, dtype):
    """Scores far past 2^24, exact in 32 bits and apart by far more than their
    roundings: a row is the value of its one largest key, or the mean of the two
    that tie for it, and never NaN or zeros.  The tie lies in two places of the
    context, so in two waves and, where it is long, two items."""
    page, dim, group = 16, 64, 4
    g, k, v, table, cu, q = batch([rows], [ctx], dtype, 2, group, dim, page, 51)
    q = torch.ones_like(q)
    pg, at = R.slots(table, 0, page, ctx + rows)
    # scores m / 16 of whole m, 64 products of 2^-10 m each
    m = torch.randint(-100, 100, (ctx + rows,), generator=g)
    top = 120 if scale > 0 else -120
    one, two = ctx // 3, ctx - 9
    m[one] = m[two] = top
    k[0, pg, :, at] = (m.double() / 1024).to(dtype)[:, None, None].expand(-1, 2, dim)
    got = attended(k, v, table, [rows], [ctx], q, None, scale=scale)
    # equal weights of exactly 1: the sum of two values and its half round once, in
    # 32 bits, before the output's rounding
    want = (v[0, pg[one], :, at[one]].float() + v[0, pg[two], :, at[two]].float()) / 2
    want = want.to(dtype)[None, :, None].expand(rows, 2, group, dim).reshape(q.shape)
    assert torch.equal(got, want)
    # the same behind the rows' own keys: the last row alone sees the largest
    m[-1] = 2 * top
    k[0, pg, :, at] = (m.double() / 1024).to(dtype)[:, None, None].expand(-1, 2, dim)
    got = attended(k, v, table, [rows], [ctx], q, None, scale=scale)
    assert torch.equal(got[:-1], want[:-1])
    last = v[0, pg[-1], :, at[-1]][:, None].expand(2, group, dim).reshape(-1, dim)
    assert torch.equal(got[-1], last)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,gap", [(2, 14.5), (2, 18.5), (40, 14.5), (40, 18.5)])
def test_attend_small_weights_beside_a_huge_row(dtype, rows, gap):
    """As test_attend_many_small_weights, every second row's scores past 2^20: the
    rows between them keep what only counts together."""
    n_ctx = 20000
    counts, lens = [rows], [n_ctx]
    g, k, v, table, cu, q = batch(counts, lens, dtype, 1, 1, 64, 256, 8)
    v, q, k = v.abs(), torch.ones_like(q), torch.zeros_like(k)
    q[1::2] = 60000
    pg, row = R.slots(table, 0, 256, n_ctx + rows)
    k[0, pg[123], :, row[123]] = gap / 64
    v[0, pg[123], :, row[123]] = 0
    seen = [[list(range(i + 1)) for i in range(rows)]]
    want, tol = R.attention(q, k, v, table, cu, lens, seen, 256, 1, 1.0)
    got = attended(k, v, table, counts, lens, q, None, scale=1.0)
    near(got[::2], want[::2], tol[::2], "small weights")
    assert not got[1::2].any()


@pytest.mark.parametrize("seqs,n,lens", [
    (40, 300, [0] * 38 + [60000, 0]),  # more items than the launch has, the last ones split
    (80, 8, [100, 0] * 40), (3, 5, [7, 7, 7])])
def test_a_cu_that_goes_back_is_not_begun(seqs, n, lens):
    """Sequences that share rows: the launch and the scratch are sized for the rows
    that there are.  No row is written, and what lies around the scratch stays."""
    page, kv, group, dim = 256, 8, 4, 64
    pages = 240
    table = torch.arange(pages, dtype=torch.int32).repeat(seqs, 1)
    k = torch.zeros(1, pages, kv, page, dim, dtype=torch.float16, device=DEV)
    cache = P.PagedCache.over(k, k.clone(), table.to(DEV))
    cu = [0] + [n, 0] * (seqs // 2) + [n] * (seqs % 2)
    rows = P.Rows(torch.tensor(cu, dtype=torch.int32, device=DEV),
                  torch.tensor(lens, dtype=torch.int32, device=DEV), n, n)
    q = torch.ones(n, kv * group * dim, dtype=torch.float16, device=DEV)
    out = torch.full_like(q, 7.0)
    need = P.attend_scratch_bytes(cache, rows, kv * group)
    room = torch.full((need + 8192,), 85, dtype=torch.uint8, device=DEV)
    scratch = room[4096:4096 + need]
    for _ in range(2):
        P.attend(cache, 0, rows, q, out, scratch=scratch)
        torch.cuda.synchronize()
        assert bool((out == 7.0).all())
        assert bool((room[:4096] == 85).all()) and bool((room[4096 + need:] == 85).all())
    # the same scratch, a step as it should be
    rows.cu.copy_(torch.tensor([0] + [n] * seqs, dtype=torch.int32))
    P.attend(cache, 0, rows, q, out, scratch=scratch)
    torch.cuda.synchronize()
    assert not out.any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("n,ctx,group", [(3, 37, 4), (3, 4000, 4), (7, 50, 4), (40, 37, 4), (40, 6000, 4),
                                         (70, 20, 3)])
def test_attend_values_that_are_not_finite(n, ctx, group, tree, dim, dtype):
    """Drafted rows whose keys are finite and some elements of whose values are not:
    the rows that see them are infinite or NaN in just those elements, in both
    kv heads' own, and right in the others; rows that do not see them are right
    everywhere."""
    counts, lens, page = [n, 2], [ctx, 50], 16
    g, k, v, table, cu, q = batch(counts, lens, dtype, 2, group, dim, page, 61)
    parents = [[-1] + [max(0, i - 2) for i in range(1, n)], [-1, 0]]
    seen = [R.ancestors(p) if tree else [list(range(i + 1)) for i in range(len(p))] for p in parents]
    mask = R.masks([js for s in seen for js in s], -(-n // 64)) if tree else None
    pg, row = R.slots(table, 0, page, ctx + n)
    odd = torch.zeros(n, 2, dim)  # what is put where, 0 elsewhere
    odd[1, 0, 3], odd[1, 0, dim - 1], odd[1, 1, 17] = math.inf, -math.inf, math.nan
    odd[2, 0, 3], odd[2, 1, 40], odd[n - 1, 1, 16] = -math.inf, math.inf, -math.inf
    if n > 66:  # rows of another 64-key tile
        odd[65, 0, 5], odd[66, 0, 5] = math.inf, math.inf
    where = odd != 0
    values = v[0, pg[ctx:], :, row[ctx:]]
    v[0, pg[ctx:], :, row[ctx:]] = torch.where(where, torch.zeros(()).to(dtype), values)
    want, tol = R.attention(q, k, v, table, cu, lens, seen, page, group, dim ** -0.5)
    v[0, pg[ctx:], :, row[ctx:]] = torch.where(where, odd.to(dtype), values)
    got = attended(k, v, table, counts, lens, q, mask)
    near(got[n:], want[n:], tol[n:], "the other sequence")
    for i in range(n):
        add = torch.stack([odd[j] for j in seen[0][i]]).sum(0).repeat_interleave(group, 0)
        fine = torch.stack([~where[j] for j in seen[0][i]]).all(0).repeat_interleave(group, 0)
        near(got[i][fine], want[i][fine], tol[i][fine], ("right elements", i))
        a, b = got[i].float()[~fine], add[~fine]
        assert torch.equal(torch.isnan(a), torch.isnan(b)), i
        assert torch.equal(a[~torch.isnan(b)], b[~torch.isnan(b)]), i


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("counts,lens,group", [
    ([40, 40, 40, 40, 40], [30, 30, 30, 30, 30], 4),       # tiles of 128 pairs, whole
    ([40, 40, 40, 40, 40], [9000, 9000, 700, 60, 60], 4),  # split: one item of several is bad
    ([2, 2, 2, 2, 2], [9000, 9000, 700, 60, 60], 4), ([5, 5, 5, 5, 5], [30, 5000, 4000, 60, 60], 4)])
def test_attend_bad_pages_and_lengths_of_split_tiles(counts, lens, group, dtype):
    """As test_attend_bad_pages_and_lengths_are_nan, tiles of 128 pairs and joined
    ones among them: a page that is none anywhere in the context makes every row
    of its sequence NaN, and no other."""
    g, k, v, table, cu, q = batch(counts, lens, dtype, 1, group, 64, 16, 10)
    seen = [[list(range(i + 1)) for i in range(n)] if s in (0, 2) else [[]] * n
            for s, n in enumerate(counts)]
    want, tol = R.attention(q, k, v, table, cu, [c if s in (0, 2) else 0 for s, c in enumerate(lens)],
                            seen, 16, group, 0.125)
    most = 16 * table.shape[1]
    for page, name in ((0, -1), (lens[1] // 32, k.shape[1]), (lens[1] // 16 - 1, 2 ** 31 - 1)):
        bad = table.clone()
        bad[1, page] = name
        rows = P.Rows.of(counts, lens[:3] + [-1, most - counts[4] + 1], DEV)
        got = attended(k, v, bad, counts, lens, q, None, rows=rows)
        seqs = [got[cu[s]:cu[s + 1]] for s in range(5)]
        assert all(torch.isnan(seqs[s]).all() for s in (1, 3, 4)), (page, name)
        for s in (0, 2):
            of = slice(cu[s], cu[s + 1])
            near(got[of], want[of], tol[of], (page, name, s))


def test_pages_beyond_32_bits_of_trees_and_commits():
    """As test_attend_beyond_32_bits: tiles of 128 pairs, whole and split, and the
    moves of accepted rows among pages past 2^32 bytes and elements of a layer."""
    kv, page, dim, group = 8, 256, 128, 4
    per = kv * page * dim
    pages = (1 << 32) // per + 9
    if torch.cuda.mem_get_info()[0] < 4 * 2 * per * pages:
        pytest.skip("not enough memory")
    k = torch.empty(2, pages, kv, page, dim, dtype=torch.float16, device=DEV)
    v = torch.empty_like(k)
    g = torch.Generator().manual_seed(12)
    at = [pages - 1, pages - 5, pages - 3, pages - 7]
    small = [torch.randn(2, 4, kv, page, dim, generator=g).half() for _ in range(2)]
    for x, p in enumerate(at):
        k[:, p], v[:, p] = small[0][:, x].to(DEV), small[1][:, x].to(DEV)
    cache = P.PagedCache.over(k, v, torch.tensor([at], dtype=torch.int32, device=DEV))
    n, tab = 20, torch.tensor([[0, 1, 2, 3]], dtype=torch.int32)
    parent = R.random_tree(n, g)
    q = torch.randn(n, kv * group, dim, generator=g).half()
    for ctx in (40, 900):
        rows = P.Rows.of([n], [ctx], DEV)
        _, slot, mask = P.plan(cache, rows, torch.tensor(parent, dtype=torch.int32, device=DEV))
        pg, row = R.slots(tab, 0, page, ctx + n)
        assert slot.tolist() == [at[int(p)] * page + int(r) for p, r in zip(pg[ctx:], row[ctx:])]
        got = P.attend(cache, 1, rows, q.to(DEV), mask=mask).cpu().view(q.shape)
        want, tol = R.attention(q, *small, tab, [0, n], [ctx], [R.ancestors(parent)], page, group,
                                1 / math.sqrt(dim), layer=1)
        near(got, want, tol, ("far pages", ctx))
    # a line from row 0 to every third row behind it
    rows = P.Rows.of([n], [500], DEV)  # from the second page into the third
    line = [max(0, (i - 1) // 3 * 3) if i % 3 == 0 else -1 for i in range(n)]
    ids = torch.arange(n, dtype=torch.int32)
    target = ids + 3
    i32 = {"dtype": torch.int32, "device": DEV}
    path, (count, nxt, new) = torch.empty(1, n, **i32), (torch.empty(1, **i32) for _ in range(3))
    P.commit(cache, rows, torch.tensor(line, **i32), ids.to(DEV), target.to(DEV), path, count, nxt, new)
    way, after = R.walk(line, ids.tolist(), target.tolist(), n)
    assert way == list(range(0, n, 3)) and path[0].tolist() == way + [-1] * (n - len(way))
    assert (count.item(), nxt.item(), new.item()) == (len(way), after, 500 + len(way))
    pg, row = R.slots(tab, 0, page, 500 + n)
    src, dst = [500 + i for i in way], list(range(500, 500 + len(way)))
    for x, pool in zip(small, (k, v)):
        x[:, pg[dst], :, row[dst]] = x[:, pg[src], :, row[src]].clone()
        for y, p in enumerate(at):
            assert torch.equal(pool[:, p].cpu(), x[:, y])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("counts,lens,group", [
    ([5, 8, 3], [40, 0, 300], 4), ([60, 9, 1], [0, 70, 500], 4), ([70, 33], [900, 0], 2), ([7], [4000], 1)])
def test_forests_planned_attended_and_committed(counts, lens, group, dtype):
    """Trees with several roots, and parents that are none, through plan,
    attention and commit: rows under another root than row 0 see their own
    ancestors, and are never accepted."""
    kv, dim, page = 2, 64, 16
    g, k, v, table, cu, q = batch(counts, lens, dtype, kv, group, dim, page, 71 + counts[0])
    trees = [R.random_forest(n, g) for n in counts]
    assert any(sum(not 0 <= p < i for i, p in enumerate(t)) > 1 for t in trees)
    anc = [R.ancestors(t) for t in trees]
    i32 = {"dtype": torch.int32, "device": DEV}
    kd, vd = k.to(DEV), v.to(DEV)
    cache = P.PagedCache.over(kd, vd, table.to(DEV))
    rows = P.Rows.of(counts, lens, DEV)
    parent = torch.tensor([p for t in trees for p in t], **i32)
    pos, slot, mask = P.plan(cache, rows, parent)
    assert torch.equal(mask.cpu(), R.masks([a for t in anc for a in t], mask.shape[1]))
    assert pos.tolist() == [c + len(a) - 1 for t, c in zip(anc, lens) for a in t]
    want, tol = R.attention(q, k, v, table, cu, lens, anc, page, group, 0.2)
    near(P.attend(cache, 0, rows, q.to(DEV), mask=mask, scale=0.2).cpu().view(q.shape), want, tol,
         "forests")
    # one token everywhere: whatever child there is, is accepted
    ids = torch.full((cu[-1],), 5, **i32)
    S, most = len(counts), max(counts)
    path, (count, nxt, new) = torch.empty(S, most, **i32), (torch.empty(S, **i32) for _ in range(3))
    P.commit(cache, rows, parent, ids, ids.clone(), path, count, nxt, new)
    torch.cuda.synchronize()
    for s, n in enumerate(counts):
        way, _ = R.walk([p if 0 <= p < i else -1 for i, p in enumerate(trees[s])], [5] * n, [5] * n, most)
        assert path[s].tolist() == way + [-1] * (most - len(way)) and count[s].item() == len(way)
        assert all(anc[s][i][0] == 0 for i in way)
        pg, row = R.slots(table, s, page, lens[s] + n)
        src, dst = [lens[s] + i for i in way], list(range(lens[s], lens[s] + len(way)))
        for pool in (k, v):
            pool[:, pg[dst], :, row[dst]] = pool[:, pg[src], :, row[src]].clone()
    for pool, now in ((k, kd), (v, vd)):
        assert torch.equal(now.cpu().view(torch.int16), pool.view(torch.int16))
