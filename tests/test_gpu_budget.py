"""Sampled verification, weights of keys and eviction on the GPU, against their
formulas in 64 bits (tests/_budget.py derives the bounds)."""
import math

import pytest

torch = pytest.importorskip("torch")

from plugins_amd import exl3 as X  # noqa: E402
from plugins_amd import paged as P  # noqa: E402
from tests import _budget as B  # noqa: E402
from tests import _paged as R  # noqa: E402
from tests.test_gpu_paged import batch  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


# --------------------------------------------------------------- verification

def drafted(counts, vocab, dtype, draft, distinct, seed, tree=True, heats=None):
    """Host tensors of a step: logits with a few likely tokens, drafts near them,
    trees whose tokens are among the likely ones."""
    g = torch.Generator().manual_seed(seed)
    T = sum(counts)
    z = torch.randn(T, vocab, generator=g)
    k = min(6, vocab)
    likely = torch.stack([torch.randperm(vocab, generator=g)[:k] for _ in range(T)]) if T else \
        torch.zeros(0, k, dtype=torch.long)
    z.scatter_(1, likely, 3 + 5 * torch.rand(T, k, generator=g))
    z = z.to(dtype)
    q = None
    if draft is not None:
        q = torch.softmax(z.float() + torch.randn(T, vocab, generator=g), -1).to(draft)
    parent, ids, at = [], [], 0
    for n in counts:
        p = R.random_forest(n, g) if tree else list(range(-1, n - 1))
        if tree and n:
            p[0] = -1
        taken = {}
        for i in range(n):
            up = p[i] if 0 <= p[i] < i else 0
            j = taken.get(up, 0)
            if not distinct and torch.rand(1, generator=g) < 0.3:
                j = int(torch.randint(0, k, (1,), generator=g))
            taken[up] = j + 1
            # distinct siblings go on past the likely ones
            ids.append(int(likely[at + up, j]) if j < k else (int(likely[at + up, 0]) + j) % vocab)
        parent += p
        at += n
    if heats is None:
        heats = [(0.7, 1.0, 0.0, 1.6)[s % 4] for s in range(len(counts))]
    u = torch.rand(T, generator=g, dtype=torch.float64)
    return z, q, parent, ids, heats, u


def expected(counts, z, q, parent, ids, heats, u, distinct):
    want, margin, at = [], math.inf, 0
    for s, n in enumerate(counts):
        own = [p if 0 <= p < i else -1 for i, p in enumerate(parent[at:at + n])]
        t, m = B.walk(own, ids[at:at + n], z[at:at + n], float(torch.tensor(heats[s], dtype=F32)),
                      u[at:at + n].tolist(), None if q is None else q[at:at + n], distinct)
        want += t
        margin = min(margin, m)
        at += n
    return want, margin


def verified(counts, z, q, parent, ids, heats, u, distinct, stream=None, **kw):
    rows = kw.pop("rows", None) or P.Rows.of(counts, [0] * len(counts), DEV)
    target = torch.full((rows.rows,), 77, dtype=torch.int32, device=DEV)
    i32 = {"dtype": torch.int32, "device": DEV}
    P.verify(rows, None if parent is None else torch.tensor(parent, **i32), torch.tensor(ids, **i32),
             z.to(DEV), u.to(DEV), target, draft=None if q is None else q.to(DEV),
             temperature=None if heats is None else torch.tensor(heats, device=DEV, dtype=F32),
             distinct=distinct, stream=stream, **kw)
    torch.cuda.synchronize()
    return target.cpu().tolist()


# f32 powers and their sum move a probability by (|score| + 8) 2^-23 or so of it: below
# 1e-5 for scores up to 80; a margin is what the nearest decision had (the sampled
# place's, in 64 bits, counts 1e7 times)
MARGIN = 1e-5


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("draft,distinct", [(None, False), (F32, False), (F16, True), (BF16, False)])
@pytest.mark.parametrize("counts,vocab,tree", [
    ([1], 1, True), ([1], 13, True), ([3, 0, 1, 6, 2], 7, True), ([5, 4, 1, 8], 1000, False),
    ([24, 9, 0, 31], 4097, True), ([33, 70], 8199, True), ([12, 7], 20011, True),
    ([1, 1, 1], 151936, True)])
def test_verify(counts, vocab, tree, draft, distinct, dtype):
    seed = 5 * vocab + 3
    while True:  # (a seed whose decisions are not at a border; found on the CPU alone)
        args = drafted(counts, vocab, dtype, draft, distinct, seed, tree)
        want, margin = expected(counts, *args, distinct)
        if margin > MARGIN:
            break
        seed += 1
    assert verified(counts, *args, distinct) == want
    if not tree:  # rows in a line need no parents
        z, q, parent, ids, heats, u = args
        assert verified(counts, z, q, None, ids, heats, u, distinct) == want


@pytest.mark.parametrize("counts,vocab,dtype,draft", [
    ([130, 90, 200, 0, 150], 67, BF16, None), ([130, 90, 200, 0, 150], 67, BF16, F32),
    ([600], 1501, BF16, None), ([64] * 9, 9001, BF16, F32),
    # read as the walks go
    ([64] * 9, 30011, BF16, F32), ([300, 0, 150], 20001, F32, F16), ([64] * 9, 151936, BF16, None),
    ([200, 0, 400], 151936, F16, None), ([9, 4, 1], 3200003, F32, None), ([3, 8, 1, 4], 600007, F32, BF16),
    ([64] * 9, 151936, F32, F16), ([30, 9], 2000003, F32, BF16)])
def test_verify_large_batches(counts, vocab, dtype, draft):
    """Batches of which the walks look at few rows."""
    seed = 1
    while True:
        args = drafted(counts, vocab, dtype, draft, draft is not None, seed)
        want, margin = expected(counts, *args, draft is not None)
        if margin > MARGIN:
            break
        seed += 1
    got = verified(counts, *args, draft is not None)
    assert got == want


@pytest.mark.parametrize("n,vocab,tree,draft", [
    (600, 67, False, None), (600, 67, True, None), (600, 151936, True, None), (600, 151936, False, None),
    (300, 60013, True, F16), (200, 1001, True, F16), (900, 151936, True, F16)])
def test_verify_a_path_that_is_deep(n, vocab, tree, draft):
    """Every row its parent's only child, and certain."""
    z = torch.zeros(n, vocab)
    ids = [(7 * i) % vocab for i in range(n)]
    for i in range(n - 1):
        z[i, ids[i + 1]] = 60.0
    z[n - 1, 5] = 60.0
    z = z.to(F16)
    q = None if draft is None else torch.full((n, vocab), 1.0 / vocab).to(draft)
    got = verified([n], z, q, list(range(-1, n - 1)) if tree else None, ids, [1.0],
                   torch.full((n,), 0.5, dtype=torch.float64), False)
    assert got == ids[1:] + [5]


@pytest.mark.parametrize("off", [1, 3])
@pytest.mark.parametrize("dtype,draft", [(F16, F32), (F32, BF16), (BF16, F16)])
def test_verify_strides_and_rows_behind(off, dtype, draft):
    """Logits and drafts within wider tensors, off their 16-byte boundaries; rows
    of no sequence, before the first and behind the last, stay as they were."""
    counts, vocab = [4, 6], 2500
    seed = 9
    while True:
        args = drafted(counts, vocab, dtype, draft, False, seed)
        want, margin = expected(counts, *args, False)
        if margin > MARGIN:
            break
        seed += 1
    z, q, parent, ids, heats, u = args

    def pad(t):
        w = torch.full((t.shape[0] + 5, vocab + 37), math.nan, dtype=t.dtype, device=DEV)
        w[2:2 + t.shape[0], off:off + vocab] = t.to(DEV)
        return w[:, off:off + vocab]

    rows = P.Rows(torch.tensor([2, 6, 12], dtype=torch.int32, device=DEV),
                  torch.zeros(2, dtype=torch.int32, device=DEV), 15, 6)
    u = torch.cat([torch.rand(2, dtype=torch.float64), u, torch.rand(3, dtype=torch.float64)])
    target = torch.full((15,), 77, dtype=torch.int32, device=DEV)
    i32 = {"dtype": torch.int32, "device": DEV}
    P.verify(rows, torch.tensor([0, 0, *parent, 0, 0, 0], **i32), torch.tensor([0, 0, *ids, 0, 0, 0], **i32),
             pad(z), u.to(DEV), target, draft=pad(q), temperature=torch.tensor(heats, device=DEV, dtype=F32))
    assert target.tolist() == [77, 77, *want, 77, 77, 77]


@pytest.mark.parametrize("rows,V", [(3, 50), (700, 50), (700, 60011)])
def test_verify_rows_without_a_distribution(rows, V):
    """NaN, +inf, nothing but -inf; temperatures that are none: the walk ends there
    with -1.  A largest logit of +inf is one at temperature 0."""
    counts = [3] * 9 + ([70] * 10 if rows > 3 else [])
    z = torch.zeros(sum(counts), V)
    z[:, 11] = 30.0  # every row says 11
    ids, parent = [11] * sum(counts), []
    for n in counts:
        parent += list(range(-1, n - 1))
    heats = [1.0] * len(counts)
    z[0, 4] = math.nan
    z[4, 2] = math.inf  # the second row of the second sequence
    z[6] = -math.inf
    heats[3], heats[4], heats[5] = -1.0, math.nan, math.inf
    heats[6] = heats[7] = 0.0
    z[18, 2] = math.inf
    z[21, 2] = math.nan
    z[25, :11], z[25, 12:] = -math.inf, -math.inf
    want = [-1, -1, -1, 11, -1, -1, -1, -1, -1] + [-1] * 9 + [2, -1, -1] + [-1, -1, -1] + [11] * 3 + \
        [11] * (sum(counts) - 27)
    u = torch.full((sum(counts),), 0.25, dtype=torch.float64)
    assert verified(counts, z, None, parent, ids, heats, u, False) == want


def test_verify_numbers_and_tokens_that_are_none():
    """u that is NaN or not below 1 accepts no child that is not certain and samples the
    last token of positive probability; a token outside the vocabulary is refused; a token
    twice among siblings has one chance; refused children are not sampled."""
    V = 40
    z = torch.full((4, V), -math.inf)
    z[:, 3], z[:, 8], z[:, 20] = 1.0, 2.0, 1.5
    u = torch.tensor([math.nan, 0.1, 0.1, 0.1], dtype=torch.float64)
    par = [-1, 0, 0, 0]

    def one(ids, u, **kw):
        return verified([4], z, kw.get("q"), par, ids, [1.0], torch.tensor(u, dtype=torch.float64), False)

    assert one([0, -5, V, 2 ** 31 - 1], [0.999999, 0.0, 0.0, 0.0])[0] == 20
    assert one([0, 1, 1, 1], [math.nan, math.nan, 0.0, 0.0])[0] == 20
    assert one([0, 8, 1, 1], [0.0, math.nan, 0.0, 0.0])[0] == 3
    assert one([0, 8, 8, 1], [1e-9, math.nan, 1e-9, 0.0])[0] == 3  # (the second 8 has nothing left)
    assert one([0, 3, 20, 8], [math.nan, math.nan, math.nan, math.nan])[0] == 20  # all refused: p itself
    assert one([0, 3, 20, 1], [0.5, 1.0, 1.0, 0.0])[0] == 8
    assert one([0, 1, 1, 1], [-1.0, 0.0, 0.0, 0.0])[0] == 3
    assert one([0, 1, 1, 1], [7.0, 0.0, 0.0, 0.0])[0] == 20
    # a token that the draft could not have drawn is taken where the target may say it
    q = torch.zeros(4, V)
    q[:, 5] = 1.0
    assert one([0, 8, 1, 1], [0.5, 0.999, 0.0, 0.0], q=q)[0] == 8
    # a draft that is the target itself accepts whatever it drew
    q = torch.softmax(z, -1)
    assert one([0, 3, 1, 1], [0.5, 0.99999, 0.0, 0.0], q=q)[0] == 3


@pytest.mark.parametrize("heat", [1e-30, 1e-42, 0.01, 1e30])
def test_verify_temperatures(heat):
    """From nearly greedy to nearly uniform."""
    V = 300
    g = torch.Generator().manual_seed(4)
    z, u = torch.randn(6, V, generator=g), torch.rand(6, generator=g, dtype=torch.float64)
    want, margin = expected([1] * 6, z, None, [-1] * 6, [0] * 6, [heat] * 6, u, False)
    assert margin > MARGIN
    assert verified([1] * 6, z, None, None, [0] * 6, [heat] * 6, u, False) == want
    if heat < 1e-20:
        assert want == z.argmax(-1).tolist()


def test_verify_a_vocabularys_tail_in_64_bits():
    """Half of the mass on one token, half spread over 151935 alike: the token that a
    number says is the formula's, whichever of the tail it is."""
    V, n = 151936, 64
    z = torch.full((n, V), 0.0)
    z[:, 0] = math.log(V - 1)
    u = torch.linspace(0.5000123, 0.99999, n, dtype=torch.float64)
    want, margin = expected([1] * n, z, None, [-1] * n, [0] * n, [1.0] * n, u, False)
    got = verified([1] * n, z, None, None, [0] * n, None, u, False)
    assert margin > 0 and got == want and len(set(want)) == n


def test_verify_graph_stream_and_commit():
    """Captured with a commit behind it, the inputs changed between replays of two
    graphs, beside an eager call; a stream of its own; calls repeat bit for bit."""
    counts, lens, vocab = [9, 1, 14], [30, 5, 80], 3001
    args = drafted(counts, vocab, F16, F32, True, 21)
    z, q, parent, ids, heats, u = args
    i32 = {"dtype": torch.int32, "device": DEV}
    g, k, v, table, cu, _ = batch(counts, lens, F16, 2, 1, 64, 16, 3)
    kd, vd = k.to(DEV), v.to(DEV)
    cache, rows = P.PagedCache.over(kd, vd, table.to(DEV)), P.Rows.of(counts, lens, DEV)
    zd, qd, ud = z.to(DEV), q.to(DEV), u.to(DEV)
    par, tok = torch.tensor(parent, **i32), torch.tensor(ids, **i32)
    heat = torch.tensor(heats, device=DEV, dtype=F32)

    def whole():
        target = torch.full((rows.rows,), 9, **i32)
        path, (count, after, new_len) = torch.empty(3, 14, **i32), (torch.empty(3, **i32) for _ in range(3))
        P.verify(rows, par, tok, zd, ud, target, draft=qd, temperature=heat, distinct=True)
        P.commit(cache, rows, par, tok, target, path, count, after, new_len)
        return target, path, count, after, new_len

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs, graphs = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=side, capture_error_mode="thread_local"):
            outs.append(whole())
        graphs.append(gr)
    for turn in range(4):
        seed = 100 + 50 * turn
        while True:
            new = drafted(counts, vocab, F16, F32, True, seed)
            want, margin = expected(counts, *new, True)
            if margin > MARGIN:
                break
            seed += 1
        zd.copy_(new[0]), qd.copy_(new[1]), par.copy_(torch.tensor(new[2])), tok.copy_(torch.tensor(new[3]))
        ud.copy_(new[5])
        torch.cuda.synchronize()
        for gr in graphs:
            gr.replay()
        eager = whole()
        torch.cuda.synchronize()
        for o in (*outs, eager):
            assert o[0].tolist() == want, turn
            at = 0
            for s, n in enumerate(counts):
                own = [p if 0 <= p < i else -1 for i, p in enumerate(new[2][at:at + n])]
                way, after = R.walk(own, new[3][at:at + n], want[at:at + n], 14)
                assert o[1][s].tolist() == way + [-1] * (14 - len(way)) and o[3][s].item() == after
                assert [x for x in want[at:at + n] if x >= 0] == [new[3][at + j] for j in way[1:]] + [after]
                at += n
    assert verified(counts, *new, True, stream=side) == want


def test_verify_many_sequences():
    """More sequences than a wave has lanes, many without rows."""
    g = torch.Generator().manual_seed(1)
    counts = [int(torch.randint(0, 4, (1,), generator=g)) for _ in range(150)]
    seed = 0
    while True:
        args = drafted(counts, 517, F32, F16, False, seed)
        want, margin = expected(counts, *args, False)
        if margin > MARGIN:
            break
        seed += 1
    assert verified(counts, *args, False) == want


# -------------------------------------------------------------------- weights

def weighed(k, table, counts, lens, q, had, mask=None, rows=None, v=None, **kw):
    kd = k.to(DEV)
    cache = P.PagedCache.over(kd, torch.empty_like(kd) if v is None else v, table.to(DEV))
    rows = rows or P.Rows.of(counts, lens, DEV)
    score = had.to(DEV)
    if kw.get("base") is not None:
        kw["base"] = torch.tensor(kw["base"], dtype=torch.int32, device=DEV)
    P.weigh(cache, kw.pop("layer", 0), rows, q.to(DEV), score, mask=None if mask is None else mask.to(DEV), **kw)
    torch.cuda.synchronize()
    return score.cpu()


def scores(seqs, kv, room, g):
    return torch.rand(seqs, kv, room, generator=g) * 3


WEIGH = [
    # counts, lens, kv, group, dim, page, window
    ([1], [0], 1, 1, 64, 16, 0),
    ([1], [2047], 2, 4, 128, 64, 0),
    ([1, 1, 1, 0], [15, 16, 17, 40], 2, 3, 64, 16, 0),
    ([5, 0, 3, 1], [31, 200, 0, 64], 2, 4, 128, 32, 0),
    ([17, 64, 2], [100, 3, 1000], 1, 8, 128, 16, 0),
    ([70, 1, 33], [0, 513, 250], 2, 5, 64, 64, 0),
    ([129], [300], 1, 2, 128, 256, 32),
    ([40, 7], [90, 700], 1, 7, 64, 128, 3),
    ([40, 7], [90, 700], 2, 4, 128, 64, 4),
    ([9, 4], [63, 1500], 3, 3, 64, 16, 0),
    ([33], [64], 5, 2, 64, 64, 1),
    ([60], [5000], 1, 4, 128, 64, 16),
    ([1, 1], [4095, 4096], 8, 1, 128, 256, 0),
    ([200], [0], 2, 2, 128, 16, 0),
    ([2, 4], [900, 33], 2, 4, 64, 32, 0),
    ([8, 3, 1], [2000, 77, 0], 2, 4, 128, 64, 0), ([17], [500], 1, 1, 64, 16, 0),
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("counts,lens,kv,group,dim,page,window", WEIGH)
@pytest.mark.parametrize("tree", [False, True])
def test_weigh(counts, lens, kv, group, dim, page, window, dtype, tree):
    g, k, v, table, cu, q = batch(counts, lens, dtype, kv, group, dim, page, 7 + sum(counts))
    parents = [R.random_tree(n, g) if n else [] for n in counts]
    seen = [R.ancestors(p) if tree else [list(range(i + 1)) for i in range(len(p))] for p in parents]
    mask = R.masks([js for s in seen for js in s], -(-max(counts) // 64)) if tree else None
    scale, room = 1 / math.sqrt(dim), max(n + c for n, c in zip(counts, lens)) + (sum(counts) % 3)
    had = scores(len(counts), kv, room, g)
    want, tol = B.weights(q, k, table, cu, lens, seen, page, group, scale, had, 0.9, window)
    got = weighed(k, table, counts, lens, q, had, mask, window=window, decay=0.9)
    off = (got.double() - want).abs() - tol
    assert not torch.isnan(got).any() and float(off.max()) <= 0, float(off.max())
    assert torch.equal(got, weighed(k, table, counts, lens, q, had, mask, window=window, decay=0.9))


@pytest.mark.parametrize("n", [1, 8, 30])
def test_weigh_base_decay_and_what_stays(n):
    """Keys from `base` on begin anew, whatever was there (NaN); keys behind the
    sequence's, sequences without rows and those that do not fit stay as they
    are, bit for bit."""
    counts, lens = [n, 0, n, n, 1], [40, 30, 10, 200, 7]
    g, k, v, table, cu, q = batch(counts, lens, F16, 2, 4, 64, 16, 8)
    room, base = 100, [12, 0, 999, 3, -4]
    had = scores(5, 2, room, g)
    had[0, :, 12:], had[2, :, 10 + n:], had[3], had[4] = math.nan, math.inf, 7.0, math.nan
    seen = [[list(range(i + 1)) for i in range(m)] for m in counts]
    fits = [0, 1, 2, 4]
    ref = had.clone()
    ref[3] = 0
    lens_ref = [c if s in fits else 0 for s, c in enumerate(lens)]
    ok = [s for s in fits if counts[s]]
    want = had.double()
    tol = torch.zeros_like(want)
    for s in ok:
        w, t = B.weights(q[cu[s]:cu[s + 1]], k, table[s:s + 1], [0, counts[s]], [lens_ref[s]], [seen[s]], 16, 4,
                         0.125, torch.nan_to_num(had[s:s + 1], nan=0.0, posinf=0.0), -0.5, 0, [base[s]])
        m = lens[s] + counts[s]
        want[s, :, :m], tol[s, :, :m] = w[0, :, :m], t[0, :, :m]
    got = weighed(k, table, counts, lens, q, had, decay=-0.5, base=base)
    for s in range(5):
        m = lens[s] + counts[s] if s in ok else 0
        assert ((got[s, :, :m].double() - want[s, :, :m]).abs() <= tol[s, :, :m]).all(), s
        assert torch.equal(got[s, :, m:].view(torch.int32), had[s, :, m:].view(torch.int32)), s


@pytest.mark.parametrize("what", [math.nan, math.inf])
@pytest.mark.parametrize("n,group", [(3, 4), (8, 4), (11, 4), (40, 4)])
def test_weigh_keeps_what_is_masked_out(what, n, group):
    """A drafted row whose key overflowed: rows that see it give NaN to what they see, the
    others' weights are as if it were not there: keys that only they see are
    finite."""
    counts, lens, page = [n, 2], [37, 50], 16
    g, k, v, table, cu, q = batch(counts, lens, BF16, 2, group, 128, page, 6)
    # two branches: odd rows under row 1 (the bad one), even ones under the root
    parents = [[-1] + [max(0, i - 2) for i in range(1, n)], [-1, 0]]
    seen = [R.ancestors(p) for p in parents]
    mask = R.masks([js for s in seen for js in s], 1)
    pg, row = R.slots(table, 0, page, 37 + n)
    k[0, pg[37 + 1], :, row[37 + 1]] = what
    had = scores(2, 2, 80, g)
    clean = k.clone()
    clean[0, pg[37 + 1], :, row[37 + 1]] = 0
    mute = [[js if 1 not in js else [] for js in s] for s in seen]
    want, tol = B.weights(q, clean, table, cu, lens, seen, page, group, 1 / math.sqrt(128), had)
    got = weighed(k, table, counts, lens, q, had, mask)
    even = [37 + i for i in range(2, n) if 1 not in seen[0][i]]
    for x in even:
        assert ((got[0, :, x].double() - want[0, :, x]).abs() <= tol[0, :, x]).all()
    assert not torch.isfinite(got[0, :, :38]).any() and not torch.isfinite(got[0, :, 38]).any()
    assert ((got[1].double() - want[1]).abs() <= tol[1]).all()
    assert mute


def test_weigh_free_masks_and_empty_rows():
    """Rows that see nothing give nothing; a key that no row sees has none."""
    counts, lens = [6, 70, 4], [0, 40, 0]
    g, k, v, table, cu, q = batch(counts, lens, F16, 2, 4, 128, 16, 5)
    seen = [[[j for j in range(n) if torch.rand(1, generator=g) < 0.4] for _ in range(n)] for n in counts]
    seen[0][2], seen[2] = [], [[] for _ in range(4)]
    mask = R.masks([js for s in seen for js in s], 3)
    had = scores(3, 2, 111, g)
    want, tol = B.weights(q, k, table, cu, lens, seen, 16, 4, 0.3, had)
    got = weighed(k, table, counts, lens, q, had, mask, scale=0.3)
    assert ((got.double() - want).abs() <= tol).all() and not got[2, :, :4].any()


@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-30, 3000.0])
@pytest.mark.parametrize("n", [2, 8, 30])
def test_weigh_scales(scale, n):
    counts, lens = [n], [150]
    g, k, v, table, cu, q = batch(counts, lens, F16, 1, 4, 64, 16, 7)
    q, k = (q * 4).round() / 4, (k * 4).round() / 4  # scores that 32 bits hold exactly
    seen = [[list(range(i + 1)) for i in range(n)]]
    had = scores(1, 1, 200, g)
    got = weighed(k, table, counts, lens, q, had, scale=scale)
    want, tol = B.weights(q, k, table, cu, lens, seen, 16, 4, scale, had)
    if abs(scale) > 1:
        # scores of 2^16 and more: their scaling's rounding, 2^-24 of a score, moves a power
        # of e by up to 2^-24 max|score|
        top = float((q.double().abs().sum(-1).max() * k[~torch.isnan(k)].double().abs().max()) * scale)
        tol = tol + (want - torch.where(torch.arange(200) < 150, had.double(), 0.0)).abs() * 2.4 * top * 2.0 ** -23
    assert ((got.double() - want).abs() <= tol).all()


def test_weigh_strides_layers_and_rows_behind():
    """q within a wider tensor, another layer, rows of no sequence, and the first
    sequence's rows not at the tensor's start."""
    counts, lens = [4, 20], [70, 130]
    for cs in (counts, [4, 3]):
        g, k, v, table, cu, q = batch(cs, lens, BF16, 2, 4, 128, 32, 9, layers=3)
        had = scores(2, 2, 160, g)
        seen = [[list(range(i + 1)) for i in range(n)] for n in cs]
        want, tol = B.weights(q, k, table, cu, lens, seen, 32, 4, 1 / math.sqrt(128), had, layer=2)
        T = sum(cs)
        wide = torch.full((T + 6, 2000), math.nan, dtype=BF16, device=DEV)
        wide[3:3 + T, 8:1032] = q.view(T, -1).to(DEV)
        rows = P.Rows(torch.tensor([3, 3 + cs[0], 3 + T], dtype=torch.int32, device=DEV),
                      torch.tensor(lens, dtype=torch.int32, device=DEV), T + 6, max(cs))
        kd, score = k.to(DEV), had.to(DEV)
        P.weigh(P.PagedCache.over(kd, torch.empty_like(kd), table.to(DEV)), 2, rows, wide[:, 8:1032], score)
        assert ((score.cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("n", [1, 8, 40])
def test_weigh_bad_pages_and_lengths(n):
    """A page number outside the cache: NaN; a length that does not fit: untouched."""
    counts, lens = [n, n, n], [100, 60, 80]
    g, k, v, table, cu, q = batch(counts, lens, F16, 2, 4, 64, 16, 12)
    had = scores(3, 2, 200, g)
    table[1, 2] = 10 ** 6
    bad = [100, 60, -1]
    got = weighed(k, table, counts, lens, q, had, rows=P.Rows.of(counts, bad, DEV))
    seen = [[list(range(i + 1)) for i in range(n)]]
    want, tol = B.weights(q[:n], k, table[:1], cu[:2], lens[:1], seen, 16, 4, 0.125, had[:1])
    assert ((got[:1].double() - want).abs() <= tol).all()
    assert torch.isnan(got[1, :, :60 + n]).all() and torch.equal(got[1, :, 60 + n:], had[1, :, 60 + n:])
    assert torch.equal(got[2], had[2])
    # cu that goes back: nothing is done
    rows = P.Rows(torch.tensor([0, n, 0, 3 * n], dtype=torch.int32, device=DEV),
                  torch.tensor(lens, dtype=torch.int32, device=DEV), 3 * n, 3 * n)
    assert torch.equal(weighed(k, table, counts, lens, q, had, rows=rows), had)


@pytest.mark.parametrize("n", [1, 7, 50])
def test_weigh_graph_and_stream(n):
    """Captured twice over the same rows, lengths and q changed between the replays,
    eager calls beside them; another stream."""
    counts, lens = [n, 2], [500, 70]
    g, k, v, table, cu, q = batch(counts, lens, BF16, 2, 4, 128, 32, 13, max_pages=40)
    had = scores(2, 2, 600, g)
    kd = k.to(DEV)
    cache, rows, qd = P.PagedCache.over(kd, torch.empty_like(kd), table.to(DEV)), P.Rows.of(counts, lens, DEV), q.to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs, graphs = [], []
    for _ in range(2):
        out = torch.empty(2, 2, 600, device=DEV)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=side, capture_error_mode="thread_local"):
            P.weigh(cache, 0, rows, qd, out, decay=0.5)
        outs.append(out)
        graphs.append(gr)
    for turn in range(3):
        new = [500 - 100 * turn, 70 - 30 * turn]
        rows.len.copy_(torch.tensor(new, dtype=torch.int32))
        qd.copy_(q * (1 + turn))
        want = weighed(k, table, counts, new, q * (1 + turn), had, decay=0.5)
        for gr, out in zip(graphs, outs):
            out.copy_(had)
            torch.cuda.synchronize()
            gr.replay()
        eager = had.to(DEV)
        P.weigh(cache, 0, rows, qd, eager, decay=0.5)
        torch.cuda.synchronize()
        for out in (*outs, eager):
            assert torch.equal(out.cpu(), want), turn
    out = had.to(DEV)
    side.wait_stream(torch.cuda.current_stream())
    P.weigh(cache, 0, rows, qd, out, decay=0.5, stream=side)
    side.synchronize()
    assert torch.equal(out.cpu(), want)


def test_weigh_many_sequences():
    g = torch.Generator().manual_seed(14)
    for most in (2, 20):
        counts = [int(torch.randint(0, most, (1,), generator=g)) for _ in range(150)]
        lens = [int(torch.randint(0, 90, (1,), generator=g)) for _ in range(150)]
        lens[70], counts[70], counts[149] = 3000, 1, 1
        _, k, v, table, cu, q = batch(counts, lens, F16, 1, 5, 64, 16, 15)
        seen = [[list(range(i + 1)) for i in range(n)] for n in counts]
        had = scores(150, 1, 3001, g)
        want, tol = B.weights(q, k, table, cu, lens, seen, 16, 5, 0.125, had)
        assert ((weighed(k, table, counts, lens, q, had).double() - want).abs() <= tol).all()


# ------------------------------------------------------------------- eviction

def evicted(k, v, score, table, lens, most, keep=None, first=0, last=0, in_place=False, stream=None):
    """(k, v, kept, new_score, new_len) after it, on the host."""
    layers, seqs, kv, _ = score.shape
    cache = P.PagedCache.over(k.to(DEV), v.to(DEV), table.to(DEV))
    i32 = {"dtype": torch.int32, "device": DEV}
    sd = score.to(DEV)
    new = sd if in_place else torch.full_like(sd, 9.0)
    kept, new_len = torch.full((layers, seqs, kv, most), 55, **i32), torch.full((seqs,), 55, **i32)
    P.evict(cache, torch.tensor(lens, **i32), sd, kept, new, new_len, first=first, last=last, stream=stream,
            keep=None if keep is None else torch.tensor(keep, **i32))
    torch.cuda.synchronize()
    return cache.k.cpu(), cache.v.cpu(), kept.cpu(), new.cpu(), new_len.cpu()


def check_evicted(k, v, score, table, lens, page, most, keep=None, first=0, last=0, in_place=False):
    got = evicted(k, v, score, table, lens, most, keep, first, last, in_place)
    kept, new_len = B.eviction(score, lens, page, table, k.shape[1], keep, most, first, last)
    wk, wv = k.clone(), v.clone()
    ws = score.clone() if in_place else torch.full_like(score, 9.0)
    assert got[4].tolist() == new_len
    for lyr in range(score.shape[0]):
        for s in range(len(lens)):
            for h in range(score.shape[2]):
                x = kept[lyr][s][h]
                if x is None:
                    assert (got[2][lyr, s, h] == -1).all()
                    continue
                assert got[2][lyr, s, h].tolist() == x + [-1] * (most - len(x)), (lyr, s, h)
                if not x:
                    continue
                at, to = torch.tensor(x), torch.arange(len(x))
                a, b = table[s, at // page].long(), table[s, to // page].long()
                for w, pool in ((wk, k), (wv, v)):
                    w[lyr, b, h, to % page] = pool[lyr, a, h, at % page]
                ws[lyr, s, h, :len(x)] = score[lyr, s, h, at]
    bits = lambda t: t.view(torch.int16 if t.element_size() == 2 else torch.int32)  # noqa: E731
    assert torch.equal(bits(got[0]), bits(wk)) and torch.equal(bits(got[1]), bits(wv))
    assert torch.equal(bits(got[3]), bits(ws))


def pool_of(lens, kv, dim, page, layers, dtype, seed, extra=2):
    g = torch.Generator().manual_seed(seed)
    table, pages = R.random_table([0] * len(lens), lens, page, extra, g)
    shape = (layers, pages, kv, page, dim)
    return g, torch.randn(shape, generator=g).to(dtype), torch.randn(shape, generator=g).to(dtype), table


EVICT = [
    # lens, kv, dim, page, layers, most, first, last, room more than the longest
    ([1], 1, 64, 16, 1, 1, 0, 0, 0),
    ([2], 1, 64, 16, 1, 1, 0, 0, 3),
    ([5, 0, 17], 2, 128, 16, 2, 4, 1, 1, 1),
    ([100, 30, 31, 29], 2, 64, 32, 2, 30, 4, 8, 0),
    ([1000, 64, 999], 2, 128, 64, 2, 300, 4, 32, 5),
    ([300], 3, 64, 256, 3, 299, 0, 0, 0),
    ([3000, 2500], 1, 128, 16, 1, 2304, 4, 2300, 0),
    ([9000], 2, 64, 128, 1, 700, 4, 32, 7),
    ([600, 700], 2, 128, 64, 1, 10, 20, 5, 0),
    ([5000], 1, 128, 64, 2, 4200, 0, 1, 2),
    ([4096, 2049, 2048], 1, 64, 16, 1, 2048, 4, 0, 0), ([16384, 4097], 1, 64, 64, 1, 8000, 1, 3, 0),
    ([20000, 9001], 1, 64, 64, 1, 9000, 3, 5, 0), ([70001, 33000], 1, 64, 256, 1, 40000, 7, 100, 3),
    ([50000], 1, 64, 256, 1, 3000, 0, 40, 0),
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lens,kv,dim,page,layers,most,first,last,more", EVICT)
@pytest.mark.parametrize("in_place", [False, True])
def test_evict(lens, kv, dim, page, layers, most, first, last, more, in_place, dtype):
    g, k, v, table = pool_of(lens, kv, dim, page, layers, dtype, 3 + sum(lens))
    score = torch.exp(2 * torch.randn(layers, len(lens), kv, max(lens) + more, generator=g))
    check_evicted(k, v, score, table, lens, page, most, None, first, last, in_place)


@pytest.mark.parametrize("kind", ["alike", "few", "signs", "strange", "ascending", "tiny", "close"])
@pytest.mark.parametrize("n", [700, 40000])
def test_evict_scores(kind, n):
    """Scores that are alike, of few values, of both signs and zeros, infinities and NaN,
    in order, below the smallest normal number, or next to one another; more of them
    than registers hold."""
    if n > 1000 and kind in ("tiny", "signs"):
        pytest.skip("the small size covers it")
    page = 64
    g, k, v, table = pool_of([n, n - 33], 1, 64, page, 1, F16, 4)
    shape = (1, 2, 1, n)
    x = torch.randn(shape, generator=g)
    score = {"alike": torch.full(shape, 0.25), "few": (x * 2).round(), "signs": torch.where(x > 0.5, 0.0, -0.0) + (x < -1) * x,
             "strange": torch.where(x > 2, math.inf, torch.where(x < -2, -math.inf, torch.where(x.abs() < 0.2, math.nan, x))),
             "ascending": torch.arange(n, dtype=F32).expand(shape).clone(), "tiny": x * 1e-41,
             "close": 1 + torch.randint(0, 300, shape, generator=g) * 2.0 ** -23}[kind]
    for most in (1, n // 3, n - 40):
        check_evicted(k, v, score.contiguous(), table, [n, n - 33], page, most, None, 2, 5, kind == "few")


def test_evict_budgets_of_sequences():
    """A budget a sequence: less than most, none (below 0: as it is), all (0), more than
    there are; lengths and pages that are not right."""
    lens = [200, 150, 90, 60, 120, 80, 40]
    g, k, v, table = pool_of(lens, 2, 128, 16, 2, BF16, 5)
    score = torch.rand(2, 7, 2, 180, generator=g)  # the first has more keys than there is room
    table[4, 3] = 10 ** 6
    table[5, 4] = -1
    check_evicted(k, v, score, table, lens, 16, 100, [50, 33, -1, 0, 20, 10, 400], 3, 4)
    # (a bad page behind the keys is nobody's)
    table[6] = torch.cat([table[6, :3], torch.full((table.shape[1] - 3,), -1, dtype=torch.int32)])
    check_evicted(k, v, score, table, lens, 16, 100, [50, 33, -1, 0, 20, 10, 7], 3, 4, True)
    out = evicted(k, v, score, table, [-5, 5000, 90, 60, 0, 0, 0], 10)
    assert out[4].tolist() == [-5, 5000, 10, 10, 0, 0, 0]


def test_evict_graph_and_stream():
    """Captured, with scores, lengths and budgets changed between replays, which go on
    from what the last left; an eager twin beside it."""
    lens = [300, 260]
    g, k, v, table = pool_of(lens, 2, 64, 16, 2, F16, 6)
    i32 = {"dtype": torch.int32, "device": DEV}
    side = torch.cuda.Stream()

    def state():
        return {"c": P.PagedCache.over(k.to(DEV), v.to(DEV), table.to(DEV)), "s": torch.empty(2, 2, 2, 300, device=DEV),
                "kept": torch.empty(2, 2, 2, 290, **i32), "n": torch.empty(2, **i32), "len": torch.tensor(lens, **i32),
                "keep": torch.tensor([290, 250], **i32)}

    def call(x, stream=None):
        P.evict(x["c"], x["len"], x["s"], x["kept"], x["s"], x["n"], keep=x["keep"], first=1, last=2, stream=stream)

    a, b = state(), state()
    side.wait_stream(torch.cuda.current_stream())
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=side, capture_error_mode="thread_local"):
        call(a)
    now = list(lens)
    for turn in range(4):
        score, keep = torch.randn(2, 2, 2, 300, generator=g), [max(1, x - 40 * turn - 3) for x in now]
        for x in (a, b):
            x["s"].copy_(score), x["keep"].copy_(torch.tensor(keep))
        torch.cuda.synchronize()
        gr.replay()
        call(b, side if turn % 2 else None)
        torch.cuda.synchronize()
        for name in ("s", "kept", "n"):
            assert torch.equal(a[name], b[name]), (turn, name)
        assert torch.equal(a["c"].k, b["c"].k) and torch.equal(a["c"].v, b["c"].v)
        now = a["n"].tolist()
        assert now == [min(x, 290) for x in keep]  # (kept holds 290)
        for x in (a, b):
            x["len"].copy_(x["n"])


# ----------------------------------------------------------------- refusals

def test_tensors_that_are_refused():
    k = torch.zeros(1, 8, 2, 16, 64, dtype=F16, device=DEV)
    cache = P.PagedCache.over(k, k.clone(), torch.zeros(2, 4, dtype=torch.int32, device=DEV))
    rows = P.Rows.of([2, 1], [5, 9], DEV)
    i32 = {"dtype": torch.int32, "device": DEV}
    z, u = torch.zeros(3, 20, device=DEV), torch.zeros(3, dtype=torch.float64, device=DEV)
    ids, target = torch.zeros(3, **i32), torch.zeros(3, **i32)
    for bad in (dict(z=z.double()), dict(z=z.int()), dict(u=u.float()), dict(target=target.long()), dict(ids=ids.long()),
                dict(heat=torch.zeros(2, device=DEV, dtype=F16))):
        a = {"z": z, "u": u, "target": target, "ids": ids, "heat": None, **bad}
        with pytest.raises(TypeError):
            P.verify(rows, None, a["ids"], a["z"], a["u"], a["target"], temperature=a["heat"])
    for bad in (dict(z=z[:2]), dict(z=z.t().contiguous().t()), dict(z=z[0]), dict(z=z.cpu()), dict(u=u[:2]),
                dict(u=u.cpu()), dict(draft=z[:, :19]), dict(target=target[:2]), dict(ids=ids.cpu()),
                dict(heat=torch.zeros(3, device=DEV)), dict(scratch=torch.zeros(9999999, dtype=torch.uint8))):
        a = {"z": z, "u": u, "target": target, "ids": ids, "heat": None, "draft": None, "scratch": None, **bad}
        with pytest.raises(ValueError):
            P.verify(rows, None, a["ids"], a["z"], a["u"], a["target"], draft=a["draft"], temperature=a["heat"],
                     scratch=a["scratch"])
    with pytest.raises(X.Exl3Error, match="PagedScratch"):
        P.verify(rows, None, ids, z, u, target, scratch=torch.zeros(16, dtype=torch.uint8, device=DEV))
    with pytest.raises(X.Exl3Error, match="PagedOverlap"):
        P.verify(rows, None, ids, z, u, ids)
    q, score = torch.zeros(3, 512, dtype=F16, device=DEV), torch.zeros(2, 2, 40, device=DEV)
    for bad in (score.half(), score.double()):
        with pytest.raises(TypeError):
            P.weigh(cache, 0, rows, q, bad)
    for bad in (score[:1], score[:, :1], score[:, :, ::2], score.cpu(), score[0]):
        with pytest.raises(ValueError):
            P.weigh(cache, 0, rows, q, bad)
    with pytest.raises(X.Exl3Error, match="PagedWindow"):
        P.weigh(cache, 0, rows, q, score, window=-1)
    with pytest.raises(OverflowError):
        P.weigh(cache, 0, rows, q, score, window=1 << 32)
    lens, kept, s4 = torch.zeros(2, **i32), torch.zeros(1, 2, 2, 4, **i32), torch.zeros(1, 2, 2, 40, device=DEV)
    for a, b, c in ((s4[0], kept, s4), (s4, kept[0], s4), (s4, kept, s4[..., :39]), (s4[:, :1], kept, s4),
                    (s4, kept[..., ::2], s4)):
        with pytest.raises(ValueError):
            P.evict(cache, lens, a, b, c, torch.zeros(2, **i32))
    with pytest.raises(X.Exl3Error, match="PagedOverlap"):
        P.evict(cache, lens, s4, kept, s4, lens)
    with pytest.raises(X.Exl3Error, match="most above 0"):
        P.evict(cache, lens, s4, kept[..., :0], s4, torch.zeros(2, **i32))
    with pytest.raises(OverflowError):
        P.evict(cache, lens, s4, kept, s4, torch.zeros(2, **i32), first=1 << 40)
