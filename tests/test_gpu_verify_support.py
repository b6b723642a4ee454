"""Sampled verification where few tokens may follow at all (a grammar's mask): a draft's
roundings then leave nothing of the target's probabilities after a refusal, or every token
that may follow is among the children.  The walk still ends in a token that may follow,
and exl3p_commit takes the same way to it."""
import math
import random

import pytest

torch = pytest.importorskip("torch")

from plugins_amd import paged as P  # noqa: E402
from tests import _paged as R  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
I32 = {"dtype": torch.int32, "device": DEV}
BELOW_ONE = 1 - 2.0 ** -53  # the largest of numbers in [0, 1)


def masked(seqs, n, fan, support, vocab, dtype, draft, seed, order):
    """Trees of n rows of which each has up to `fan` children, among the `support` tokens
    that its logits leave; draft: the softmax of the same logits, rounded."""
    rng, g = random.Random(seed), torch.Generator(device=DEV).manual_seed(seed)
    T = seqs * n
    one = [-1] + [(i - 1) // fan for i in range(1, n)]
    tokens = torch.randint(0, vocab // support, (T, support), generator=g, device=DEV) + \
        torch.arange(support, device=DEV) * (vocab // support)
    z = torch.full((T, vocab), float("-inf"), dtype=dtype, device=DEV)
    some = torch.randn(T, support, generator=g, device=DEV).to(dtype)
    z.scatter_(1, tokens, some)
    q = None
    if draft is not None:
        q = torch.zeros(T, vocab, dtype=draft, device=DEV)
        q.scatter_(1, tokens, torch.softmax(some.double(), -1).to(draft))
    may, ids = tokens.tolist(), []
    for s in range(seqs):
        taken = {}
        for i in range(n):
            up = s * n + max(0, one[i])
            if up not in taken:
                taken[up] = list(may[up])
                if order == "any":
                    rng.shuffle(taken[up])
                elif order == "twice":  # drawn with replacement
                    taken[up] = [rng.choice(may[up]) for _ in range(fan + 1)]
            ids.append(taken[up].pop(0) if i and taken[up] else may[up][0])
    u = [BELOW_ONE if rng.random() < 0.6 else rng.random() for _ in range(T)]
    return z, q, one * seqs, ids, torch.tensor(u, dtype=torch.float64), may


@pytest.mark.parametrize("seqs,n,fan,support,vocab,dtype,draft,order", [
    # one launch: lines, and trees of certain tokens
    (400, 2, 1, 2, 40, F16, BF16, "any"), (400, 5, 1, 2, 4100, F32, F16, "any"), (300, 3, 1, 3, 60, BF16, F32, "any"),
    (300, 4, 3, 3, 50, F32, None, "any"), (100, 13, 3, 3, 9000, F16, None, "any"), (200, 2, 1, 1, 30, F16, BF16, "any"),
    # rounds: drawn siblings
    (300, 3, 2, 2, 40, F16, BF16, "any"), (300, 3, 2, 2, 40, F16, BF16, "twice"), (100, 7, 2, 2, 5000, BF16, F16, "any"),
    (100, 13, 3, 3, 300, F32, BF16, "any"), (100, 13, 3, 3, 300, F32, F32, "twice"),
    # the lone workgroup's
    (50, 60, 3, 3, 900, F16, BF16, "any"), (60, 40, 5, 5, 9000, F32, F16, "twice"), (8, 300, 4, 4, 2000, BF16, BF16, "any"),
    # read as the walks go
    (80, 13, 3, 3, 151936, F16, None, "any"), (90, 13, 3, 3, 151936, F16, BF16, "any"),
    (90, 13, 3, 3, 151936, BF16, F16, "twice"), (3, 200, 3, 3, 500009, F16, BF16, "any")])
def test_a_walk_ends_in_a_token_that_may_follow(seqs, n, fan, support, vocab, dtype, draft, order):
    for seed in range(3):
        z, q, parent, ids, u, may = masked(seqs, n, fan, support, vocab, dtype, draft, seed, order)
        target = torch.full((seqs * n,), 77, **I32)
        P.verify(P.Rows.of([n] * seqs, [0] * seqs, DEV), None if fan == 1 and seed else torch.tensor(parent, **I32),
                 torch.tensor(ids, **I32), z, u.to(DEV), target, draft=q,
                 distinct=order == "any" and fan > 1)
        target = target.tolist()
        for s in range(seqs):
            at, got = s * n, target[s * n:s * n + n]
            path, after = R.walk(parent[at:at + n], ids[at:at + n], got, n)
            assert [i for i in range(n) if got[i] != -1] == path, (seed, s, path, got[:8])
            for i in path:
                assert got[i] in may[at + i], (seed, s, i)
            assert after == got[path[-1]] != -1


@pytest.mark.parametrize("draft", [None, BF16])
def test_nothing_left_is_accepted_after_all(draft):
    """Two tokens may follow, of 0.6 and 0.4; the draft's nearest numbers of 8 bits are above
    both (154 / 256 and 205 / 512): a number next to 1 refuses the first by the rounding alone, and no token
    has anything left.  Without a draft both are children, and certain."""
    V, n = 64, 4
    z = torch.full((n, V), float("-inf"), device=DEV)
    z[:, 5], z[:, 40] = 0.4054651, 0.0  # ln 1.5
    q = None
    if draft is not None:
        q = torch.zeros(n, V, device=DEV, dtype=draft)
        q[:, 5], q[:, 40] = 154 / 256, 205 / 512
    for ids, parent, distinct, path in (([1, 5, 40, 5], [-1, 0, 0, 1], True, None), ([1, 40, 5, 40], [-1, 0, 0, 1], True, None),
                                        ([1, 5, 40, 5], [-1, 0, 1, 2], False, [0, 1, 2, 3])):
        if draft is None and path:
            continue  # (in a line the other token is left)
        target = torch.empty(n, **I32)
        u = torch.tensor([0.3] + [BELOW_ONE] * 3, dtype=torch.float64, device=DEV)
        P.verify(P.Rows.of([n], [0], DEV), torch.tensor(parent, **I32), torch.tensor(ids, **I32), z, u, target, draft=q,
                 distinct=distinct)
        got = target.tolist()
        way, after = R.walk(parent, ids, got, n)
        assert after in (5, 40) and len(way) >= 2
        if path:
            assert way == path and got[:3] == ids[1:]


def test_a_token_that_may_not_follow_is_not_accepted_for_want_of_others():
    """The draft's token has no probability at all and what it leaves of the others is below
    its own roundings: the others stay as they were."""
    V = 64
    z = torch.full((2, V), float("-inf"), device=DEV)
    z[:, 5], z[:, 40] = 0.4054651, 0.0
    q = torch.zeros(2, V, device=DEV, dtype=BF16)
    q[:, 5], q[:, 40], q[:, 9] = 154 / 256, 205 / 512, 1 / 512
    for token in (9, -3, V):
        for first, want in ((0.3, 5), (0.7, 40)):
            target = torch.empty(2, **I32)
            u = torch.tensor([first, 0.5], dtype=torch.float64, device=DEV)
            P.verify(P.Rows.of([2], [0], DEV), None, torch.tensor([1, token], **I32), z, u, target, draft=q)
            assert target.tolist() == [want, -1]


@pytest.mark.parametrize("how", ["line", "siblings", "distinct", "certain"])
@pytest.mark.parametrize("tokens,near", [(2, 0.0), (3, 0.0), (3, 0.5)])
def test_tokens_are_as_often_as_the_target_says(tokens, near, how):
    """The first token behind 196605 roots, whose drafts (of 8 bits) are the target itself or
    near it.  A share's standard deviation is at most sqrt(1 / 4 / 196605) = 0.00113; six of
    them, and what the draft's roundings move: half a step, 2^-8 of a share of at most 1."""
    V, S, n = 48, 65535, {"line": 2, "siblings": 4, "distinct": 1 + tokens, "certain": tokens}[how]
    g = torch.Generator(device=DEV).manual_seed(tokens)
    may = torch.tensor([5, 40, 21][:tokens], device=DEV)
    x = torch.tensor([0.41, 0.0, -0.7][:tokens], device=DEV)
    p = torch.softmax(x.double(), 0)
    q = torch.softmax(x.double() + near * torch.tensor([1.0, -1.0, 0.3][:tokens], device=DEV), 0).to(BF16)
    z = torch.full((1, V), float("-inf"), device=DEV)
    z[0, may] = x
    draft = torch.zeros(1, V, dtype=BF16, device=DEV)
    draft[0, may] = q
    z, draft = z.repeat(S * n, 1), draft.repeat(S * n, 1)
    parent = torch.tensor(([-1] + [0] * (n - 1)) * S, **I32)
    seen = torch.zeros(V, dtype=torch.long, device=DEV)
    for _ in range(3):
        key = torch.empty(S, n, tokens, device=DEV).exponential_(generator=g)
        if how in ("distinct", "certain"):
            pick = (key[:, 0] / q.float()).argsort(-1)
            ids = torch.cat([pick[:, :1], pick], 1)[:, :n]
        else:
            ids = (key / q.float()).argmin(-1)
        target = torch.empty(S * n, **I32)
        u = torch.rand(S * n, dtype=torch.float64, generator=g, device=DEV)
        P.verify(P.Rows.of([n] * S, [0] * S, DEV), parent, may[ids].flatten().int(), z, u, target,
                 draft=None if how == "certain" else draft, distinct=how == "distinct")
        seen += torch.bincount(target.view(S, n)[:, 0].clamp(min=0), minlength=V)
    off = (seen[may].double() / (3 * S) - p).abs()
    assert int(seen.sum() - seen[may].sum()) == 0
    assert (off < 6 * 0.00113 + (0 if how == "certain" else 2.0 ** -8)).all(), off.tolist()


@pytest.mark.parametrize("bad", [float("nan"), 1.0, 7.0, -1.0])
@pytest.mark.parametrize("seqs,n,fan,support,vocab,dtype,draft,order", [
    (200, 3, 1, 2, 40, F16, BF16, "any"), (200, 3, 2, 2, 40, F16, BF16, "any"), (100, 13, 3, 3, 9000, BF16, F16, "twice"),
    (40, 60, 3, 3, 900, F32, BF16, "any"), (100, 4, 3, 3, 50, F32, None, "any"), (90, 13, 3, 3, 151936, F16, BF16, "any")])
def test_numbers_that_are_none_beside_others(seqs, n, fan, support, vocab, dtype, draft, order, bad):
    """Any of the numbers is NaN, or not in [0, 1): every row of a walk still has a token that may
    follow, and calls repeat."""
    z, q, parent, ids, u, may = masked(seqs, n, fan, support, vocab, dtype, draft, 5, order)
    u[torch.rand(len(u), generator=torch.Generator().manual_seed(2)) < 0.5] = bad
    out = []
    for _ in range(3):
        target = torch.full((seqs * n,), 77, **I32)
        P.verify(P.Rows.of([n] * seqs, [0] * seqs, DEV), torch.tensor(parent, **I32), torch.tensor(ids, **I32), z, u.to(DEV),
                 target, draft=q, distinct=order == "any" and fan > 1)
        out.append(target.tolist())
    assert out[0] == out[1] == out[2]
    for t, x in enumerate(out[0]):
        assert x == -1 or x in may[t] or bad < 0
        assert t % n or x != -1


def kept_walk(parent, ids, p, u, q, distinct):
    """(target, margin) of one sequence in 64 bits, as tests._budget.walk, with the rule for
    refusals that leave nothing; p, q: {token: probability} of each row, what is not there is 0."""
    n, target, margin, at = len(ids), [-1] * len(ids), math.inf, 0
    while True:
        rest, A, B, share, to = dict(p[at]), 1.0, 1.0, 0.0, None
        for c in (c for c in range(at + 1, n) if parent[c] == at):
            x = ids[c]
            mine, drawn = rest.get(x, 0.0), 1.0 if q is None else q[at].get(x, 0.0)
            step = A if q is None else A / max(B, 2.0 ** -53)
            need = u[c] * step * drawn
            if max(need, mine) > 0:
                margin = min(margin, abs(need - mine) / max(need, mine))
            if need < mine:
                to = c
                break
            B -= drawn if distinct else 0.0
            if q is None:
                less = {k: 0.0 if k == x else v for k, v in rest.items()}
            else:
                less = {k: max(v - (share + step) * q[at].get(k, 0.0) * (1 + 2.0 ** -48), 0.0) for k, v in p[at].items()}
            if any(less.values()):
                rest, share = less, share + step
                A = A - mine if q is None else sum(rest.values())
                margin = min(margin, 1e5 * A)  # (what 32 bits do not see)
            elif mine > 0:
                to = c
                break
        if to is not None:
            target[at] = ids[to]
            at = to
            continue
        whole, run = sum(rest.values()), 0.0
        for k in sorted(rest):
            run += rest[k]
            margin = min(margin, 1e7 * abs(run / whole - u[0])) if rest[k] else margin
            if run > u[0] * whole:
                target[at] = k
                return target, margin
        return target, 0.0


@pytest.mark.parametrize("seqs,n,fan,support,vocab,dtype,draft,order", [
    (500, 2, 1, 2, 40, F16, BF16, "any"), (300, 5, 1, 3, 4100, F32, F16, "any"), (300, 4, 3, 3, 50, F32, None, "any"),
    (500, 3, 2, 2, 40, F16, BF16, "any"), (400, 5, 4, 2, 40, F16, BF16, "twice"), (200, 13, 3, 3, 300, F32, BF16, "any"),
    (100, 31, 5, 5, 9000, BF16, BF16, "any"), (60, 60, 6, 4, 900, F32, F16, "twice"), (10, 300, 6, 6, 2000, F16, BF16, "any"),
    (90, 13, 3, 3, 151936, F16, BF16, "any"), (90, 13, 6, 3, 151936, BF16, BF16, "twice"), (3, 200, 6, 6, 500009, F16, BF16, "any")])
def test_walks_by_the_rule(seqs, n, fan, support, vocab, dtype, draft, order):
    """Numbers near 1 and others: the walks are the rule's in 64 bits, but for sequences whose
    nearest decision is within 1e-5 of its border."""
    checked = scant = 0
    for seed in range(3):
        z, q, parent, ids, _, may = masked(seqs, n, fan, support, vocab, dtype, draft, 50 + seed, order)
        rng = random.Random(seed)
        u = [1 - 10 ** rng.uniform(-5, -1) if rng.random() < 0.8 else rng.random() for _ in range(seqs * n)]
        distinct = order == "any" and fan > 1
        target = torch.full((seqs * n,), 77, **I32)
        P.verify(P.Rows.of([n] * seqs, [0] * seqs, DEV), torch.tensor(parent, **I32), torch.tensor(ids, **I32), z,
                 torch.tensor(u, dtype=torch.float64, device=DEV), target, draft=q, distinct=distinct)
        got = target.tolist()
        cols = torch.tensor(may, device=DEV)
        ps = torch.softmax(z.gather(1, cols).double(), 1).tolist()
        qs = None if q is None else q.gather(1, cols).double().tolist()
        for s in range(seqs):
            at = slice(s * n, s * n + n)
            p_of = [dict(zip(m, x)) for m, x in zip(may[at], ps[at])]
            q_of = None if qs is None else [dict(zip(m, x)) for m, x in zip(may[at], qs[at])]
            want, margin = kept_walk(parent[at], ids[at], p_of, u[at], q_of, distinct)
            if margin > 1e-5:
                checked += 1
                assert got[at] == want, (seed, s)
            else:
                scant += 1
    assert checked > 5 * scant
