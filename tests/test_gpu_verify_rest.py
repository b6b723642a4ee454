"""What is left of the target's probabilities where a walk of sampled verification ends:
draft rows that the rule does not use, on every path that verify takes (few rows in one
launch, rounds, the lone workgroup, statistics as the walks go)."""
import math
import random

import pytest

torch = pytest.importorskip("torch")

from plugins_amd import paged as P  # noqa: E402
from tests import _budget as B  # noqa: E402
from tests.test_gpu_budget import MARGIN  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
I32 = {"dtype": torch.int32, "device": DEV}


class OnHost:
    """Rows of a tensor on the device, each brought to the host when it is looked at."""

    def __init__(self, t):
        self.t, self.shape = t, t.shape

    def __getitem__(self, i):
        return OnHost(self.t[i]) if isinstance(i, slice) else self.t[i].cpu()


def trees(counts, fan, rng):
    """Parents of rows (fan 0: lines); a row has about `fan` children."""
    out = []
    for n in counts:
        out += [-1][:n] + [i - 1 if fan == 0 else min(i - 1, rng.randint(0, i // fan)) for i in range(1, n)]
    return out


def leaves(counts, parent):
    """The step's rows that no row follows."""
    at, out = 0, []
    for n in counts:
        out += [at + i for i in range(n) if i not in parent[at:at + n]]
        at += n
    return out


def drawn(counts, vocab, dtype, draft, distinct, fan, seed, high):
    """A step on the device: logits with 12 likely tokens a row, a draft near them, drafted
    tokens among them; of the numbers a share `high` refuses most of what it can."""
    g, rng = torch.Generator(device=DEV).manual_seed(seed), random.Random(seed)
    T, k = sum(counts), 12
    parent = trees(counts, fan, rng)
    z = torch.randn(T, vocab, generator=g, device=DEV)
    likely = torch.randint(0, vocab - k, (T, 1), generator=g, device=DEV) + torch.arange(k, device=DEV)
    z.scatter_(1, likely, 12 + 3 * torch.rand(T, k, generator=g, device=DEV))
    z = z.to(dtype)
    q = torch.empty(T, vocab, dtype=draft, device=DEV)
    for i in range(0, T, 64):
        x = z[i:i + 64].float()
        q[i:i + 64] = torch.softmax(x + torch.randn(x.shape, generator=g, device=DEV), -1).to(draft)
    first, ids, taken, at = likely[:, 0].tolist(), [], {}, 0
    for n in counts:
        for i in range(n):
            up = at + max(0, parent[at + i])
            j = taken[up] = taken.get(up, -1) + 1
            ids.append(first[up] + (j if distinct else rng.choice([0, j % k, j % k])))
        at += n
    u = torch.tensor([rng.uniform(0.9, 1.0) if rng.random() < high else rng.random() for _ in range(T)],
                     dtype=torch.float64)
    heats = [(1.0, 0.8, 1.3)[s % 3] for s in range(len(counts))]
    return z, q, parent, ids, heats, u


def wanted(counts, z, q, parent, ids, heats, u, distinct):
    """(targets, margin, most needs of a walk: rows got to and refusals with siblings left)"""
    want, margin, needs, at = [], math.inf, 0, 0
    for s, n in enumerate(counts):
        own, tok = parent[at:at + n], ids[at:at + n]
        t, m = B.walk(own, tok, OnHost(z)[at:at + n], float(torch.tensor(heats[s], dtype=F32)),
                      u[at:at + n].tolist(), OnHost(q)[at:at + n], distinct)
        had = 0
        for i in (i for i in range(n) if t[i] >= 0):
            under = [c for c in range(n) if own[c] == i]
            hit = [j for j, c in enumerate(under) if t[c] >= 0 and tok[c] == t[i]]
            had += 1 + (hit[0] if hit else max(0, len(under) - 1))
        want, margin, needs = want + t, min(margin, m), max(needs, had)
        at += n
    return want, margin, needs


def verified(counts, z, q, parent, ids, heats, u, distinct):
    target = torch.full((sum(counts),), 77, **I32)
    P.verify(P.Rows.of(counts, [0] * len(counts), DEV), None if parent is None else torch.tensor(parent, **I32),
             torch.tensor(ids, **I32), z, u.to(DEV), target, draft=q,
             temperature=torch.tensor(heats, dtype=F32, device=DEV), distinct=distinct)
    return target.tolist()


def settled(counts, vocab, dtype, draft, distinct, fan, high, least=0):
    for seed in range(7, 200):  # one whose decisions are not at a border, by the formula alone
        args = drawn(counts, vocab, dtype, draft, distinct, fan, seed, high)
        want, margin, needs = wanted(counts, *args, distinct)
        if margin > MARGIN and needs >= least and any(want[t] >= 0 for t in leaves(counts, args[2])):
            return args, want
    raise AssertionError("no such step")


@pytest.mark.parametrize("what", [math.nan, math.inf])
@pytest.mark.parametrize("counts,vocab,fan,distinct,dtype,draft", [
    ([4, 1, 3, 0, 5], 4099, 0, False, F16, F32), ([4, 1, 3], 20011, 0, False, F32, BF16),
    ([2, 1, 2], 8191, 1, True, BF16, F16),                           # one launch
    ([3, 6, 1, 4], 8200, 2, True, F16, F16), ([7, 5], 151936, 2, False, BF16, F32),  # rounds
    ([60, 1, 40], 5003, 1, True, F16, BF16), ([200, 30], 4099, 2, False, F32, F32),  # the lone workgroup
    ([16] * 60, 151936, 1, True, F16, BF16), ([140, 0, 20], 900007, 3, False, BF16, F16)])  # as the walks go
def test_draft_rows_behind_leaves_are_not_read(counts, vocab, fan, distinct, dtype, draft, what):
    """Half of each leaf's draft row is NaN or infinite, as memory that nobody filled may
    be: no token of a leaf was refused, so the target's own probabilities stand."""
    args, want = settled(counts, vocab, dtype, draft, distinct, fan, 0.0)
    z, q, parent, ids, heats, u = args
    q[leaves(counts, parent), ::2] = what
    assert verified(counts, *args, distinct) == want
    if fan == 0:
        assert verified(counts, z, q, None, ids, heats, u, distinct) == want


@pytest.mark.parametrize("counts,vocab,fan,distinct,dtype,draft,needs", [
    ([16] * 64, 151936, 4, False, BF16, BF16, 6), ([16] * 64, 151936, 6, True, F16, F32, 6),
    ([300, 0, 150], 400011, 6, True, F16, F16, 7), ([300, 0, 150], 400011, 4, False, BF16, F32, 7),
    ([40, 9], 3000017, 5, False, F16, BF16, 6), ([64, 20], 1000003, 6, True, F32, F16, 6)])
def test_walks_that_read_as_they_go_and_are_refused(counts, vocab, fan, distinct, dtype, draft, needs):
    """Drawn siblings in more than 268 MB of logits: rows' statistics are formed when a walk
    gets there, and refusals beyond the launched rounds are the lone workgroup's."""
    assert sum(counts) * vocab * (4 if dtype is F32 else 2) > 8 << 25
    args, want = settled(counts, vocab, dtype, draft, distinct, fan, 0.8, needs)
    assert verified(counts, *args, distinct) == want

