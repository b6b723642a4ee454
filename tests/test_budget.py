"""Sampled verification, weights of keys and eviction without a GPU: what the walk's
rule promises, and the refusals, which launch nothing."""
import ctypes
import random
import re

import pytest

torch = pytest.importorskip("torch")

from plugins_amd import exl3 as X  # noqa: E402
from plugins_amd import paged as P  # noqa: E402
from tests import _budget as B  # noqa: E402
from tests.test_paged import desc, step  # noqa: E402


@pytest.mark.parametrize("how", ["certain", "line", "siblings", "distinct"])
def test_the_walk_keeps_the_targets_distribution(how):
    """The token after the root, over many drafts and random numbers: as often as the
    target's probability says.  A share's standard deviation is at most
    sqrt(1/4 / 20000) = 0.0035; five of them (and five tokens) leave one run in a
    million."""
    rng, g = random.Random(how), torch.Generator().manual_seed(3)
    V, N = 5, 20000
    z, zq = torch.randn(1, V, generator=g) * 1.5, torch.randn(1, V, generator=g)
    p, q = B.probabilities(z[0], 0.8), B.probabilities(zq[0], 1.0)
    rows = {"certain": 4, "line": 2, "siblings": 4, "distinct": 4}[how]
    draft = None if how == "certain" else q.expand(rows, V)
    logits = z.expand(rows, V)
    seen = [0] * V
    for _ in range(N):
        if how == "certain":
            ids = [0, 3, 1, 3]
        elif how == "distinct":
            ids, left = [0], list(range(V))
            for _ in range(3):
                ids.append(rng.choices(left, [float(q[x]) for x in left])[0])
                left.remove(ids[-1])
        else:
            ids = [0] + rng.choices(range(V), q.tolist(), k=rows - 1)
        t, _ = B.walk([-1] + [0] * (rows - 1), ids, logits, 0.8, [rng.random() for _ in range(rows)],
                      draft, how == "distinct")
        seen[t[0]] += 1
    for v in range(V):
        assert abs(seen[v] / N - float(p[v])) < 5 * 0.0035, (how, v)


def entries(c, r, **kw):
    """The three entries on arguments that nothing reads; kw replaces some."""
    L = P.paged_lib()
    A = dict(parent=64, ids=64, vocab=100, logits=1 << 20, lt=X.DT_F16, ls=100, draft=1 << 21,
             dt=X.DT_F32, ds=100, distinct=0, temp=64, u=64, target=1 << 16, scratch=1 << 24, bytes=1 << 22,
             layer=0, heads=8, q=1 << 30, qs=1024, mask=64, words=1, scale=1.0, window=0, decay=1.0,
             base=64, score=1 << 31, room=64, seqs=2, len=64, keep=64, most=8, first=1, last=1,
             kept=1 << 32, new_score=1 << 33, new_len=128)
    A.update(kw)
    c, r = ctypes.byref(c), ctypes.byref(r)
    return {
        "verify": lambda: L.exl3p_verify(r, A["parent"], A["ids"], A["vocab"], A["logits"], A["lt"], A["ls"],
                                         A["draft"], A["dt"], A["ds"], A["distinct"], A["temp"], A["u"],
                                         A["target"], A["scratch"], A["bytes"], None),
        "weigh": lambda: L.exl3p_weigh(c, A["layer"], r, A["heads"], A["q"], A["qs"], A["mask"], A["words"],
                                       A["scale"], A["window"], A["decay"], A["base"], A["score"],
                                       A["room"], A["scratch"], A["bytes"], None),
        "evict": lambda: L.exl3p_evict(c, A["seqs"], A["len"], A["score"], A["room"], A["keep"], A["most"],
                                       A["first"], A["last"], A["kept"], A["new_score"], A["new_len"], None),
    }


V, W, E = ("verify",), ("weigh",), ("evict",)


@pytest.mark.parametrize("names,kw,why", [
    (V, dict(vocab=0), "PagedVerifyVocab"), (V, dict(vocab=-1), "PagedVerifyVocab"),
    (V, dict(vocab=(1 << 24) + 1, ls=1 << 30, ds=1 << 30), "2\\^24"),
    (V, dict(lt=X.DT_I32), "PagedVerifyDtype"), (V, dict(dt=X.DT_I32), "PagedVerifyDtype"),
    (V, dict(ls=99), "rows overlap"), (V, dict(ds=99), "rows overlap"),
    (V, dict(logits=(1 << 20) + 1), "Alignment"), (V, dict(draft=(1 << 21) + 2), "Alignment"),
    (V, dict(u=68), "Alignment"), (V, dict(logits=None), "missing"), (V, dict(ids=None), "missing"),
    (V, dict(u=None), "missing"), (V, dict(target=None), "missing"),
    (V + W, dict(scratch=None), "PagedScratch"), (V + W, dict(scratch=(1 << 24) + 4), "PagedScratch"),
    (V + W, dict(bytes=16), "PagedScratch"),
    (V, dict(target=64), "PagedOverlap"), (V, dict(target=(1 << 20) + 40), "PagedOverlap"),
    (V, dict(scratch=1 << 21), "PagedOverlap"), (V, dict(target=1 << 24), "PagedOverlap"),
    (W, dict(layer=2), "PagedLayer"), (W, dict(heads=7), "PagedHeads"),
    (W, dict(mask=None), "PagedMask"), (W, dict(scale=float("inf")), "PagedScale"),
    (W, dict(scale=float("nan")), "PagedScale"), (W, dict(scale=3e38), "PagedScale"),
    (W, dict(decay=float("nan")), "PagedDecay"), (W, dict(decay=float("-inf")), "PagedDecay"),
    (W, dict(window=-1), "PagedWindow"), (W, dict(q=(1 << 30) + 8), "PagedMatrixAlignment"),
    (W, dict(qs=1020), "PagedMatrixAlignment"), (W, dict(qs=512), "PagedMatrixStride"),
    (W, dict(q=None), "missing"), (W + E, dict(score=None), "missing"),
    (W + E, dict(score=(1 << 31) + 2), "PagedScore"), (W + E, dict(room=0), "PagedScore"),
    (W, dict(score=64), "PagedOverlap"), (W, dict(score=1 << 30), "PagedOverlap"),
    (W, dict(score=4096), "PagedOverlap"), (W, dict(scratch=1 << 30), "PagedOverlap"),
    (W, dict(score=1 << 24), "PagedOverlap"),
    (E, dict(seqs=4), "more sequences"), (E, dict(seqs=-1), "more sequences"), (E, dict(most=0), "PagedEvict"),
    (E, dict(first=-1), "PagedEvict"), (E, dict(last=-1), "PagedEvict"), (E, dict(len=None), "missing"),
    (E, dict(kept=None), "missing"), (E, dict(new_len=None), "missing"), (E, dict(new_score=None), "missing"),
    (E, dict(new_len=64), "PagedOverlap"), (E, dict(kept=64), "PagedOverlap"),
    (E, dict(kept=1 << 31), "PagedOverlap"), (E, dict(new_score=(1 << 31) + 4), "PagedOverlap"),
    (E, dict(new_score=1 << 32), "PagedOverlap"), (E, dict(new_score=4096), "PagedOverlap"),
    (E, dict(kept=4096), "PagedOverlap"), (E, dict(score=4096, new_score=4096), "PagedOverlap"),
    (E, dict(new_len=1 << 33), "PagedOverlap")])
def test_what_is_refused(names, kw, why):
    e = entries(desc(), step(), **kw)
    for name in names:
        v = e[name]()
        assert v.code != X.OK and re.search(why, v.reason), (name, v.reason)


def test_descriptors_that_are_refused():
    for name in ("weigh", "evict"):
        assert "another version" in entries(desc(size=8), step())[name]().reason
    for name in ("weigh", "verify"):
        for kw in (dict(size=1), dict(seqs=-1), dict(rows=-1), dict(max_rows=7), dict(cu=None), dict(seqs=65536)):
            assert entries(desc(seqs=1 << 20), step(**kw))[name]().code != X.OK, kw
    assert "1024 rows" in entries(desc(), step(rows=3000, max_rows=1025))["verify"]().reason
    L = P.paged_lib()
    assert L.exl3p_verify_scratch_bytes(ctypes.byref(step()), 0) == 0
    assert L.exl3p_weigh_scratch_bytes(ctypes.byref(desc()), ctypes.byref(step()), 8, -1, 64) == 0
    assert L.exl3p_weigh_scratch_bytes(ctypes.byref(desc()), ctypes.byref(step()), 8, 0, 0) == 0


def test_calls_too_large_for_a_launch():
    e = entries(desc(), step(rows=1 << 23, max_rows=4), vocab=1 << 20, ls=1 << 20, ds=1 << 20, bytes=1 << 60)
    v = e["verify"]()
    assert v.code == X.TOO_LARGE and "too many rows" in v.reason
    v = entries(desc(), step(rows=1 << 29, max_rows=1 << 29), words=1 << 23, bytes=1 << 60)["weigh"]()
    assert v.code == X.TOO_LARGE
    v = entries(desc(layers=32767, kv_heads=256, seqs=3), step(), seqs=3)["evict"]()
    assert v.code == X.TOO_LARGE


def test_nothing_to_do_launches_nothing():
    for kw in (dict(rows=0, max_rows=0), dict(seqs=0)):
        e = entries(desc(), step(**kw), target=None, score=None, scratch=None)
        assert e["verify"]().code == X.OK and e["weigh"]().code == X.OK
    assert entries(desc(), step(), seqs=0, kept=None)["evict"]().code == X.OK


def test_scratch_sizes_grow_with_what_they_hold():
    """A sampler's parts go by its rows and vocabulary; few pairs keep their scores
    (4 bytes a pair and key) until they would take over 2^30 bytes."""
    L = P.paged_lib()
    r = step(seqs=2, rows=6, max_rows=4)
    small, large = (L.exl3p_verify_scratch_bytes(ctypes.byref(r), v) for v in (1000, 151936))
    assert 0 < small < large < 1 << 20
    c = desc(seqs=64, kv_heads=8)
    one = step(seqs=64, rows=64, max_rows=1)
    size = lambda room: L.exl3p_weigh_scratch_bytes(  # noqa: E731
        ctypes.byref(c), ctypes.byref(one), 32, 0, room)
    assert size(8192) - size(16) == 64 * 8 * 4 * (8192 - 16) * 4
    assert size(1 << 20) < 1 << 24
