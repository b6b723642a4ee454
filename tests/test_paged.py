"""The paged KV cache without a GPU: the header's symbols, the book of pages
against a plain restatement, and the refusals, which launch nothing."""
import ctypes
import os
import random
import re

import pytest

from plugins_amd import exl3 as X
from plugins_amd import paged as P

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_paged_header_symbols_are_exported():
    text = open(os.path.join(ROOT, "include", "exl3_paged.h")).read()
    declared = set(re.findall(r"\b(exl3p_[a-z_0-9]+)\s*\(", text))
    L = X.lib()
    for name in sorted(declared):
        assert hasattr(L, name), name
    assert declared == set(P._SIGS), declared ^ set(P._SIGS)


# ------------------------------------------------------------------ the book

class PlainBook:
    """The book with lists of pages and a set of free ones."""

    def __init__(self, pages, page, seqs, max_pages):
        self.page, self.max_pages, self.free = page, max_pages, set(range(pages))
        self.has = [[] for _ in range(seqs)]

    def holders(self, p):
        return sum(p in h for h in self.has)

    def take(self):
        p = min(self.free)
        self.free.remove(p)
        return p

    def reserve(self, seq, start, stop):
        need, h = -(-stop // self.page), list(self.has[seq])
        if need > self.max_pages:
            return None
        first = start // self.page if stop > start else need
        redo = [i for i in range(first, min(need, len(h))) if self.holders(h[i]) > 1]
        if len(redo) + max(0, need - len(h)) > len(self.free):
            return None
        src, dst = [], []
        for i in redo:
            p = self.take()
            if i * self.page < start:
                src.append(h[i])
                dst.append(p)
            h[i] = p
        while len(h) < need:
            h.append(self.take())
        self.has[seq] = h
        return src, dst

    def fork(self, src, dst, keys):
        n = -(-keys // self.page)
        if src == dst or self.has[dst] or n > len(self.has[src]):
            return None
        self.has[dst] = self.has[src][:n]
        return True

    def trim(self, seq, keys):
        n = -(-keys // self.page)
        gone, self.has[seq] = self.has[seq][n:], self.has[seq][:n]
        self.free |= {p for p in gone if self.holders(p) == 0}


@pytest.mark.parametrize("seed", range(6))
def test_book_against_a_plain_one(seed):
    rng = random.Random(seed)
    pages, page, seqs, most = rng.randint(5, 40), rng.choice([16, 64]), rng.randint(2, 6), rng.randint(2, 12)
    a, b = P.Book(pages, page, seqs, most), PlainBook(pages, page, seqs, most)
    for _ in range(400):
        do, s = rng.choice(["reserve", "reserve", "fork", "trim", "compact"]), rng.randrange(seqs)
        if do == "reserve":
            stop = rng.randint(0, most * page + page)
            start = rng.randint(0, stop)
            want = b.reserve(s, start, stop)
            if want is None:
                with pytest.raises(X.Exl3Error) as e:
                    a.reserve(s, start, stop)
                assert e.value.code == X.TOO_LARGE
            else:
                assert a.reserve(s, start, stop) == want
        elif do == "fork":
            t, keys = rng.randrange(seqs), rng.randint(0, most * page)
            if b.fork(s, t, keys) is None:
                with pytest.raises(X.Exl3Error):
                    a.fork(s, t, keys)
            else:
                a.fork(s, t, keys)
        elif do == "trim":
            keys = rng.randint(0, most * page)
            a.trim(s, keys)
            b.trim(s, keys)
        elif rng.random() < 0.3:
            room = rng.choice([None, 0, 1, 3])
            src, dst = a.compact(room)
            assert not set(src) & set(dst) and len(set(dst)) == len(dst)
            used = sorted({p for h in b.has for p in h})
            if room is None:
                assert set(used) - set(src) | set(dst) == set(range(len(used)))
            to = dict(zip(src, dst))
            b.has = [[to.get(p, p) for p in h] for h in b.has]
            b.free = set(range(pages)) - {p for h in b.has for p in h}
        t = a.table()
        for s2, h in enumerate(b.has):
            assert t[s2].tolist() == h + [-1] * (most - len(h))
            assert a.held(s2) == len(h)
        assert a.free_pages() == len(b.free)
        for p in range(pages):
            assert a.shared(p) == b.holders(p)


def test_book_refuses():
    for bad in ((0, 16, 1, 1), (1, 15, 1, 1), (1, 8, 1, 1), (1, 512, 1, 1), (1, 48, 1, 1),
                (1, 16, 0, 1), (1, 16, 1, 0)):
        with pytest.raises(X.Exl3Error, match="PagedBookShape"):
            P.Book(*bad)
    with pytest.raises(X.Exl3Error) as e:
        P.Book(1 << 27, 16, 1, 1)
    assert e.value.code == X.TOO_LARGE
    b = P.Book(4, 16, 2, 3)
    for call in (lambda: b.reserve(2, 0, 1), lambda: b.reserve(-1, 0, 1), lambda: b.reserve(0, 5, 4),
                 lambda: b.reserve(0, -1, 4), lambda: b.fork(0, 0, 0), lambda: b.fork(0, 2, 0),
                 lambda: b.fork(0, 1, 1), lambda: b.fork(0, 1, -1), lambda: b.trim(2, 0),
                 lambda: b.trim(0, -1)):
        with pytest.raises(X.Exl3Error):
            call()
    assert b.free_pages() == 4 and b.held(5) == -1 and b.shared(4) == -1
    # no room for the pair: nothing happens
    b.reserve(0, 0, 20)
    b.fork(0, 1, 20)
    n = ctypes.c_int32(5)
    v = P.paged_lib().exl3p_book_reserve(b._b, 1, 20, 21, None, None, 0, ctypes.byref(n))
    assert v.code == X.TOO_LARGE and n.value == 0 and b.table().tolist() == [[0, 1, -1], [0, 1, -1]]


def test_a_rollback_after_a_fork():
    """A fork that goes back and writes again: only the pages of the keys that
    reserve names are its own; those held behind them stay the other sequence's
    too, until a reserve that covers them or a trim.  Header and mirror promise
    no more."""
    def forked():
        b = P.Book(16, 16, 2, 5)
        b.reserve(0, 0, 80)
        b.fork(0, 1, 80)
        return b

    b = forked()
    assert b.reserve(1, 5, 10) == ([0], [5])
    assert b.table().tolist() == [[0, 1, 2, 3, 4], [5, 1, 2, 3, 4]]
    assert [b.shared(p) for p in range(6)] == [1, 2, 2, 2, 2, 1] and b.held(1) == 5
    assert b.reserve(1, 10, 40) == ([], [])  # page 5 is its own already
    assert b.table()[1].tolist() == [5, 6, 7, 3, 4] and b.shared(3) == 2
    b = forked()
    b.trim(1, 5)
    assert b.reserve(1, 5, 10) == ([0], [5])
    assert b.held(1) == 1 and [b.shared(p) for p in range(5)] == [1] * 5
    # what is written about it
    text = " ".join(open(os.path.join(ROOT, "include", "exl3_paged.h")).read().split())
    assert "given up" not in text and "and those behind" not in P.PagedCache.reserve.__doc__
    assert all("shared" in d for d in (P.PagedCache.reserve.__doc__, P.Book.reserve.__doc__))


def test_the_table_keeps_its_book():
    """The view is of the book's memory: it lasts as long as any view does."""
    import gc
    import weakref
    b = P.Book(4, 16, 2, 3)
    b.reserve(0, 0, 20)
    t, ref = b.table()[:1], weakref.ref(b)
    del b
    gc.collect()
    assert ref() is not None and t.tolist() == [[0, 1, -1]]
    ref().reserve(0, 20, 40)
    assert t.tolist() == [[0, 1, 2]]
    del t
    gc.collect()
    assert ref() is None
    b = P.Book(4, 16, 2, 3)
    b.close()
    with pytest.raises(ValueError):
        b.table()


class HostCache(P.PagedCache):
    """A cache whose device is lists: pages of the text they hold, the table, and
    copies that fail when told to (some of a call's pairs done, as where one of
    its launches fails)."""

    def __init__(self, pages, seqs, monkeypatch):
        self.book, self.data, self.fail = P.Book(pages, 16, seqs, 6), [None] * pages, 0
        self.rows = self.book.table().tolist()
        monkeypatch.setattr(P, "copy_pages", self.copied)

    def copied(self, cache, src, dst, stream=None):
        assert cache is self and not set(src) & set(dst)
        for n, (a, b) in enumerate(zip(src, dst)):
            if self.fail and n >= len(src) // 2:
                raise RuntimeError("a launch failed")
            self.data[b] = self.data[a]

    def _sync(self, seq=None, stream=None):
        if self.fail == 2:
            raise RuntimeError("a copy failed")
        t = self.book.table().tolist()
        self.rows = t if seq is None else [t[s] if s == seq else r for s, r in enumerate(self.rows)]

    def text(self, seq):
        return [None if p < 0 else self.data[p] for p in self.rows[seq]]

    def write(self, seq, what):
        for p, w in zip(self.rows[seq], what):
            self.data[p] = w


@pytest.mark.parametrize("then", ["reserve", "fork", "trim", "compact"])
@pytest.mark.parametrize("first", ["reserve", "compact", "trim", "fork"])
def test_a_failed_copy_is_made_up_for(first, then, monkeypatch):
    """The book has changed when a copy to the device fails.  Until the copy is
    made the device keeps the table and pages of before; whatever is called next
    makes it first."""
    c = HostCache(12, 4, monkeypatch)
    c.reserve(3, 0, 32)
    c.reserve(0, 0, 40)
    c.write(0, "abc")
    c.fork(0, 1, 40)
    c.trim(3, 0)  # pages 0 and 1 are free
    before = [c.text(s) for s in range(4)]
    c.fail = 2
    with pytest.raises(RuntimeError):
        {"reserve": lambda: c.reserve(1, 36, 50), "compact": c.compact,
         "trim": lambda: c.trim(1, 0), "fork": lambda: c.fork(0, 2, 20)}[first]()
    assert [c.text(s) for s in range(4)] == before
    with pytest.raises(RuntimeError):  # and again: nothing more is given out
        c.reserve(3, 0, 90)
    assert [c.text(s) for s in range(4)] == before and c.book.held(3) == 0
    c.fail = 0
    {"reserve": lambda: c.reserve(3, 0, 16), "fork": lambda: c.fork(0, 3, 16),
     "trim": lambda: c.trim(3, 0), "compact": c.compact}[then]()
    assert c.rows == c.book.table().tolist()
    assert c.text(0)[:3] == list("abc")
    assert c.text(1)[:3] == ([None] * 3 if first == "trim" else list("abc"))
    assert c.text(2)[:2] == (list("ab") if first == "fork" else [None] * 2)


# ------------------------------------------------------------------- refusals

def desc(**kw):
    """A cache whose arrays are addresses that nothing reads."""
    f = dict(size=ctypes.sizeof(P.CacheDesc), dtype=X.DT_F16, k=4096, v=8192, layers=2, pages=8,
             kv_heads=2, page=16, dim=128, seqs=3, max_pages=4, table=64)
    f.update(kw)
    return P.CacheDesc(**f)


def step(**kw):
    f = dict(size=ctypes.sizeof(P.RowsDesc), seqs=2, rows=6, max_rows=4, cu=64, len=64)
    f.update(kw)
    return P.RowsDesc(**f)


def entries(c, r, **kw):
    """Every operator's entry on these, with arguments that nothing reads; kw
    replaces some of them."""
    L, A = P.paged_lib(), dict(parent=64, pos=64, slot=64, mask=64, words=1, layer=0, heads=8,
                               q=4096, qs=1024, kn=None, eps=1e-6, theta=1e4, out=4096, os=1024,
                               ks=256, scale=1.0, scratch=4096, bytes=1 << 40, ids=64, target=64,
                               path=64, most=4, count=64, new_len=128, src=(0,), dst=(1,), n=None,
                               rows=6)
    A.update(kw)
    c, r = ctypes.byref(c), ctypes.byref(r)
    arr = lambda x: (ctypes.c_int32 * max(1, len(x)))(*x)  # noqa: E731
    return {
        "plan": lambda: L.exl3p_tree_plan(c, r, A["parent"], A["pos"], A["slot"], A["mask"],
                                          A["words"], None),
        "append": lambda: L.exl3p_qkv_append(c, A["layer"], A["rows"], A["heads"], A["q"], A["qs"],
                                             A["q"], A["ks"], A["q"], A["ks"], None, A["kn"],
                                             A["pos"], A["slot"], A["out"], A["os"], A["eps"],
                                             A["theta"], None),
        "attend": lambda: L.exl3p_attend(c, A["layer"], r, A["heads"], A["q"], A["qs"], A["mask"],
                                         A["words"], A["scale"], A["out"], A["os"], A["scratch"],
                                         A["bytes"], None),
        "commit": lambda: L.exl3p_commit(c, r, A["parent"], A["ids"], A["target"], A["path"],
                                         A["most"], A["count"], A["count"], A["new_len"], None),
        "copy": lambda: L.exl3p_copy_pages(c, arr(A["src"]), arr(A["dst"]),
                                           len(A["src"]) if A["n"] is None else A["n"], None),
    }


@pytest.mark.parametrize("kw,why", [
    (dict(size=8), "another version"), (dict(dtype=X.DT_F32), "PagedCacheDtype"),
    (dict(k=None), "missing"), (dict(v=None), "missing"), (dict(table=None), "missing"),
    (dict(k=4100), "Alignment"), (dict(dim=96), "PagedCacheDim"), (dict(dim=256), "PagedCacheDim"),
    (dict(page=8), "PagedCachePage"), (dict(page=48), "PagedCachePage"),
    (dict(page=512), "PagedCachePage"), (dict(pages=0), "PagedCacheShape"),
    (dict(layers=-1), "PagedCacheShape"), (dict(pages=1 << 27), "2\\^31"),
    (dict(max_pages=(1 << 26) + 1), "2\\^30"), (dict(kv_heads=65536), "65535")])
def test_caches_that_are_refused(kw, why):
    for name, call in entries(desc(**kw), step()).items():
        v = call()
        assert v.code != X.OK and re.search(why, v.reason), (name, v)
    assert P.paged_lib().exl3p_attend_scratch_bytes(ctypes.byref(desc(**kw)), ctypes.byref(step()), 8) == 0


@pytest.mark.parametrize("kw,why", [
    (dict(size=1), "another version"), (dict(seqs=-1), "PagedRows"), (dict(seqs=65536), "65535"), (dict(seqs=4), "more sequences"),
    (dict(rows=-1), "PagedRows"), (dict(max_rows=7), "PagedRows"), (dict(max_rows=-1), "PagedRows"),
    (dict(cu=None), "missing"), (dict(len=None), "missing")])
def test_rows_that_are_refused(kw, why):
    e = entries(desc(), step(**kw))
    for name in ("plan", "attend", "commit"):
        v = e[name]()
        assert v.code != X.OK and re.search(why, v.reason), (name, v)


@pytest.mark.parametrize("names,kw,why", [
    (("plan", "attend"), dict(mask=None), "PagedMask"), (("plan", "attend"), dict(words=0), "PagedMask"),
    (("plan", "attend"), dict(words=-1), "PagedMask"),
    (("plan", "append"), dict(pos=None), "missing"), (("plan", "append"), dict(slot=None), "missing"),
    (("append", "attend"), dict(layer=2), "PagedLayer"), (("append", "attend"), dict(layer=-1), "PagedLayer"),
    (("append", "attend"), dict(heads=7), "PagedHeads"), (("append", "attend"), dict(heads=0), "PagedHeads"),
    (("append", "attend"), dict(q=None), "missing"), (("append", "attend"), dict(q=4104), "Alignment"),
    (("append", "attend"), dict(qs=1020), "Alignment"), (("append", "attend"), dict(qs=1016), "overlap"),
    (("append", "attend"), dict(out=None), "missing"), (("append", "attend"), dict(os=512), "overlap"),
    (("append",), dict(ks=128), "overlap"), (("append",), dict(theta=0.0), "PagedTheta"),
    (("append",), dict(theta=float("nan")), "PagedTheta"),
    (("append",), dict(theta=float("inf")), "PagedTheta"),
    (("append",), dict(kn=68), "Alignment"), (("append",), dict(rows=-1), "PagedRows"),
    (("attend",), dict(scratch=None), "PagedScratch"), (("attend",), dict(scratch=4100), "PagedScratch"),
    (("attend",), dict(bytes=100), "PagedScratch"),
    (("attend",), dict(scale=float("nan")), "PagedScale"),
    (("attend",), dict(scale=float("-inf")), "PagedScale"),
    (("commit",), dict(most=0), "PagedPath"), (("commit",), dict(path=None), "missing"),
    (("commit",), dict(ids=None), "missing"), (("commit",), dict(target=None), "missing"),
    (("commit",), dict(new_len=64), "over len"), (("commit",), dict(count=None), "missing"),
    (("copy",), dict(n=-1), "below 0"), (("copy",), dict(src=(8,)), "outside"),
    (("copy",), dict(dst=(-1,)), "outside"), (("copy",), dict(src=(0, 1), dst=(2, 2)), "twice"),
    (("copy",), dict(src=(0, 1), dst=(1, 2)), "both"), (("copy",), dict(src=(3,), dst=(3,)), "both"),
    (("copy",), dict(src=tuple([0] * 9), dst=tuple(range(9))), "twice")])
def test_calls_that_are_refused(names, kw, why):
    e = entries(desc(), step(), **kw)
    for name in names:
        v = e[name]()
        assert v.code != X.OK and re.search(why, v.reason), (name, v)


def test_masks_and_trees_too_large_are_refused():
    big = step(rows=5000, max_rows=1025)
    e = entries(desc(), big, words=17)
    assert "1024" in e["plan"]().reason and "1024" in e["commit"]().reason
    for name in ("plan", "attend"):
        assert "PagedMask" in entries(desc(), big, words=16)[name]().reason


def test_nothing_to_do_is_no_refusal():
    """No rows, no sequences, no pages: accepted before any launch."""
    none = step(rows=0, max_rows=0)
    e = entries(desc(), none, words=0, mask=None, rows=0, src=(), dst=())
    for name in ("plan", "append", "attend", "copy"):
        assert e[name]().code == X.OK, name
    e = entries(desc(), step(seqs=0), words=1)
    assert e["attend"]().code == X.OK and e["commit"]().code == X.OK


@pytest.mark.parametrize("kw", [
    dict(count=2 << 20), dict(count=(2 << 20) + 20), dict(count=3 << 20), dict(new_len=(1 << 20) + 4),
    dict(new_len=64 + 8), dict(path=(4 << 20) - 4), dict(path=(4 << 20) + 20), dict(path=64 + 4)])
def test_commit_refuses_outputs_over_inputs(kw):
    """Several workgroups read a sequence's tree: `next` in place of ids, say,
    would change it under them."""
    far = dict(parent=1 << 20, ids=2 << 20, target=3 << 20, path=5 << 20, count=6 << 20,
               new_len=7 << 20)
    if kw.get("path", 0) >> 20:
        far["parent"] = 4 << 20
    far.update(kw)
    v = entries(desc(), step(len=64 + 12), **far)["commit"]()
    assert v.code == X.UNSUPPORTED and "over an input" in v.reason, v


def test_calls_past_a_grid_are_refused():
    """A launch counts threads in 32 bits: 2^24 workgroups of 256 are too many."""
    e = entries(desc(), step(rows=(1 << 30) + 1, max_rows=0), rows=1 << 24)
    for name, why in (("append", "2\\^24"), ("plan", "2\\^30"), ("attend", "2\\^30"),
                      ("commit", "2\\^30")):
        v = e[name]()
        assert v.code == X.TOO_LARGE and re.search(why, v.reason), (name, v)
    many = desc(kv_heads=65535, seqs=4)
    for r in (step(rows=4096, max_rows=4), step(rows=32768, max_rows=256)):
        e = entries(many, r, heads=65535, qs=65535 * 128, os=65535 * 128, words=4)
        v = e["attend"]()
        assert v.code == X.TOO_LARGE and "too many rows and heads" in v.reason, v


def test_scales_past_32_bits_are_refused():
    for scale in (3e38, -3e38):
        assert "PagedScale" in entries(desc(), step(), scale=scale)["attend"]().reason


@pytest.mark.parametrize("eps", [-1e-6, float("nan"), float("inf"), float("-inf")])
def test_a_norm_refuses_an_eps_that_is_none(eps):
    """Roots of numbers below 0, or of none."""
    v = entries(desc(), step(), eps=eps, kn=64, q=1 << 24, out=1 << 25)["append"]()
    assert v.code == X.UNSUPPORTED and "PagedEps" in v.reason, v


def test_operators_take_no_number_for_another():
    """Layer 2^32 is not layer 0, 2^32 + 1 rows are not one."""
    import types
    torch = pytest.importorskip("torch")
    P._t()
    i = torch.zeros(2, dtype=torch.int32)
    for rows, most in ((1 << 32, 1), (1, (1 << 32) + 1), (-(1 << 32), 0)):
        with pytest.raises(OverflowError):
            P.Rows(i, i[:1], rows, most)
    c = types.SimpleNamespace(index=-1, device="cpu", dtype=torch.float16, head_dim=64, kv_heads=1,
                              _ref=None)
    r = types.SimpleNamespace(rows=2, max_rows=2, seqs=1, index=-1, _ref=None)
    x, b = torch.zeros(2, 64, dtype=torch.float16), torch.zeros(64, dtype=torch.uint8)
    for layer in (1 << 32, 1 << 31, -(1 << 32) - 1):
        with pytest.raises(OverflowError):
            P.qkv_append(c, layer, x, x, x, None, None, i, i, x)
        with pytest.raises(OverflowError):
            P.attend(c, layer, r, x, x, scratch=b)


# ------------------------------------------------- memory that two tensors share

def bytes_of(base, rows, width, stride):
    """The bytes of a matrix, in units of 16 (all sizes here are multiples)."""
    return {(base + r * stride + x) // 16 for r in range(rows) for x in range(0, width, 16)}


def append_on(rows, heads, kv, q, qs, k, ks, v, vs, out, os_, **kw):
    """The append of matrices at these addresses (strides in elements) of a cache
    far from them.  Its eps is refused last, so nothing is ever launched."""
    a = dict(rows=rows, layer=0, pos=1 << 40, slot=1 << 41, kn=1 << 42, qn=None, eps=-1.0)
    a.update(kw)
    c = ctypes.byref(desc(kv_heads=kv, dim=64, k=1 << 43, v=1 << 44))
    return P.paged_lib().exl3p_qkv_append(c, a["layer"], rows, heads, q, qs, k, ks, v, vs, a["qn"],
                                          a["kn"], a["pos"], a["slot"], out, os_, a["eps"], 1e4, None)


@pytest.mark.parametrize("seed", range(8))
def test_append_refuses_what_lies_over_its_output(seed):
    """Random matrices in a small space, slices of common rows and others: refused
    just where q_out shares a byte with k, v or, unless it is q itself, q."""
    rng = random.Random(seed)
    seen = {True: 0, False: 0}
    for _ in range(1500):
        rows, kv, group = rng.choice([1, 1, 2, 3, 5, 9]), rng.choice([1, 2]), rng.choice([1, 2])
        wide = {"q": 64 * kv * group, "k": 64 * kv, "v": 64 * kv, "out": 64 * kv * group}
        common = rng.choice([256, 384, 512, 640, 1024])
        at = {}
        for x, w in wide.items():
            stride = max(w, common if rng.random() < 0.7 else w + 8 * rng.randint(0, 40))
            at[x] = (1 << 20) + 16 * rng.randint(0, rng.choice([100, 2000])), stride
        if rng.random() < 0.3:
            at["out"] = at["q"]
        mem = {x: bytes_of(b, rows, 2 * wide[x], 2 * s) for x, (b, s) in at.items()}
        same = at["out"][0] == at["q"][0] and (at["out"][1] == at["q"][1] or rows == 1)
        want = bool(mem["out"] & (mem["k"] | mem["v"] | (set() if same else mem["q"])))
        seen[want] += 1
        v = append_on(rows, kv * group, kv, *at["q"], *at["k"], *at["v"], *at["out"])
        assert v.code == X.UNSUPPORTED
        assert ("PagedOverlap" if want else "PagedEps") in v.reason, (rows, at, v)
    assert min(seen.values()) > 100


@pytest.mark.parametrize("kw", [
    dict(pos=1 << 20), dict(pos=(1 << 20) + 3 * 2048 + 1024 - 4), dict(slot=(1 << 20) + 64),
    dict(kn=(1 << 20) + 8), dict(qn=(1 << 20) + 1024 * 2 + 8), dict(pos=(1 << 43) + 8),
    dict(slot=(1 << 44) - 4), dict(qn=1 << 43), dict(q=1 << 43), dict(k=(1 << 44) + 4096),
    dict(v=(1 << 43) - 16), dict(out=(1 << 44) + 16), dict(v=(1 << 44) + 8 * 2 * 16 * 64 * 2 - 16)])
def test_append_refuses_what_lies_over_its_other_memory(kw):
    """Positions, slots and weights under q_out; anything under the pages that the
    layer's keys and values go to."""
    a = dict(q=1 << 30, k=1 << 31, v=1 << 32, out=1 << 20)
    args = dict(rows=4, heads=8, kv=2, qs=1024, ks=256, vs=256, os_=1024)
    assert "PagedEps" in append_on(**a, **args).reason
    for x in a:
        if x in kw:
            a[x] = kw.pop(x)
    v = append_on(**a, **args, **kw)
    assert v.code == X.UNSUPPORTED and "PagedOverlap" in v.reason, v


def test_append_refuses_keys_over_values():
    for v in (1 << 30, (1 << 30) + 8 * 2 * 16 * 64 * 2 - 16):  # the layer's last bytes
        c = ctypes.byref(desc(dim=64, k=1 << 30, v=v))
        v = P.paged_lib().exl3p_qkv_append(c, 0, 4, 8, 1 << 20, 512, 1 << 21, 256, 1 << 22, 256, None,
                                           None, 64, 1 << 19, 1 << 23, 512, 0.0, 1e4, None)
        assert v.code == X.UNSUPPORTED and "keys over values" in v.reason, v


@pytest.mark.parametrize("kw", [
    dict(pos=1 << 20), dict(slot=(1 << 20) + 20), dict(mask=(1 << 20) - 40), dict(pos=(1 << 21) + 8),
    dict(slot=(1 << 22) - 20), dict(mask=(1 << 22) - 40), dict(pos=(1 << 23) + 3 * 4 * 4 - 4),
    dict(mask=1 << 23), dict(slot=1 << 24), dict(mask=(1 << 24) + 16), dict(mask=(1 << 25) + 16)])
def test_plan_refuses_outputs_over_anything(kw):
    """One workgroup's positions or slots over another's tree, lengths or pages."""
    a = dict(parent=1 << 20, pos=1 << 24, slot=1 << 25, mask=1 << 26)
    a.update(kw)
    v = entries(desc(table=1 << 23), step(cu=1 << 21, len=1 << 22), **a)["plan"]()
    assert v.code == X.UNSUPPORTED and "PagedOverlap" in v.reason, v


def commit_on(c, r, **kw):
    a = dict(parent=1 << 20, ids=2 << 20, target=3 << 20, path=4 << 20, count=5 << 20, next=6 << 20,
             new_len=7 << 20)
    a.update(kw)
    return P.paged_lib().exl3p_commit(ctypes.byref(c), ctypes.byref(r), a["parent"], a["ids"],
                                      a["target"], a["path"], 4, a["count"], a["next"], a["new_len"],
                                      None)


@pytest.mark.parametrize("kw", [
    dict(next=5 << 20), dict(next=(5 << 20) + 4), dict(count=(4 << 20) + 2 * 4 * 4 - 4),
    dict(new_len=(4 << 20) - 4), dict(new_len=6 << 20), dict(path=(9 << 20) + 8), dict(count=9 << 20),
    dict(next=(9 << 20) + 3 * 4 * 4 - 4), dict(new_len=(9 << 20) - 4), dict(path=1 << 30),
    dict(count=(1 << 31) + 4096), dict(next=(1 << 30) - 4), dict(ids=1 << 30), dict(target=1 << 31)])
def test_commit_refuses_outputs_over_outputs_table_and_cache(kw):
    """`next` in place of count, an output in the table that other workgroups look
    pages up in, anything in the memory that the rows move in."""
    c = desc(table=9 << 20, k=1 << 30, v=1 << 31)
    v = commit_on(c, step(cu=10 << 20, len=11 << 20), **kw)
    assert v.code == X.UNSUPPORTED and "PagedOverlap" in v.reason, v


def test_commit_refuses_keys_over_values():
    c = desc(table=9 << 20, k=1 << 30, v=(1 << 30) + 2 * 8 * 2 * 16 * 128 * 2 - 16)
    v = commit_on(c, step(cu=10 << 20, len=11 << 20))
    assert v.code == X.UNSUPPORTED and "PagedOverlap" in v.reason, v


@pytest.mark.parametrize("kw", [
    dict(out=(1 << 20) + 16), dict(out=(1 << 20) + 1024), dict(os=1032), dict(out=(1 << 20) - 5 * 2048 - 16),
    dict(out=(1 << 24) + 2048), dict(out=(1 << 25) - 16), dict(out=1 << 27), dict(out=(1 << 28) - 64),
    dict(out=1 << 29), dict(out=1 << 30), dict(out=(1 << 31) + 8 * 2 * 16 * 128 * 2 - 16),
    dict(scratch=1 << 20), dict(scratch=(1 << 20) + 5 * 2048), dict(scratch=1 << 27),
    dict(scratch=(1 << 28)), dict(scratch=1 << 29), dict(scratch=1 << 26), dict(scratch=1 << 30),
    dict(scratch=(1 << 31) + 4096)])
def test_attend_refuses_outputs_over_anything(kw):
    """An output over q at another place or stride than q's own, output or scratch
    over masks, lengths, table or the layer's pages, or over each other."""
    c = desc(table=1 << 29, k=1 << 30, v=1 << 31)
    r = step(cu=1 << 27, len=1 << 28)
    need = P.paged_lib().exl3p_attend_scratch_bytes(ctypes.byref(c), ctypes.byref(r), 8)
    a = dict(q=1 << 20, out=1 << 20, qs=1024, os=1024, mask=1 << 26, words=1, scratch=(1 << 25) - need,
             bytes=need)
    a["scratch"] &= ~15
    if kw.get("out") == (1 << 24) + 2048:
        a["mask"] = 1 << 24 | 4096
    a.update(kw)
    v = entries(c, r, **a)["attend"]()
    assert v.code == X.UNSUPPORTED and "PagedOverlap" in v.reason, v


def test_a_step_without_sequences_needs_no_lengths():
    e = entries(desc(), step(seqs=0, rows=0, max_rows=0, len=None), words=0, mask=None)
    for name in ("plan", "attend", "commit"):
        assert e[name]().code == X.OK, name


def test_the_book_takes_no_number_for_another():
    b = P.Book(4, 16, 2, 3)
    for call in (lambda: P.Book(1 << 32, 16, 1, 1), lambda: b.reserve(0, 0, (1 << 32) + 16),
                 lambda: b.reserve(1 << 32, 0, 16), lambda: b.fork(0, (1 << 32) + 1, 0),
                 lambda: b.trim(0, 1 << 32), lambda: b.trim(1 << 32, 0)):
        with pytest.raises(OverflowError):
            call()
    assert b.free_pages() == 4 and b.held(0) == 0


# ------------------------------------------------- the decoder over the cache

def decoder_without_a_gpu():
    """A PagedDecoder that has nothing to launch with: what forward refuses, it
    refuses before that."""
    import types
    torch = pytest.importorskip("torch")
    from plugins_amd import qwen3 as Q
    P._t()
    d = Q.PagedDecoder.__new__(Q.PagedDecoder)
    d.P, d.torch, d.cfg, d.m = P, torch, Q.Qwen3Config(layers=0, vocab=16), None
    d.cache = types.SimpleNamespace(index=-1, device="cpu", dtype=torch.float16)
    return torch, d, types.SimpleNamespace(rows=4, seqs=1, max_rows=4, index=-1, device="cpu")


@pytest.mark.parametrize("make,why", [
    (lambda t: t.zeros(4, dtype=t.int64), TypeError), (lambda t: t.zeros(3, dtype=t.int32), ValueError),
    (lambda t: t.zeros(5, dtype=t.int32), ValueError),
    (lambda t: t.zeros(8, dtype=t.int32)[::2], ValueError)])
def test_decoder_refuses_ids_that_are_not_one_a_row(make, why):
    """The embedding reads `rows` 32-bit numbers from wherever ids begins: 64-bit
    ones would be other tokens, fewer a read behind them."""
    torch, d, rows = decoder_without_a_gpu()
    for call in (d.forward, d.verify):
        with pytest.raises(why, match="ids"):
            call(rows, make(torch))


def test_streams_of_other_devices_are_refused():
    """A launch goes to the cache's device: another one's stream is none of its."""
    import types
    torch, d, rows = decoder_without_a_gpu()
    other = types.SimpleNamespace(cuda_stream=5, device_index=1)
    ids = torch.zeros(4, dtype=torch.int32)
    x = torch.zeros(4, 64, dtype=torch.float16)
    c = d.cache
    c.head_dim, c.kv_heads, c._ref, rows._ref = 64, 1, None, None
    calls = (lambda s: P.plan(c, rows, stream=s), lambda s: P.copy_pages(c, [0], [1], stream=s),
             lambda s: P.attend(c, 0, rows, x, x, scratch=x, stream=s),
             lambda s: P.tree_plan(c, rows, None, ids, ids, stream=s),
             lambda s: P.qkv_append(c, 0, x, x, x, None, None, ids, ids, x, stream=s),
             lambda s: P.commit(c, rows, None, ids, ids, ids[:1][None], ids[:1], ids[:1], ids[:1],
                                stream=s),
             lambda s: d.forward(rows, ids, stream=s), lambda s: d.verify(rows, ids, stream=s))
    for call in calls:
        with pytest.raises(ValueError, match="the stream is on device 1"):
            call(other)
    # one that says nothing but its handle is taken for the cache's
    assert P._stream(c, types.SimpleNamespace(cuda_stream=7)) == 7


def test_decoder_runs_on_its_caches_device(monkeypatch):
    """With another device current, the whole step is done under the cache's: the
    linears and norms go by the current one."""
    torch, d, rows = decoder_without_a_gpu()
    now = [1]

    class guard:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            now.append(self.index)

        def __exit__(self, *e):
            now.pop()

    def plan(*a):
        raise StopIteration(now[-1])

    monkeypatch.setattr(P, "_device", lambda: now[-1])
    monkeypatch.setattr(P, "plan", plan)
    monkeypatch.setattr(torch.cuda, "device", guard)
    for call in (d.forward, d.verify):
        with pytest.raises(StopIteration) as e:
            call(rows, torch.zeros(4, dtype=torch.int32))
        assert e.value.value == d.cache.index and now == [1]
