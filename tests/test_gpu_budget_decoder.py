"""A decoder that samples what it verifies, keeps the weights of its cached keys and
evicts the lightest: prompts, trees, forks and evictions together, against the
formulas in 64 bits and against itself taken token by token."""
import math

import pytest

torch = pytest.importorskip("torch")

from plugins_amd import paged as P  # noqa: E402
from plugins_amd import qwen3 as Q  # noqa: E402
from tests import _budget as B  # noqa: E402
from tests.test_gpu_budget import MARGIN  # noqa: E402
from tests.test_gpu_paged_decoder import CFG, DEV, model, rel, tokens  # noqa: E402,F401

pytestmark = pytest.mark.gpu
I32 = {"dtype": torch.int32, "device": DEV}


def decoder(model, window=0, decay=1.0, seqs=3, pages=40, max_pages=12, page=16):  # noqa: F811
    return Q.PagedDecoder(model, seqs, pages, max_pages, page, window, decay)


@pytest.fixture
def weighs(monkeypatch):
    """What each call of weigh had and gave, on the host."""
    calls, own = [], P.weigh

    def weigh(cache, layer, rows, q, score, mask=None, scale=None, window=0, decay=1.0, **kw):
        call = {"layer": layer, "cu": rows.cu.tolist(), "lens": rows.len.tolist(), "q": q.cpu(), "mask": mask,
                "had": score.cpu(), "table": cache.table[:rows.seqs].cpu(), "k": cache.k.cpu(),
                "window": window, "decay": decay}
        own(cache, layer, rows, q, score, mask, scale, window, decay, **kw)
        call["got"] = score.cpu()
        calls.append(call)

    monkeypatch.setattr(P, "weigh", weigh)
    return calls


def check_weighs(calls):
    for c in calls:
        assert c["mask"] is None
        counts = [b - a for a, b in zip(c["cu"], c["cu"][1:])]
        q = c["q"].view(len(c["q"]), CFG.heads, -1)
        want, tol = B.weights(q, c["k"], c["table"], c["cu"], c["lens"],
                              [[list(range(i + 1)) for i in range(n)] for n in counts], 16,
                              CFG.heads // CFG.kv_heads, 1 / math.sqrt(q.shape[2]), c["had"], c["decay"],
                              c["window"], layer=c["layer"])
        assert ((c["got"].double() - want).abs() <= tol).all()


def tree_of(first, certain, decoys):
    """A root, and for each certain token a row behind a decoy, siblings."""
    ids, parent, at = [first], [-1], 0
    for c, d in zip(certain, decoys):
        ids += [d, c]
        parent += [at, at]
        at = len(ids) - 1
    return torch.tensor(ids, **I32), torch.tensor(parent, **I32)


@pytest.mark.parametrize("window,decay", [(0, 1.0), (4, 0.5)])
def test_weights_of_prompts_tokens_and_accepted_rows(model, weighs, window, decay):  # noqa: F811
    """Each pass's weights are the formula's; a verified tree leaves those of its accepted
    rows alone, as the same tokens in a line leave (f16 roundings in other places)."""
    d, line = decoder(model, window, decay), decoder(model, window, decay)
    ids = tokens(29, 1)
    for x in (d, line):
        x.cache.reserve(0, 0, 29)
        x.forward(P.Rows.of([29], [0], DEV), ids)
    text = tokens(4, 2)
    line.cache.reserve(0, 29, 33)
    line.forward(P.Rows.of([4], [29], DEV), text)
    t = text.tolist()
    tree, parent = tree_of(t[0], t[1:], [(x + 1) % CFG.vocab for x in t[1:]])
    d.cache.reserve(0, 29, 29 + len(tree))
    # numbers that accept what the tree says: draft's probabilities on it, a flat target
    heat = torch.full((1,), 1e30, device=DEV)
    draft = torch.full((len(tree), CFG.vocab), 0.0, device=DEV)
    up = parent.long().clamp(min=0)
    for i, at in enumerate(up.tolist()):
        if i:
            draft[at, tree[i].long()] += 1e-9 if tree[i].item() in t else 0.5
    # a decoy: u 0.99 of 0.5 is not below 1/vocab
    u = torch.tensor([0.5] + [0.99, 0.0] * 3, dtype=torch.float64, device=DEV)
    path, count, _, new_len = d.verify(P.Rows.of([len(tree)], [29], DEV), tree, parent, temperature=heat,
                                       draft=draft, u=u)
    assert path[0, :4].tolist() == [0, 2, 4, 6] and new_len.item() == 33
    torch.cuda.synchronize()
    check_weighs(weighs)
    assert len(weighs) == 4 * CFG.layers
    assert rel(d.score[:, 0, :, :33], line.score[:, 0, :, :33]) < 1e-2
    assert not d.score[:, 1:].any()
    if not window:  # every row's weights are one together
        total = d.score[:, 0].double().sum(-1)
        assert ((total / (33 * CFG.heads // CFG.kv_heads) - 1).abs() < 1e-4).all()


def test_sampled_trees_are_the_walks_of_their_logits(model):  # noqa: F811
    """verify's path and next are what the rule says of the pass's own logits, and its
    greedy ones those at temperature 0."""
    d = decoder(model)
    g = torch.Generator().manual_seed(5)
    counts, lens = [7, 1, 5], [20, 33, 0]
    for s, n in enumerate(lens):
        d.cache.reserve(s, 0, n + counts[s])
        if n:
            d.forward(P.Rows.of([0] * s + [n], [0] * (s + 1), DEV), tokens(n, 20 + s))
    parent = [-1, 0, 0, 1, 1, 2, 4, -1, -1, 0, 1, 1, 3]
    rows = P.Rows.of(counts, lens, DEV)
    ids = tokens(13, 3)
    par = torch.tensor(parent, **I32)
    logits = d.forward(rows, ids, par, queries=[]).cpu()
    # siblings among the likely tokens
    at = 0
    for n in counts:
        for i in range(1, n):
            ids[at + i] = logits[at + parent[at + i]].topk(3).indices[i % 3]
        at += n
    heats = [0.2, 0.7, 0.1]
    agreed = 0
    for turn in range(6):
        logits = d.forward(rows, ids, par, queries=[]).cpu()
        pool, score = (d.cache.k.clone(), d.cache.v.clone()), d.score.clone()
        u = torch.rand(13, dtype=torch.float64, generator=g)
        want, at, margin = [], 0, math.inf
        for s, n in enumerate(counts):
            own = [p if 0 <= p < i else -1 for i, p in enumerate(parent[at:at + n])]
            h = 0.0 if turn == 0 else float(torch.tensor(heats[s]))
            w, m = B.walk(own, ids[at:at + n].tolist(), logits[at:at + n], h, u[at:at + n].tolist())
            want.append((own, w))
            margin = min(margin, m)
            at += n
        heat = torch.tensor([0.0] * 3 if turn == 0 else heats, device=DEV)
        outs = [d.verify(rows, ids, par, temperature=heat, u=u.to(DEV))]
        if turn == 0:
            d.cache.k.copy_(pool[0]), d.cache.v.copy_(pool[1]), d.score.copy_(score)
            outs.append(d.verify(rows, ids, par))
        if margin > MARGIN:
            agreed += 1
            for path, count, after, new_len in outs:
                at = 0
                for s, (own, w) in enumerate(want):
                    on = [i for i, x in enumerate(w) if x >= 0]
                    assert path[s, :len(on)].tolist() == on and count[s] == len(on)
                    assert after[s] == w[on[-1]] and new_len[s] == lens[s] + len(on)
                    assert [ids[at + i].item() for i in on[1:]] == [w[i] for i in on[:-1]]
                    at += counts[s]
    assert agreed >= 4
    with pytest.raises(ValueError, match="temperature"):
        d.verify(rows, ids, par, u=torch.zeros(13, dtype=torch.float64, device=DEV))
    # numbers of torch's generator
    torch.manual_seed(3)
    a = [t.clone() for t in d.verify(rows, ids, par, temperature=heat)]
    assert (a[1] > 0).all() and (a[2] >= 0).all()


def test_evicted_keys_and_the_text_behind_them(model):  # noqa: F811
    """Two sequences that share a prompt, one of them over its budget: what stays is what
    the weights say, the fork is as it was, and what follows is written at its place in
    the text and reads the kept keys alone."""
    d, whole = decoder(model), decoder(model)
    ids = tokens(90, 7)
    for x in (d, whole):
        x.cache.reserve(0, 0, 90)
        x.forward(P.Rows.of([90], [0], DEV), ids)
        x.fork(0, 2, 60)
    assert torch.equal(d.score[:, 2, :, :60], d.score[:, 0, :, :60]) and not d.score[:, 2, :, 60:].any()
    pool = d.cache.k.cpu(), d.cache.v.cpu()
    score, table = d.score.cpu(), d.cache.table.cpu()
    lens, kept = d.evict([90, 0, 60], 70, 4, 8)
    assert lens == [70, 0, 60] and d.gone.tolist() == [20, 0, 0]
    want, new_len = B.eviction(score, [90, 0, 60], 16, table, 40, None, 70, 4, 8)
    assert new_len == lens and d.cache.book.held(0) == 5
    now, tab = (d.cache.k.cpu(), d.cache.v.cpu()), d.cache.table.cpu()
    for lyr in range(CFG.layers):
        assert (kept[lyr, 1:] == -1).all()
        for h in range(CFG.kv_heads):
            x = want[lyr][0][h]
            assert kept[lyr, 0, h].tolist() == x
            for s, at in ((0, torch.tensor(x)), (2, torch.arange(60))):
                to = torch.arange(len(at))
                for a, b in zip(now, pool):
                    assert torch.equal(a[lyr, tab[s, to // 16].long(), h, to % 16],
                                       b[lyr, table[s, at // 16].long(), h, at % 16])
                assert torch.equal(d.score[lyr, s, h, :len(at)].cpu(), score[lyr, s, h, at])
    # the next tokens: layer 0's keys are those of the same text with nothing evicted
    # (by the token and its place alone), and the other sequence goes on as it would
    more = tokens(6, 8)
    got = []
    for x, n in ((d, 70), (whole, 90)):
        x.cache.reserve(0, n, n + 3)
        x.cache.reserve(2, 60, 63)
        got.append(x.forward(P.Rows.of([3, 0, 3], [n, 0, 60], DEV), more))
        t = x.cache.table.cpu().long()
        at = torch.arange(n, n + 3)
        got.append(x.cache.k.cpu()[0, t[0, at // 16], :, at % 16])
    assert torch.equal(got[1], got[3]) and torch.equal(got[0][3:], got[2][3:])
    assert torch.isfinite(got[0].float()).all()
    lens, _ = d.evict([73, 0, 63], 16, 2, 4)
    assert lens == [16, 0, 16] and d.gone.tolist() == [77, 0, 47] and d.cache.book.held(0) == 1
    d.cache.reserve(1, 0, 2)
    x = d.forward(P.Rows.of([0, 2, 0], [16, 0, 16], DEV), more[:2])
    assert torch.isfinite(x.float()).all() and d.gone.tolist() == [77, 0, 47]
    d.restart(0)
    assert d.gone.tolist() == [0, 0, 47] and d.cache.book.held(0) == 0


def test_evicting_whole_pages_is_a_cache_without_them(model):  # noqa: F811
    """first and last leave the same keys in every head: the logits that follow are those
    of a cache whose table has only their pages."""
    d, cut = decoder(model), decoder(model)
    ids, more = tokens(96, 9), tokens(5, 10)
    for x in (d, cut):
        x.cache.reserve(1, 0, 96)
        x.forward(P.Rows.of([0, 96], [0, 0], DEV), ids)
    assert d.evict([0, 96, 0], 64, 32, 32)[0] == [0, 64, 0]
    table = cut.cache.table
    table[1, 2:4] = table[1, 4:6].clone()
    table[1, 4:] = -1
    table[1, 4] = 39
    cut.gone[1] = 32
    d.cache.reserve(1, 64, 69)
    rows = P.Rows.of([0, 5, 0], [0, 64, 0], DEV)
    assert torch.equal(d.forward(rows, more), cut.forward(rows, more))


def test_a_sampled_step_in_a_graph(model):  # noqa: F811
    """Plan to weights captured in one of two graphs, replayed with eager work between."""
    d = decoder(model, 3, 0.75)
    for s, n in enumerate((9, 25)):
        d.cache.reserve(s, 0, n + 40)
        d.forward(P.Rows.of([0] * s + [n], [0] * (s + 1), DEV), tokens(n, 4 + s))
    parent = torch.tensor([-1, 0, 0, 1, 2] * 2, **I32)
    ids, rows = tokens(10, 6), P.Rows.of([5, 5], [9, 25], DEV)
    heat = torch.tensor([0.3, 1.0], device=DEV)
    u = torch.rand(10, dtype=torch.float64, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    d.verify(rows, ids, parent, temperature=heat, u=u, stream=side)  # sizes the linears' scratch
    torch.cuda.synchronize()
    graphs, got = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side, capture_error_mode="thread_local"):
            got.append(d.verify(rows, ids, parent, temperature=heat, u=u))
    for turn in range(4):
        ids.copy_(tokens(10, 20 + turn))
        logits = d.forward(rows, ids, parent, queries=[])
        ids[1] = logits[0].argmax()
        ids[7] = logits[5].topk(2).indices[1]
        u.copy_(torch.rand(10, dtype=torch.float64, generator=torch.Generator().manual_seed(turn)))
        rows.len.copy_(torch.tensor([9 - turn, 25 + turn], dtype=torch.int32))
        d.gone.copy_(torch.tensor([turn, 0, 0], dtype=torch.int32))
        state = [t.clone() for t in (d.cache.k, d.cache.v, d.score)]

        def restore():
            for t, x in zip((d.cache.k, d.cache.v, d.score), state):
                t.copy_(x)

        want = [t.clone() for t in d.verify(rows, ids, parent, temperature=heat, u=u)]
        after = [t.clone() for t in (d.cache.k, d.cache.v, d.score)]
        for gr, out in zip(graphs, got):
            restore()
            for t in out:
                t.fill_(-9)
            torch.cuda.synchronize()
            gr.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(a, b), turn
            for a, b in zip((d.cache.k, d.cache.v, d.score), after):
                assert torch.equal(a, b), turn


def test_decoders_and_evictions_that_are_refused(model):  # noqa: F811
    d = Q.PagedDecoder(model, 2, 8, 4, 16)
    with pytest.raises(RuntimeError, match="window"):
        d.evict([3, 0], 2)
    d = decoder(model)
    with pytest.raises(ValueError):
        d.evict([3], 2)
    with pytest.raises(ValueError):
        d.evict([3, 0, 0], 0)
    with pytest.raises(ValueError, match="holds pages"):
        d.evict([0, 33, 0], 2)
    # steps without rows, and rows of no sequence
    rows, none = P.Rows.of([0] * 2, [5] * 2, DEV), tokens(0, 1)
    _, count, _, new_len = d.verify(rows, none, none, temperature=torch.ones(2, device=DEV))
    assert count.tolist() == [0, 0] and new_len.tolist() == [5, 5]
    d.cache.reserve(0, 0, 6)
    rows = P.Rows(torch.tensor([0, 4], **I32), torch.tensor([0], **I32), 9, 4)
    parent = torch.tensor([-1, 0, 0, 1] + [7] * 5, **I32)
    path, count, _, _ = d.verify(rows, tokens(9, 3), parent, temperature=torch.zeros(1, device=DEV))
    assert count.item() >= 1 and torch.isfinite(d.score).all() and not d.score[:, :, :, count.item():].any()
