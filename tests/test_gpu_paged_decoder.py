"""A decoder over the paged cache: prompts, single tokens and verified trees run
through plan, append, attention and commit together, against the decoder that
keeps one contiguous cache a sequence and against itself taken token by token."""
import pytest

torch = pytest.importorskip("torch")

from plugins_amd import exl3 as X  # noqa: E402
from plugins_amd import paged as P  # noqa: E402
from plugins_amd import qwen3 as Q  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
CFG = Q.Qwen3Config(layers=2, hidden=1024, heads=8, kv_heads=2, inter=2048, vocab=1024)


def rel(a, b):
    a, b = a.double(), b.double()
    return float((a - b).norm() / b.norm())


def tokens(n, seed):
    return torch.randint(0, CFG.vocab, (n,), generator=torch.Generator().manual_seed(seed),
                         dtype=torch.int32).to(DEV)


def paged(model, seqs=3, pages=40, max_pages=12, page=16):
    return Q.PagedDecoder(model, seqs, pages, max_pages, page)


@pytest.fixture(scope="module")
def model():
    return Q.Qwen3Decoder(CFG, 1, 100, seed=5)


def by_steps(model, ids):
    """Logits of a line of tokens from the contiguous decoder, one a step."""
    out = []
    for i, t in enumerate(ids.tolist()):
        model.ids.fill_(t)
        model.pos.fill_(i)
        out.append(model.step().clone())
    return torch.cat(out)


def test_prompt_and_tokens_against_the_contiguous_decoder(model):
    """37 tokens as one prompt, as two pieces, and one by one: f16 roundings in
    other places (1e-2 relative Frobenius, as the contiguous step is held to
    against its float32 restatement)."""
    ids = tokens(37, 1)
    want = by_steps(model, ids)
    d = paged(model)
    for s, cuts in enumerate(([37], [20, 17], [1] * 37)):
        at, got = 0, []
        for n in cuts:
            d.cache.reserve(s, at, at + n)
            rows = P.Rows.of([0] * s + [n], [0] * s + [at], DEV)
            got.append(d.forward(rows, ids[at:at + n]))
            at += n
        r = rel(torch.cat(got), want)
        assert r < 1e-2, (cuts, r)
    # the last row's logits alone
    d.cache.trim(0, 0)
    d.cache.reserve(0, 0, 37)
    last = d.forward(P.Rows.of([37], [0], DEV), ids, only=torch.tensor([36], device=DEV))
    assert rel(last, want[-1:]) < 1e-2


def test_sequences_side_by_side_are_as_they_are_alone(model):
    """Three sequences of unlike lengths in one pass."""
    lens, new = [0, 13, 30], [21, 1, 6]
    ids = [tokens(a + b, 10 + i) for i, (a, b) in enumerate(zip(lens, new))]
    d = paged(model)
    for s, n in enumerate(lens):
        d.cache.reserve(s, 0, n + new[s])
        if n:
            d.forward(P.Rows.of([0] * s + [n], [0] * (s + 1), DEV), ids[s][:n])
    got = d.forward(P.Rows.of(new, lens, DEV), torch.cat([x[n:] for x, n in zip(ids, lens)]))
    at = 0
    for s, n in enumerate(lens):
        want = by_steps(model, ids[s])[n:]
        assert rel(got[at:at + new[s]], want) < 1e-2, s
        at += new[s]


def test_a_verified_tree_goes_on_as_the_accepted_tokens(model):
    """Trees whose accepted path is known: the model's own continuation among
    decoys.  What follows reads the moved keys and values: logits as of the
    same tokens in a line, and the same tokens greedily."""
    d, line = paged(model), paged(model)
    prompt = tokens(19, 3)
    for x in (d, line):
        x.cache.reserve(0, 0, 19)
        first = x.forward(P.Rows.of([19], [0], DEV), prompt)[-1]
    have, token, said = 19, int(first.float().argmax()), []
    # the line's greedy continuation
    at, t = 19, token
    for _ in range(12):
        said.append(t)
        line.cache.reserve(0, at, at + 1)
        logits = line.forward(P.Rows.of([1], [at], DEV),
                              torch.tensor([t], dtype=torch.int32, device=DEV))
        t, at = int(logits[0].float().argmax()), at + 1
    kept = [token]
    while len(kept) < 9:
        # row 0 the certain token; a path of 3 true tokens at scattered rows,
        # decoys around it
        a = len(kept)
        true = said[a:a + 3]
        decoy = [(x + 1) % CFG.vocab for x in true]
        ids = [kept[-1], decoy[0], true[0], decoy[1], true[1], decoy[2], true[2]]
        parent = [-1, 0, 0, 1, 2, 2, 4]
        d.cache.reserve(0, have, have + 7)
        rows = P.Rows.of([7], [have], DEV)
        path, count, after, new_len = d.verify(
            rows, torch.tensor(ids, dtype=torch.int32, device=DEV),
            torch.tensor(parent, dtype=torch.int32, device=DEV))
        assert path[0, :4].tolist() == [0, 2, 4, 6] and count.item() == 4
        have = new_len.item()
        d.cache.trim(0, have)
        kept += true + [after.item()]
    # the same tokens as the line's, and the next logits too
    n = min(len(kept), len(said))
    assert kept[:n] == said[:n]
    text = torch.cat([prompt, torch.tensor(kept, dtype=torch.int32, device=DEV)])
    d.cache.reserve(0, have, have + 1)
    got = d.forward(P.Rows.of([1], [have], DEV), text[have:have + 1])
    want = by_steps(model, text[:have + 1])[-1:]
    assert rel(got, want) < 1e-2


def test_a_verified_step_in_a_graph(model):
    """plan to commit captured, replayed with eager work between: every replay is
    the eager step's result, lengths and tokens changed in place."""
    d = paged(model)
    prompts = [tokens(9, 4), tokens(25, 5)]
    for s, p in enumerate(prompts):
        d.cache.reserve(s, 0, len(p) + 40)
        d.forward(P.Rows.of([0] * s + [len(p)], [0] * (s + 1), DEV), p)
    parent = torch.tensor([-1, 0, 0, 1, 2] * 2, dtype=torch.int32, device=DEV)
    ids = tokens(10, 6)
    rows = P.Rows.of([5, 5], [9, 25], DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    d.verify(rows, ids, parent, stream=side)  # sizes the linears' scratch of the stream
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side, capture_error_mode="thread_local"):
        got = d.verify(rows, ids, parent)
    for turn in range(4):
        ids.copy_(tokens(10, 20 + turn))
        rows.len.copy_(torch.tensor([9 - turn, 25 + turn], dtype=torch.int32))
        pool = d.cache.k.clone(), d.cache.v.clone()
        want = [t.clone() for t in d.verify(rows, ids, parent)]
        after = d.cache.k.clone(), d.cache.v.clone()
        d.cache.k.copy_(pool[0])
        d.cache.v.copy_(pool[1])
        for t in got:
            t.fill_(-9)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), turn
        assert torch.equal(d.cache.k, after[0]) and torch.equal(d.cache.v, after[1])


@pytest.mark.parametrize("fill", [-1, CFG.vocab, 2 ** 31 - 1, -2 ** 31])
def test_padding_rows_may_hold_any_id(model, fill):
    """Rows behind the last sequence, and a drafted row of a token that the
    vocabulary has not: the embedding reads inside its table, and the other rows
    are what they are beside ids of the vocabulary."""
    got = []
    for pad, odd in ((0, 0 if fill < 0 else CFG.vocab - 1), (fill, fill)):
        d = paged(model)
        d.cache.reserve(0, 0, 6)
        rows = P.Rows(torch.tensor([0, 6], dtype=torch.int32, device=DEV),
                      torch.tensor([0], dtype=torch.int32, device=DEV), 9, 6)
        ids = torch.cat([tokens(6, 30), torch.full((3,), pad, dtype=torch.int32, device=DEV)])
        ids[4] = odd
        got.append(d.forward(rows, ids)[:6].clone())
    assert torch.isfinite(got[0].float()).all() and torch.equal(*got)


@pytest.mark.parametrize("seqs", [0, 2])
def test_steps_without_rows(model, seqs):
    """Nothing drafted and nothing prompted: no logits, nothing accepted, lengths
    as they were."""
    d = paged(model)
    rows, ids = P.Rows.of([0] * seqs, [5] * seqs, DEV), tokens(0, 1)
    none = torch.empty(0, dtype=torch.int64, device=DEV)
    for only in (None, none):
        assert d.forward(rows, ids, only=only).shape == (0, CFG.vocab)
    with pytest.raises(IndexError):
        d.forward(rows, ids, only=torch.zeros(1, dtype=torch.int64, device=DEV))
    path, count, after, new_len = d.verify(rows, ids, ids)
    assert path.tolist() == [[-1]] * seqs and count.tolist() == [0] * seqs
    assert after.tolist() == [-1] * seqs and new_len.tolist() == [5] * seqs
    torch.cuda.synchronize()


def test_more_rows_than_a_grid_has_in_one_dimension(model):
    """Prompts of 65600 rows in one step: the embedding of every row, and the last
    prompt's logits as of the same prompt alone (f16 roundings in other places)."""
    n = [30000, 35000, 600]
    ids = tokens(sum(n), 40)
    h = torch.empty(sum(n), CFG.hidden, device=DEV)
    Q.embed(ids, model.embed_table, h)
    assert torch.equal(h, model.embed_table[ids.long()].float())
    ssq = torch.empty(sum(n), CFG.hidden // 128, device=DEV)
    h.zero_()
    Q.embed(ids, model.embed_table, h, ssq)
    assert torch.equal(h, model.embed_table[ids.long()].float())
    # a sum of 128 squares in 32 bits, in any order: 128 roundings of it at most
    want = h.double().view(sum(n), -1, 128).pow(2).sum(-1)
    assert bool(((ssq.double() - want).abs() <= 128 * 2.0 ** -24 * want).all())
    d = paged(model, 3, 262, 140, 256)
    for s, m in enumerate(n):
        d.cache.reserve(s, 0, m)
    last = torch.arange(65000, 65600, device=DEV)
    got = d.forward(P.Rows.of(n, [0] * 3, DEV), ids, only=last)
    d.cache.trim(2, 0)
    d.cache.reserve(2, 0, 600)
    alone = d.forward(P.Rows.of([0, 0, 600], [0] * 3, DEV), ids[65000:])
    assert rel(got, alone) < 1e-2


def test_a_path_of_no_rows_is_refused(model):
    """most=0 is no default; of 1 the certain token alone is accepted."""
    d = paged(model)
    d.cache.reserve(0, 0, 3)
    rows, ids = P.Rows.of([3], [0], DEV), tokens(3, 50)
    with pytest.raises(X.Exl3Error, match="PagedPath"):
        d.verify(rows, ids, most=0)
    path, count, _, new_len = d.verify(rows, ids, most=1)
    assert path.tolist() == [[0]] and count.tolist() == [1] and new_len.tolist() == [1]
