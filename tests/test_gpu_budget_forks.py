"""A decoder's forks of sequences that have evicted keys: the rows that follow are at the
places that their text has.  Verified steps without sequences."""
import pytest

torch = pytest.importorskip("torch")

from plugins_amd import paged as P  # noqa: E402
from tests.test_gpu_budget_decoder import decoder  # noqa: E402
from tests.test_gpu_paged_decoder import CFG, DEV, model, tokens  # noqa: E402,F401

pytestmark = pytest.mark.gpu


def put(d, seq, have, ids):
    d.cache.reserve(seq, have, have + len(ids))
    return d.forward(P.Rows.of([0] * seq + [len(ids)], [0] * seq + [have], DEV), ids)


def first_keys(d, seq, at, n):
    """Layer 0's keys from number `at` on: by the token and its place in the text alone."""
    t, x = d.cache.table[seq].cpu().long(), torch.arange(at, at + n)
    return d.cache.k.cpu()[0, t[x // 16], :, x % 16]


def test_forks_after_an_eviction(model):  # noqa: F811
    """90 keys brought down to 70: the first 4 and the last 8 are the text's, in between every
    head kept its own."""
    d, after = decoder(model, seqs=6), {}
    ids, more = tokens(90, 7), tokens(5, 8)
    put(d, 0, 0, ids)
    for x in (4, 3, 90, 84):  # what follows texts of these lengths
        w = decoder(model, seqs=1)
        put(w, 0, 0, ids[:x])
        put(w, 0, x, more)
        after[x] = first_keys(w, 0, x, 5)
    assert d.evict([90, 0, 0, 0, 0, 0], 70, 4, 8)[0][0] == 70
    for dst, keys, text in ((1, 4, 4), (2, 3, 3), (3, 70, 90), (4, 64, 84)):
        d.fork(0, dst, keys)
        put(d, dst, keys, more)
        assert torch.equal(first_keys(d, dst, keys, 5), after[text]), keys
    assert d.gone.tolist() == [20, 0, 0, 20, 20, 0]
    for keys in (5, 30, 61):
        with pytest.raises(ValueError, match="evicted"):
            d.fork(0, 5, keys)
    assert d.cache.book.held(5) == 0
    # (the fork at 4 has evicted nothing)
    d.restart(5)
    d.fork(1, 5, 9)
    assert d.gone.tolist()[5] == 0


def test_forks_after_several_evictions_and_restarts(model):  # noqa: F811
    d = decoder(model, seqs=4)
    ids = tokens(120, 3)
    put(d, 0, 0, ids[:80])
    d.evict([80, 0, 0, 0], 50, 6, 20)    # numbers 30 .. 49 are 60 .. 79 of the text
    put(d, 0, 50, ids[80:100])           # 50 .. 69 are 80 .. 99
    d.evict([70, 0, 0, 0], 60, 10, 45)   # 15 .. 59: of these 20 .. 59 were 30 .. 69
    assert d.gone.tolist() == [40, 0, 0, 0]
    for keys, gone in ((6, 0), (20, 40), (60, 40), (33, 40)):
        d.fork(0, 1, keys)
        assert d.gone.tolist()[1] == gone, keys
        d.restart(1)
    for keys in (7, 15, 19):
        with pytest.raises(ValueError, match="evicted"):
            d.fork(0, 1, keys)
    # a fork keeps what its source knows, a restart forgets it
    d.fork(0, 1, 40)
    with pytest.raises(ValueError, match="evicted"):
        d.fork(1, 2, 15)
    d.fork(1, 2, 30)
    d.restart(1)
    put(d, 1, 0, ids[:30])
    d.fork(1, 3, 15)
    assert d.gone.tolist() == [40, 0, 40, 0]
    # first and last that keep everything else alike: no key between them is any head's own
    d.restart(2), d.restart(3)
    put(d, 2, 0, ids[:40])
    d.evict([0, 0, 40, 0], 24, 8, 16)
    for keys, gone in ((8, 0), (9, 16), (24, 16)):
        d.fork(2, 3, keys)
        assert d.gone.tolist()[3] == gone
        d.restart(3)


def test_forks_without_evictions_and_without_weights(model):  # noqa: F811
    d = decoder(model, seqs=3)
    put(d, 0, 0, tokens(40, 1))
    d.evict([40, 0, 0], 40)  # nothing goes
    d.fork(0, 1, 17)
    assert d.gone.tolist() == [0, 0, 0]
    with pytest.raises(Exception):
        d.fork(0, 1, 3)  # holds pages already
    plain = decoder(model, None, seqs=2)
    put(plain, 0, 0, tokens(40, 1))
    plain.fork(0, 1, 17)
    assert CFG.layers and plain.gone is None


@pytest.mark.parametrize("window", [None, 0, 2])
def test_a_verified_step_of_no_sequences(model, window):  # noqa: F811
    """Rows that pad a step whose sequences are all gone."""
    d = decoder(model, window, seqs=2)
    i32 = {"dtype": torch.int32, "device": DEV}
    rows = P.Rows(torch.zeros(1, **i32), torch.empty(0, **i32), 5, 0)
    for kw in ({}, {"temperature": torch.empty(0, device=DEV)}):
        path, count, after, new_len = d.verify(rows, tokens(5, 1), None, **kw)
        assert path.shape == (0, 1) and count.shape == after.shape == new_len.shape == (0,)
    assert not d.cache.k.any() and (window is None or not d.score.any())
