"""Sampled verification, weights of keys and eviction where offsets pass 32 bits, where
sequences share pages, and where calls run at once or share a scratch: each equals
the plain call of the same data bit for bit."""
import pytest

torch = pytest.importorskip("torch")

from plugins_amd import paged as P  # noqa: E402
from tests.test_gpu_budget import drafted  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16 = torch.float16, torch.bfloat16
I32 = {"dtype": torch.int32, "device": DEV}
FAR = 33800  # pages of 128 KB: 4.4 GB a pool


def far_pools(shape, small, table):
    """(k, v, table): the same keys on pages of which most lie past 2^32 bytes."""
    to = torch.arange(small[0].shape[1])
    to = torch.where(to % 3 == 1, to + 5, FAR - 1 - to)
    big = []
    for x in small:
        far = torch.empty(x.shape[0], FAR, *shape, dtype=x.dtype, device=DEV)
        far[:, to.to(DEV)] = x
        big.append(far)
    return big[0], big[1], torch.where(table < 0, -1, to[table.clamp(min=0)]).to(torch.int32)


@pytest.mark.parametrize("n,window", [(1, 0), (8, 0), (40, 0), (40, 8)])
def test_weigh_pools_past_32_bits(n, window):
    g = torch.Generator(device=DEV).manual_seed(n)
    shape = (2, 256, 128)
    k = torch.randn(1, 5, *shape, generator=g, device=DEV).to(F16)
    table = torch.tensor([[3, 0, 4], [1, 2, -1]], dtype=torch.int32)
    rows = P.Rows.of([n, n], [700, 300], DEV)
    q = torch.randn(2 * n, 8 * 128, generator=g, device=DEV).to(F16)
    had = torch.rand(2, 2, 768, generator=g, device=DEV)
    got = []
    for kk, vv, t in ((k, torch.empty_like(k), table), far_pools(shape, (k, k), table)):
        score = had.clone()
        P.weigh(P.PagedCache.over(kk, vv, t.to(DEV)), 0, rows, q, score, window=window)
        got.append(score)
    assert not torch.equal(got[0], had) and torch.equal(got[0], got[1])


def test_evict_pools_past_32_bits():
    g = torch.Generator(device=DEV).manual_seed(2)
    shape = (2, 256, 128)
    k, v = (torch.randn(1, 5, *shape, generator=g, device=DEV).to(BF16) for _ in range(2))
    table = torch.tensor([[3, 0, 4], [1, 2, -1]], dtype=torch.int32)
    lens = torch.tensor([760, 500], **I32)
    score = torch.rand(1, 2, 2, 768, generator=g, device=DEV)
    got = []
    for kk, vv, t in ((k.clone(), v.clone(), table), far_pools(shape, (k, v), table)):
        kept, new, new_len = torch.empty(1, 2, 2, 400, **I32), score.clone(), torch.empty(2, **I32)
        P.evict(P.PagedCache.over(kk, vv, t.to(DEV)), lens, score, kept, new, new_len, first=2, last=30)
        pages = t.clamp(min=0).long().to(DEV)
        got.append([kk[:, pages[s, :2]] for s in range(2)] + [vv[:, pages[s, :2]] for s in range(2)] +
                   [kept, new, new_len])
    assert all(torch.equal(a, b) for a, b in zip(*got))
    assert got[0][-1].tolist() == [400, 400] and not torch.equal(got[0][0], k[:, [3, 0]])


@pytest.mark.parametrize("counts,draft", [([1, 1, 1], None), ([3], None), ([3], F16), ([1, 2], F16)])
def test_verify_rows_past_32_bits(counts, draft):
    """Rows 1.2 * 10^9 elements apart."""
    V, far = 5003, 1_200_000_000
    z, q, parent, ids, heats, u = drafted(counts, V, F16, draft, False, 5)
    z, q = z.to(DEV), None if q is None else q.to(DEV)
    rows = P.Rows.of(counts, [0] * len(counts), DEV)

    def apart(x):
        if x is None:
            return None
        y = torch.empty(2 * far + V, dtype=F16, device=DEV).as_strided((3, V), (far, 1))
        y.copy_(x)
        return y

    got = []
    for zz, qq in ((z, q), (apart(z), apart(q))):
        target = torch.full((3,), 9, **I32)
        P.verify(rows, torch.tensor(parent, **I32), torch.tensor(ids, **I32), zz, u.to(DEV), target, qq,
                 torch.tensor(heats, device=DEV))
        got.append(target.tolist())
    assert got[0] == got[1]


@pytest.mark.parametrize("n", [1, 40])
def test_weigh_sequences_that_share_pages(n):
    """A page in two tables, and twice in one of them."""
    g = torch.Generator(device=DEV).manual_seed(n)
    k = torch.randn(1, 6, 2, 64, 64, generator=g, device=DEV).to(BF16)
    shared = torch.tensor([[1, 0, 2], [1, 0, 3], [4, 1, 1]], dtype=torch.int32)
    alone = k[:, shared.flatten().long().to(DEV)]
    rows = P.Rows.of([n, n, n], [130, 120, 128], DEV)
    q = torch.randn(3 * n, 4 * 64, generator=g, device=DEV).to(BF16)
    got = []
    for kk, t in ((k, shared), (alone, torch.arange(9, dtype=torch.int32).view(3, 3))):
        score = torch.zeros(3, 2, 192, device=DEV)
        P.weigh(P.PagedCache.over(kk, torch.empty_like(kk), t.to(DEV)), 0, rows, q, score)
        got.append(score)
    assert torch.equal(got[0], got[1]) and float(got[0].sum()) == pytest.approx(3 * n * 4, rel=1e-4)


def calls_of(seed):
    """The three operators on data of the seed: a function of (scratches), and its outputs."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    V, n = 40007, 12
    z = 3 * torch.randn(2 * n, V, generator=g, device=DEV)
    q = torch.softmax(torch.randn(2 * n, V, generator=g, device=DEV), -1)
    parent = torch.tensor([max(-1, (i - 1) // 2) for i in range(n)] * 2, **I32)
    ids = torch.randint(0, V, (2 * n,), generator=g, device=DEV).int()
    u = torch.rand(2 * n, generator=g, device=DEV, dtype=torch.float64)
    k, v = (torch.randn(1, 70, 2, 64, 128, generator=g, device=DEV).to(F16) for _ in range(2))
    table = torch.arange(70, **I32).view(2, 35)
    c = P.PagedCache.over(k, v, table)
    rows = P.Rows.of([n, n], [2000, 1500], DEV)
    x = torch.randn(2 * n, 8 * 128, generator=g, device=DEV).to(F16)
    score = torch.zeros(1, 2, 2, 35 * 64, device=DEV)
    kept, new_len = torch.empty(1, 2, 2, 700, **I32), torch.empty(2, **I32)
    target, new = torch.empty(2 * n, **I32), torch.zeros_like(score)
    lens = torch.tensor([2000 + n, 1500 + n], **I32)

    def call(a=None, b=None):
        P.verify(rows, parent, ids, z, u, target, q, scratch=a)
        score.zero_()
        P.weigh(c, 0, rows, x, score[0], scratch=b)
        P.evict(c, lens, score, kept, new, new_len, first=4, last=20)

    start = (k.clone(), v.clone())

    def back():
        k.copy_(start[0]), v.copy_(start[1]), new.zero_(), kept.zero_(), target.zero_()

    sizes = (P.verify_scratch_bytes(rows, V), P.weigh_scratch_bytes(c, rows, 8, 0, 35 * 64))
    return call, back, (target, score, k, v, kept, new, new_len), sizes


def test_calls_at_once_and_graphs_of_one_scratch():
    """Two streams at once, with scratches of torch's allocator; then two graphs that hold
    the same scratch, replayed one after the other several times."""
    pairs = [calls_of(1), calls_of(2)]
    want = []
    for call, back, out, _ in pairs:
        call()
        want.append([x.clone() for x in out])
        back()

    def check(which):
        for w, x in zip(want[which], pairs[which][2]):
            assert torch.equal(w, x)
        pairs[which][1]()

    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for (call, _, _, _), s in zip(pairs, streams):
            with torch.cuda.stream(s):
                call()
        torch.cuda.synchronize()
        check(0), check(1)
        torch.cuda.synchronize()
    a, b = (torch.empty(n, dtype=torch.uint8, device=DEV) for n in pairs[0][3])
    graphs = []
    for call, back, _, _ in pairs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(a, b)
        graphs.append(graph)
        back()
    for _ in range(3):
        graphs[0].replay()
        graphs[1].replay()
        check(1), check(0)
        torch.cuda.synchronize()
        a.fill_(255), b.fill_(255)  # what a scratch holds before a call is nothing's
