"""Weights of keys: a row's weights add up to one however large its scores are, whichever
path its pairs take."""
import pytest

torch = pytest.importorskip("torch")

from tests import _budget as B  # noqa: E402
from tests.test_gpu_budget import weighed  # noqa: E402
from tests.test_gpu_paged import batch  # noqa: E402

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("dtype,size", [(F16, 8), (F16, 64), (F16, 96), (F16, 512), (BF16, 32), (BF16, 128)])
@pytest.mark.parametrize("n,group,window", [(1, 4, 0), (8, 4, 0), (9, 4, 0), (40, 1, 0), (129, 3, 0), (200, 2, 33)])
def test_weights_of_large_scores_add_up(n, group, window, dtype, size):
    """Scores of 63 * 64 size (2^19 for 128) and a few more, whole numbers that 32 bits hold:
    what differs between a row's keys is those few (at most 10), so a weight is as exact
    as one of small scores: powers and the sum of `keys` terms (keys + 64) 2^-23, the
    scale's own rounding 10 * 2^-24 log2(e).  Scores of 2^20 powers of two and more are
    rounded when they are scaled, and those of up to 32 pairs are always: there all keys of
    a row are alike, and their scores too."""
    counts, lens, page = [n, 3], [300, 70], 16
    g, k, v, table, cu, _ = batch(counts, lens, dtype, 2, group, 64, page, 3)
    pairs = (window or n) * group
    alike = pairs <= 32 or 63 * 64 * size * 1.4427 * 2 >= 2 ** 20
    k = torch.full_like(k, size)
    q = torch.full((sum(counts), 2 * group, 64), 64.0).to(dtype)
    k[..., 0] = 0 if alike else torch.randint(0, 6, k.shape[:-1], generator=g).to(dtype)
    q[..., 0] = torch.randint(0, 3, q.shape[:-1], generator=g).to(dtype)
    seen = [[list(range(i + 1)) for i in range(m)] for m in counts]
    had = torch.zeros(2, 2, 600)
    want, _ = B.weights(q, k, table, cu, lens, seen, page, group, 1.0, had, 1.0, window)
    got = weighed(k, table, counts, lens, q, had, scale=1.0, window=window).double()
    off = (got - want).abs() - want * ((300 + n + 64) * 2.0 ** -23 + 10 * 1.5 * 2.0 ** -24 + (pairs + 4) * 2.0 ** -24)
    assert float(off.max()) <= 2.0 ** -100
    total = got[0].sum(-1)
    assert ((total / pairs - 1).abs() < 1e-4).all()
