"""The operators over a paged KV cache restated in 64 bits on the CPU, from
their formulas, and the bounds that the kernels' roundings give them."""
import math

import torch

F64 = torch.float64


def half_step(dtype) -> float:
    """The most that one rounding moves a value, relative to it."""
    return torch.finfo(dtype).eps / 2


def slots(table, s, page, keys):
    """Pool slots (page number, row) of a sequence's first `keys` keys."""
    at = torch.arange(keys)
    return table[s, at // page].long(), at % page


def ancestors(parent):
    """Index lists: row i's ancestors and itself (a parent that does not lie
    before its row counts as none)."""
    out = []
    for i, p in enumerate(parent):
        out.append((out[p] if 0 <= p < i else []) + [i])
    return out


def masks(rows_of, words):
    """Ancestor lists of all rows as int64 words."""
    m = torch.zeros(len(rows_of), words, dtype=torch.int64)
    for t, js in enumerate(rows_of):
        for j in js:
            bit = 1 << (j % 64)
            m[t, j // 64] |= bit - (1 << 64) if bit >> 63 else bit
    return m


def attention(q, kpool, vpool, table, cu, lens, seen, page, group, scale, layer=0):
    """(out, bound): attention of every row in 64 bits, `seen[s][i]` the rows of
    its sequence that row i sees besides the context, and how far a kernel may be
    off that rounds its weights and its output to the pool's type:

      A = sum of weight * |value| bounds |out|;
      a weight rounded by half a step u, over a sum of rounded weights: 2 u A;
      a score's f32 sum of `dim` products and its scaling: off by at most es =
      (dim + 4) 2^-24 * (sum |q k| scale), a weight by the factor e^es: 2 es A
      (es below 1/4, so e^es - 1 <= 1.2 es: 2.4);
      f32 powers, sums and divisions: (keys + 64) 2^-23 A;
      weights below f16's smallest, 2^-24 where the row's reference weighs 2^11 (half of
        a step of 2^-24 is 2^-36 of it): keys 2^-36 max|v|;
      the output's own rounding: u |out|, or half of the type's smallest number.
    """
    dt = q.dtype
    u, tiny = half_step(dt), torch.finfo(dt).tiny * torch.finfo(dt).eps / 2
    n_all, heads, dim = q.shape
    out = torch.zeros(n_all, heads, dim, dtype=F64)
    tol = torch.zeros_like(out)
    for s in range(len(lens)):
        n = cu[s + 1] - cu[s]
        if n == 0:
            continue
        pg, row = slots(table, s, page, lens[s] + n)
        K = kpool[layer, pg, :, row].to(F64)  # [keys, kv, dim]
        V = vpool[layer, pg, :, row].to(F64)
        for i in range(n):
            at = torch.tensor(list(range(lens[s])) + [lens[s] + j for j in seen[s][i]],
                              dtype=torch.long)
            if len(at) == 0:
                tol[cu[s] + i] = 0
                continue
            for h in range(heads):
                k, v = K[at, h // group], V[at, h // group]
                x = q[cu[s] + i, h].to(F64)
                p = torch.softmax(k @ x * scale, 0)
                o = p @ v
                A = p @ v.abs()
                es = float((k.abs() @ x.abs()).max()) * abs(scale) * (dim + 4) * 2.0 ** -24
                out[cu[s] + i, h] = o
                tol[cu[s] + i, h] = (A * (2 * u + 2.4 * es + (len(at) + 64) * 2.0 ** -23)
                                     + len(at) * 2.0 ** -36 * v.abs().amax(0) + u * o.abs() + tiny)
    return out, tol


def rotated(x, w, pos, eps, theta):
    """(out, bound) of norm and rotation, x [rows, heads, dim].

    The f32 sum of squares, root and products move a normalized value by at most
    (dim + 8) 2^-24 of it; an angle's remainder (at most a turn, rounded to 32
    bits, 2^-24 turns) and the f32 sine move a product by at most (2 pi 2^-24 +
    2^-21) of it; one rounding to the type at the end."""
    dt, dim = x.dtype, x.shape[-1]
    u, tiny = half_step(dt), torch.finfo(dt).tiny * torch.finfo(dt).eps / 2
    y = x.to(F64)
    if w is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * w.to(F64)
    half = dim // 2
    a = pos.to(F64)[:, None, None] * theta ** (-torch.arange(half, dtype=F64) / half)
    c, s = torch.cos(a), torch.sin(a)
    p, r = y[..., :half], y[..., half:]
    out = torch.cat([p * c - r * s, r * c + p * s], -1)
    most = torch.cat([p.abs() + r.abs()] * 2, -1)
    return out, most * ((dim + 8) * 2.0 ** -24 + 2 * math.pi * 2.0 ** -24 + 2.0 ** -21) \
        + u * out.abs() + tiny


def walk(parent, ids, target, most):
    """The accepted rows of one tree and the token after them."""
    if not ids:
        return [], -1
    path = [0]
    while len(path) < most:
        fits = [j for j in range(path[-1] + 1, len(ids))
                if parent[j] == path[-1] and ids[j] == target[path[-1]]]
        if not fits:
            break
        path.append(fits[0])
    return path, target[path[-1]]


def random_tree(n, g):
    """Parents of n rows under one root."""
    return [-1] + [int(torch.randint(0, i, (1,), generator=g)) for i in range(1, n)]


def random_forest(n, g):
    """Parents of n rows, about a third of them roots, and some that are parents of
    nothing that comes behind: the row itself, a later one, a negative number."""
    out = random_tree(n, g) if n else []
    for i in range(n):
        x = int(torch.randint(0, 12, (1,), generator=g))
        if x < 6:
            out[i] = {0: i, 1: i + 1, 2: -7}.get(x, -1)
    return out


def random_table(counts, lens, page, extra, g, max_pages=None):
    """A table whose pages lie in the pool in a random order, and the pool's pages."""
    need = [-(-(n + c) // page) for n, c in zip(counts, lens)]
    pages = sum(need) + extra
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.full((len(counts), max_pages or max(need + [1])), -1, dtype=torch.int32)
    for s, k in enumerate(need):
        for x in range(k):
            table[s, x] = order.pop()
    return table, pages
