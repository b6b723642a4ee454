"""Sampled verification, weights of keys and eviction restated in 64 bits on the
CPU, from their formulas, and the bounds that the kernels' roundings give."""
import math

import torch

from tests._paged import slots

F64 = torch.float64


def probabilities(z, heat):
    """A row's softmax in 64 bits; None where it has none."""
    z = z.to(F64)
    if torch.isnan(z).any() or not (z > -math.inf).any() or not 0 <= heat < math.inf:
        return None
    if heat == 0:
        p = torch.zeros_like(z)
        p[(z == z.max()).nonzero()[0, 0]] = 1.0
        return p
    if torch.isinf(z.max()):
        return None
    e = torch.exp((z - z.max()) / heat)
    return e / e.sum()


def walk(parent, ids, z, heat, u, draft=None, distinct=False):
    """(target, margin) of one sequence: the tokens that follow the rows of its
    walk, -1 for others, and how near the closest decision was to its border
    (relative; what a kernel's rounding may not reach)."""
    n, V = len(ids), z.shape[1]
    target, margin, at = [-1] * n, math.inf, 0
    if n == 0:
        return target, margin
    while True:
        p = probabilities(z[at], heat)
        if p is None:
            return target, margin
        rest, A, B, taken, to = p.clone(), 1.0, 1.0, 0.0, None
        q = None if draft is None else draft[at].to(F64)
        for c in (c for c in range(at + 1, n) if parent[c] == at):
            inside = 0 <= ids[c] < V
            pc = float(rest[ids[c]]) if inside else 0.0
            qc = 1.0 if q is None else float(q[ids[c]]) if inside else 0.0
            step = A if q is None else A / max(B, 2.0 ** -53)
            need = u[c] * step * qc
            if heat > 0 and max(need, pc) > 0:
                margin = min(margin, abs(need - pc) / max(need, pc))
            if pc == 1.0 if heat == 0 else need < pc:
                to = c
                break
            if heat == 0:
                continue
            if q is None:
                A -= pc
                if inside:
                    rest[ids[c]] = 0.0
            else:
                taken += step
                B -= qc if distinct else 0.0
                rest = (p - taken * q).clamp(min=0)
                A = float(rest.sum())
        if to is not None:
            target[at] = ids[to]
            at = to
            continue
        if heat == 0:
            target[at] = int(p.argmax())
            return target, margin
        r = rest if float(rest.sum()) > 0 else p
        c = r.cumsum(0)
        border = u[0] * float(c[-1])
        over = ((c > border) & (r > 0)).nonzero()
        v = int(over[0, 0]) if len(over) else int((r > 0).nonzero()[-1, 0])
        if len(over):
            margin = min(margin, 1e7 * float((c - border).abs()[r > 0].min() / c[-1]))
        target[at] = v
        return target, margin


def weights(q, kpool, table, cu, lens, seen, page, group, scale, had, decay=1.0, window=0, base=None,
            layer=0):
    """(score, bound) after a step, in 64 bits, from the scores `had` [seqs, kv,
    room]; seen[s][i]: rows of its sequence that row i sees besides the context.

    A weight w = e^(x - max) / sum has, in 32 bits: a score's sum of `dim` products and
    its scaling, off by at most es = (dim + 4) 2^-24 (sum |q k| scale), so a factor of e^es in
    its power and one in the sum (2 es; es below 1/4: 2.4); the power, the sum of `keys`
    terms, the division and the product, (keys + 64) 2^-23; powers below 2^-126 are
    lost.  The sum over the pairs and what was there: 2^-24 of it a step."""
    n_all, heads, dim = q.shape
    kv = heads // group
    out = had.to(F64).clone()
    tol = torch.zeros_like(out)
    for s in range(len(lens)):
        n = cu[s + 1] - cu[s]
        if n == 0:
            continue
        keys = lens[s] + n
        pg, row = slots(table, s, page, keys)
        K = kpool[layer, pg, :, row].to(F64)
        b = lens[s] if base is None else base[s]
        total = torch.zeros(kv, keys, dtype=F64)
        slack = torch.zeros(kv, keys, dtype=F64)
        rows = range(n - window if 0 < window < n else 0, n)
        for i in rows:
            at = torch.tensor(list(range(lens[s])) + [lens[s] + j for j in seen[s][i]], dtype=torch.long)
            if len(at) == 0:
                continue
            for h in range(heads):
                k, x = K[at, h // group], q[cu[s] + i, h].to(F64)
                w = torch.softmax(k @ x * scale, 0)
                es = float((k.abs() @ x.abs()).max()) * abs(scale) * (dim + 4) * 2.0 ** -24
                total[h // group, at] += w
                slack[h // group, at] += w * (2.4 * es + (len(at) + 64) * 2.0 ** -23) + 2.0 ** -120
        first = torch.where(torch.arange(keys) < b, decay * out[s, :, :keys], 0.0)
        out[s, :, :keys] = first + total
        tol[s, :, :keys] = slack + (len(rows) * group + 4) * 2.0 ** -24 * (first.abs() + total) + 2.0 ** -126
    return out, tol


def eviction(score, lens, page, table, pages, keep, most, first, last):
    """kept, new_len: lists of each [layer][sequence][kv head]'s kept key numbers (None: as it
    is).  score [layers, seqs, kv, room]."""
    layers, seqs, kv, room = score.shape
    kept = [[[None] * kv for _ in range(seqs)] for _ in range(layers)]
    new_len = list(lens)
    for s, n in enumerate(lens):
        b = most if keep is None else min(keep[s], most)
        if b < 0 or n <= b or n > room or n > table.shape[1] * page:
            continue
        held = table[s, :-(-n // page)]
        if ((held < 0) | (held >= pages)).any():
            continue
        new_len[s] = b
        f = min(first, b)
        t = min(last, b - f)
        for lyr in range(layers):
            for h in range(kv):
                x = score[lyr, s, h, :n].to(F64)
                x = torch.where(torch.isnan(x), -math.inf, x).tolist()
                nan = torch.isnan(score[lyr, s, h, :n]).tolist()
                among = sorted(range(f, n - t), key=lambda i: (nan[i], -x[i], i))[:b - f - t]
                kept[lyr][s][h] = sorted([*range(f), *among, *range(n - t, n)])
    return kept, new_len
