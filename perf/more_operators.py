"""Operators of a paged cache that samples its drafted tokens and keeps a budget
of keys, as cases that can be timed.

Beside the operators of `perf/operators.py` a serving loop runs three more:

 * verify: drafted tokens (lines and trees) against the target's probabilities,
           from given random numbers: what is accepted has the target's
           distribution, and a token is sampled where the walk ends.  Without
           drafted rows it is the sampler of a decode step;
 * weigh:  the attention weight that every cached key gets from a step's rows,
           added to what it had (keys [sequences][kv heads][room]);
 * evict:  of each layer's and kv head's keys those of most weight stay, up to a
           budget, in their order; keys and values move together in their pages.

`run` computes each in its plain form (torch operations in 32 bits; the walk and
what is sampled in 64, since they lie next to borders), or, where `own` is true,
through `plugins_amd.paged`.  Shapes are those of the decoder that this
repository times (vocabulary 151936, 32 query and 8 kv heads of 128, 36 layers)
and others of the same ranges.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # The next token of one sequence, sampled: the smallest call, all latency.
        {"name": "verify_1", "kind": "verify", "seqs": 1, "rows": 1, "tree": False, "draft": "",
         "distinct": False, "vocab": 151936, "dtype": "f16"},
        # Lines of up to 5 rows of 8 sequences, drawn from a draft model.
        {"name": "verify_line_8", "kind": "verify", "seqs": 8, "rows": 5, "tree": False,
         "draft": "f32", "distinct": False, "vocab": 151936, "dtype": "f16"},
        # Trees whose siblings were drawn without replacement.
        {"name": "verify_tree_4", "kind": "verify", "seqs": 4, "rows": 24, "tree": True,
         "draft": "f16", "distinct": True, "vocab": 151936, "dtype": "f16"},
        # A full batch's trees of a draft's most likely tokens: the most logits.
        {"name": "verify_tree_64", "kind": "verify", "seqs": 64, "rows": 64, "tree": True,
         "draft": "", "distinct": False, "vocab": 151936, "dtype": "bf16"},
        # One new token of one sequence over 2048 keys.
        {"name": "weigh_1", "kind": "weigh", "seqs": 1, "rows": 1, "ctx": 2048, "kv": 8, "group": 4,
         "dim": 128, "page": 64, "dtype": "f16", "tree": False, "window": 0, "decay": 1.0, "pad": 0},
        # One new token of each of 64 ragged sequences: the cache's bytes.
        {"name": "weigh_64", "kind": "weigh", "seqs": 64, "rows": 1, "ctx": 8192, "kv": 8, "group": 4,
         "dim": 128, "page": 64, "dtype": "bf16", "tree": False, "window": 0, "decay": 0.95, "pad": 0},
        # The last 32 rows of two prompts observe long contexts.
        {"name": "weigh_window", "kind": "weigh", "seqs": 2, "rows": 2048, "ctx": 30000, "kv": 8,
         "group": 4, "dim": 128, "page": 64, "dtype": "f16", "tree": False, "window": 32,
         "decay": 1.0, "pad": 0},
        # Every row of ragged prompts: the largest product.
        {"name": "weigh_prompt", "kind": "weigh", "seqs": 3, "rows": 2048, "ctx": 2048, "kv": 8,
         "group": 4, "dim": 128, "page": 64, "dtype": "bf16", "tree": False, "window": 0,
         "decay": 1.0, "pad": 0},
        # One sequence a little over its budget, in 36 layers.
        {"name": "evict_1", "kind": "evict", "seqs": 1, "ctx": 1100, "keep": 1024, "first": 4,
         "last": 256, "layers": 36, "kv": 8, "dim": 128, "page": 64, "dtype": "f16", "pad": 0},
        # A long prompt brought down to 2048 keys: the scores count too.
        {"name": "evict_prompt", "kind": "evict", "seqs": 1, "ctx": 32768, "keep": 2048, "first": 4,
         "last": 32, "layers": 8, "kv": 8, "dim": 128, "page": 64, "dtype": "bf16", "pad": 0},
        # A batch halved: the keys' and values' bytes.
        {"name": "evict_16", "kind": "evict", "seqs": 16, "ctx": 4096, "keep": 2048, "first": 4,
         "last": 256, "layers": 8, "kv": 8, "dim": 128, "page": 64, "dtype": "f16", "pad": 0},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["verify", "verify", "weigh", "weigh", "weigh", "evict", "evict"])
    if kind == "verify":
        tree = rng.random() < 0.6
        draft = rng.choice(["", "f32", "f16", "bf16"])
        rows = _log_int(rng, 1, 64 if tree else 16)
        return {"kind": kind, "seqs": _log_int(rng, 1, 48 if not draft else 12), "rows": rows,
                "tree": tree, "draft": draft, "distinct": tree and rng.random() < 0.5,
                "vocab": _log_int(rng, 700, 152000), "dtype": rng.choice(["f16", "bf16", "f32"])}
    page = rng.choice([16, 32, 64, 64, 128, 256])
    dtype = rng.choice(["f16", "bf16"])
    dim, kv = rng.choice([64, 128, 128]), rng.choice([1, 2, 4, 8])
    pad = rng.choice([0, 0, 1, 6])
    if kind == "weigh":
        case = {"kind": kind, "kv": kv, "group": rng.choice([1, 2, 3, 4, 4, 5, 8]), "dim": dim,
                "page": page, "dtype": dtype, "decay": rng.choice([1.0, 0.9]), "pad": pad}
        x = rng.random()
        if x < 0.6:  # single tokens and trees
            tree = rng.random() < 0.5
            seqs = _log_int(rng, 1, 48)
            return {**case, "seqs": seqs, "rows": _log_int(rng, 1, 70) if tree else 1,
                    "ctx": _log_int(rng, 1, min(60000, 160000 // seqs)), "tree": tree, "window": 0}
        if x < 0.8:  # windows
            return {**case, "seqs": rng.randint(1, 3), "rows": _log_int(rng, 1, 1500),
                    "ctx": _log_int(rng, 1, 24000), "tree": False, "window": _log_int(rng, 1, 64)}
        return {**case, "group": min(case["group"], 4), "seqs": rng.randint(1, 3),
                "rows": _log_int(rng, 30, 1500), "ctx": _log_int(rng, 1, 1500), "tree": False,
                "window": 0}
    seqs, layers = _log_int(rng, 1, 24), rng.randint(1, 8)
    ctx = _log_int(rng, 40, 60000 // seqs)
    keep = _log_int(rng, 1, ctx)
    return {"kind": kind, "seqs": seqs, "ctx": ctx, "keep": keep,
            "first": rng.choice([0, 4, 4]), "last": rng.choice([0, 32, keep // 4]),
            "layers": layers, "kv": kv, "dim": dim, "page": page, "dtype": dtype, "pad": pad}


# ------------------------------------------------------------------ their sizes

def _sizes(case):
    """(rows, context) of each sequence: the first has the most rows over the
    longest context, the others are ragged, by the case alone."""
    rows, ctx = case.get("rows", 0), case.get("ctx", 0)
    rng = random.Random("%d %d %d" % (case["seqs"], rows, ctx))
    n = [rows] + [rng.randint(min(1, rows), rows) for _ in range(case["seqs"] - 1)]
    c = [ctx] + [rng.randint(0, ctx) for _ in range(case["seqs"] - 1)]
    return n, c


def _watching(rows, case):
    """Rows of a sequence whose weights count."""
    return min(rows, case["window"]) if case["window"] else rows


def work(case):
    kind = case["kind"]
    n, c = _sizes(case)
    total, seqs = sum(n), case["seqs"]
    if kind == "verify":
        # every row's logits, and of the drafts those of the row where a walk ends:
        # without knowing where it will, what one pass over the inputs reads
        size = DTYPES[case["dtype"]].itemsize
        drafted = DTYPES[case["draft"]].itemsize * seqs if case["draft"] else 0
        return {"bytes": case["vocab"] * (total * size + drafted) + total * 20 + seqs * 8, "flops": 0}
    if kind == "weigh":
        dim, kv, group = case["dim"], case["kv"], case["group"]
        keys = sum(rows + ctx for rows, ctx in zip(n, c))
        seen = watch = 0.0
        for rows, ctx in zip(n, c):
            w = _watching(rows, case)
            watch += w
            seen += w * ctx
            seen += w * (math.log2(rows) + 1) if case["tree"] else w * (rows - (w - 1) / 2)
        words = -(-max(n) // 64) if case["tree"] else 0
        return {"bytes": keys * kv * dim * 2 + 2 * keys * kv * 4
                + watch * (kv * group * dim * 2 + 8 * words),
                "flops": 2 * dim * kv * group * seen}
    bytes_ = 0
    for ctx in c:
        bytes_ += 4 * case["keep"]
        if ctx > case["keep"]:
            still = case["first"] + max(0, ctx - case["first"] - case["last"]) // (ctx - case["keep"] + 1)
            moved = max(0, case["keep"] - still)
            bytes_ += 4 * ctx + 4 * case["keep"] + moved * 2 * 2 * case["dim"] * 2
    return {"bytes": bytes_ * case["layers"] * case["kv"] + 8 * seqs, "flops": 0}


# ------------------------------------------------------------------ inputs

def _trees(n, rng):
    """A parent of each row (an index into its own sequence's rows, -1 for the
    root): recent rows have more children, as drafts that go deep have."""
    out = []
    for rows in n:
        out += [-1][:rows] + [int(i * math.sqrt(rng.random())) for i in range(1, rows)]
    return out


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(shape, dtype, g):
    return torch.randn(shape, generator=g, device=DEV, dtype=dtype)


def _rows(st, n, c):
    cu = [0]
    for rows in n:
        cu.append(cu[-1] + rows)
    i32 = {"dtype": torch.int32, "device": DEV}
    st.update(cu=torch.tensor(cu, **i32), len=torch.tensor(c, **i32), total=cu[-1], max_rows=max(n),
              max_keys=max(r + k for r, k in zip(n, c)))


def _pages(st, case, n, c, rng):
    """A table whose pages lie in the pool in a random order, with pages of others
    between them, and the keys that a sequence's scores have room for."""
    page = case["page"]
    need = [-(-(rows + ctx) // page) for rows, ctx in zip(n, c)]
    pages = sum(need) + 3
    order = list(range(pages))
    rng.shuffle(order)
    most = max(need + [1])
    table = torch.full((len(n), most), -1, dtype=torch.int32)
    at = 0
    for s, k in enumerate(need):
        table[s, :k] = torch.tensor(order[at:at + k], dtype=torch.int32)
        at += k
    st["table"], st["room"] = table.to(DEV), most * page + case["pad"]
    return pages


def prepare(case, seed):
    kind, g = case["kind"], _gen(seed)
    st = {"kind": kind, "case": case}
    n, c = _sizes(case)
    rng = random.Random("%d" % seed)
    _rows(st, n, c)
    if kind == "verify":
        _drafted(st, case, n, g, rng)
        if own:
            from plugins_amd import paged as P
            st["rows"] = P.Rows(st["cu"], st["len"], st["total"], st["max_rows"])
        return st
    pages = _pages(st, case, n, c, rng)
    dt, kv, dim, layers = DTYPES[case["dtype"]], case["kv"], case["dim"], case.get("layers", 1)
    shape = (layers, pages, kv, case["page"], dim)
    st["k"] = _randn(shape, dt, g)
    # what keys have gathered so far: a few have most of it
    st["score"] = torch.empty(layers, case["seqs"], kv, st["room"], device=DEV).log_normal_(
        -1.0, 1.5, generator=g)
    if kind == "weigh":
        st["v"] = torch.empty_like(st["k"])  # not read
        heads = kv * case["group"]
        st["q"] = _randn((st["total"], heads * dim), dt, g)
        st["scale"] = 1.0 / math.sqrt(dim)
        st["parent"] = torch.tensor(_trees(n, rng), dtype=torch.int32, device=DEV)
        st["mask"] = _masks(st) if case["tree"] else None
    else:
        st["v"] = _randn(shape, dt, g)
        i32 = {"dtype": torch.int32, "device": DEV}
        st["kept"] = torch.empty(layers, case["seqs"], kv, case["keep"], **i32)
        st["new_score"] = torch.zeros_like(st["score"])
        st["new_len"] = torch.empty(case["seqs"], **i32)
    if own:  # the handles that a program keeps over the tensors it has
        from plugins_amd import paged as P
        st["cache"] = P.PagedCache.over(st["k"], st["v"], st["table"])
        st["rows"] = P.Rows(st["cu"], st["len"], st["total"], st["max_rows"])
    return st


def _drafted(st, case, n, g, rng):
    """Logits of a target whose mass lies on a few tokens, a draft that is near it,
    and tokens from the draft: drawn (siblings with or without replacement) where
    its probabilities are given, its most likely ones in a random order where they
    are not.  Some sequences are greedy."""
    T, V, S = st["total"], case["vocab"], case["seqs"]
    dt = DTYPES[case["dtype"]]
    parent = torch.tensor(_trees(n, rng), dtype=torch.int32, device=DEV)
    if not case["tree"]:
        parent = torch.cat([torch.arange(-1, rows - 1, dtype=torch.int32, device=DEV) for rows in n])
    temp = torch.tensor([rng.choice([0.0, 0.6, 0.8, 1.0, 1.0, 1.3]) if s else 0.9 for s in range(S)],
                        device=DEV)
    first = st["cu"][:-1].long()
    of = torch.repeat_interleave(torch.arange(S, device=DEV), torch.tensor(n, device=DEV))
    up = first[of] + parent.clamp(min=0).long()  # a row's parent in the step's tensors
    likely = torch.randint(0, V, (T, 24), generator=g, device=DEV)
    top = 4 + 9 * torch.rand(T, 24, generator=g, device=DEV)
    z = _randn((T, V), dt, g)
    z.scatter_(1, likely, top.to(dt))
    near = top + 0.7 * torch.randn(T, 24, generator=g, device=DEV)  # the draft's view of them
    heat = temp[of].clamp(min=0.5)[:, None]
    seen, number = {}, []  # a row's number among its siblings
    for x in up.tolist():
        number.append(seen.get(x, 0))
        seen[x] = number[-1] + 1
    num = torch.tensor(number, device=DEV)
    gumbel = -torch.log(torch.empty(T, 24, device=DEV).exponential_(generator=g))
    if case["draft"] and not case["distinct"]:
        pick = (near / heat)[up] + gumbel  # every row its own draw
        rank = torch.zeros_like(num)
    else:
        pick = ((near / heat) + gumbel)[up]  # siblings share one: its order
        rank = num % 24
    ids = likely[up].gather(1, pick.argsort(-1, descending=True).gather(1, rank[:, None]))[:, 0]
    st.update(logits=z, parent=parent if case["tree"] else None, up=parent, ids=ids.int(), temp=temp,
              u=torch.rand(T, generator=g, device=DEV, dtype=torch.float64), of=of,
              target=torch.empty(T, dtype=torch.int32, device=DEV), draft=None)
    if case["draft"]:
        q = torch.randn(T, V, generator=g, device=DEV)
        q.scatter_(1, likely, near)
        st["draft"] = torch.softmax(q / heat, -1).to(DTYPES[case["draft"]])


def _masks(st):
    """Ancestor masks of the rows' trees, 64-bit words."""
    n, row, there = _padded(st)
    most = st["max_rows"]
    up = torch.where(there, st["parent"][row].long(), -1)
    sees = torch.eye(most, device=DEV).expand(len(n), most, most).clone()
    sees.scatter_add_(2, up.clamp(min=0)[..., None], (up >= 0).float()[..., None])
    for _ in range(max(0, (most - 1).bit_length())):
        sees = (torch.bmm(sees, sees) > 0).float()
    words = -(-most // 64)
    bits = torch.zeros(len(n), most, words * 64, dtype=torch.int64, device=DEV)
    bits[..., :most] = sees.long()
    weight = torch.ones(64, dtype=torch.int64, device=DEV) << torch.arange(64, device=DEV)
    return (bits.view(len(n), most, words, 64) * weight).sum(-1)[there].contiguous()


# ------------------------------------------------------------------ one pass

def run(state):
    kind, case = state["kind"], state["case"]
    if own:
        from plugins_amd import paged as P
        if kind == "verify":
            P.verify(state["rows"], state["parent"], state["ids"], state["logits"], state["u"],
                     state["target"], draft=state["draft"], temperature=state["temp"],
                     distinct=case["distinct"])
        elif kind == "weigh":
            P.weigh(state["cache"], 0, state["rows"], state["q"], state["score"][0],
                    mask=state["mask"], scale=state["scale"], window=case["window"],
                    decay=case["decay"])
        else:
            P.evict(state["cache"], state["len"], state["score"], state["kept"], state["new_score"],
                    state["new_len"], first=case["first"], last=case["last"])
    elif kind == "verify":
        _verify(state)
    elif kind == "weigh":
        _weigh(state)
    else:
        _evict(state)
    return {x: state[x] for x in _OUTPUTS[kind]}


_OUTPUTS = {"verify": ("target",), "weigh": ("score",),
            "evict": ("k", "v", "kept", "new_score", "new_len")}


# ------------------------------------------------------------------ plain forms

def _padded(st):
    """Row numbers [S, most rows] and which of them are there."""
    n = (st["cu"][1:] - st["cu"][:-1]).long()
    i = torch.arange(st["max_rows"], device=DEV)
    there = i[None] < n[:, None]
    return n, torch.where(there, st["cu"][:-1, None].long() + i, 0), there


def _slots(st, keys):
    """Pool slots of key numbers [..., any] of the sequences (dim 0 of table); -1
    where the table has no page."""
    page = st["case"]["page"]
    at = (keys // page).clamp(0, st["table"].shape[1] - 1)
    of = st["table"].gather(1, at).long()
    return torch.where(of < 0, -1, of * page + keys % page)


def _verify(st):
    case, z, q = st["case"], st["logits"], st["draft"]
    V, temp = case["vocab"], st["temp"].double()
    n, row, there = _padded(st)
    seqs = len(n)
    greedy = temp == 0
    # every row's largest logit, where it is, and the sum of its weights
    zf = z.float()
    top = zf.amax(-1)
    best = torch.where(zf == top[:, None], torch.arange(V, device=DEV, dtype=torch.int32), V).amin(-1)
    heat = torch.where(greedy, 1.0, temp)
    mass = torch.exp((zf - top[:, None]) / heat.float()[st["of"]][:, None]).sum(-1, dtype=torch.float64)
    # every row's token among its parent's
    up = st["up"][row].long()
    by = row.gather(1, up.clamp(min=0))
    ids = st["ids"][row].long()
    p = torch.exp((zf[by, ids].double() - top[by].double()) / heat[:, None]) / mass[by]
    u = st["u"][row]
    said = q[by, ids].double() if q is not None else torch.ones_like(p)
    if q is None:  # a token that a sibling before it had is not there any more
        same = (up[:, :, None] == up[:, None]) & (ids[:, :, None] == ids[:, None]) & there[:, None]
        p = torch.where(same.tril(-1).any(-1), 0.0, p)
    at = torch.zeros(seqs, dtype=torch.long, device=DEV)
    one = torch.ones(seqs, dtype=torch.float64, device=DEV)
    left, drawn, taken = one, one, torch.zeros_like(one)  # what p has left, what q has, q's share
    target = torch.full_like(st["target"], -1)
    siblings = case["tree"] and q is not None
    for i in range(1, st["max_rows"]):  # children come behind their parents
        test = there[:, i] & (up[:, i] == at)
        if q is None:
            hit = u[:, i] * left < p[:, i]
            less = left - p[:, i]
        else:
            rate = left / drawn.clamp(min=2.0 ** -53)
            hit = u[:, i] * rate * said[:, i] < (p[:, i] - taken * said[:, i]).clamp(min=0)
        hit = test & torch.where(greedy, best[by[:, i]] == ids[:, i], hit)
        miss = test & ~hit
        if q is not None:
            taken = torch.where(miss, taken + rate, taken)
            if case["distinct"]:
                drawn = torch.where(miss, drawn - said[:, i], drawn)
            here = row.gather(1, at[:, None])[:, 0]
            if siblings:
                w = torch.exp((zf[here] - top[here, None]) / heat.float()[:, None]) / mass[here, None].float()
                w = (w - taken.float()[:, None] * q[here].float()).clamp(min=0)
                less = w.sum(-1, dtype=torch.float64)
            else:
                less = left
        left = torch.where(miss, less, left)
        here = row.gather(1, at[:, None])[:, 0]
        target[here] = torch.where(hit, ids[:, i].int(), target[here])
        at = torch.where(hit, i, at)
        left, drawn = torch.where(hit, 1.0, left), torch.where(hit, 1.0, drawn)
        taken = torch.where(hit, 0.0, taken)
    # what is left of the last row's probabilities, in 64 bits
    here = row.gather(1, at[:, None])[:, 0]
    w = torch.exp((zf[here].double() - top[here, None].double()) / heat[:, None]) / mass[here, None]
    if q is None:
        child = there & (up == at[:, None]) & (torch.arange(st["max_rows"], device=DEV) > 0)
        gone = torch.zeros(seqs, V + 1, dtype=torch.bool, device=DEV)
        gone.scatter_(1, torch.where(child, ids, V), True)
        r = torch.where(gone[:, :V], 0.0, w)
    else:
        r = (w - taken[:, None] * q[here].double()).clamp(min=0)
    r = torch.where(r.sum(-1, keepdim=True) > 0, r, w)
    c = r.cumsum(-1)
    over = (c > u[:, :1] * c[:, -1:]) & (r > 0)
    v = torch.where(over, torch.arange(V, device=DEV), V).amin(-1)
    target[here] = torch.where(greedy, best[here].long(), v).int()
    st["target"] = target


def _weigh(st):
    case = st["case"]
    kv, group, dim, page = case["kv"], case["group"], case["dim"], case["page"]
    n = (st["cu"][1:] - st["cu"][:-1]).long()
    most, keys, seqs = st["max_rows"], st["max_keys"], case["seqs"]
    if case["window"]:
        most = min(most, case["window"])
    i = torch.arange(most, device=DEV) + (n - most).clamp(min=0)[:, None]  # the rows that count
    there = i < n[:, None]
    row = torch.where(there, st["cu"][:-1, None].long() + i, 0)
    key = torch.arange(keys, device=DEV).expand(seqs, keys)
    slot = _slots(st, key).clamp(min=0)
    k = st["k"][0, slot // page, :, slot % page].float()  # [S, keys, kv, D]
    q = st["q"][row].float().view(seqs, most, kv, group, dim)
    q = q.permute(0, 2, 1, 3, 4).reshape(seqs * kv, most * group, dim)
    k = k.permute(0, 2, 3, 1).reshape(seqs * kv, dim, keys).contiguous()
    j = key - st["len"][:, None].long()  # a key's row among the new ones
    if st["mask"] is None:
        new = j[:, None] <= i[..., None]
    else:
        word = st["mask"][row].gather(2, (j.clamp(min=0, max=st["max_rows"] - 1) // 64)[:, None]
                                      .expand(seqs, most, keys))
        new = ((word >> (j.clamp(min=0) % 64)[:, None]) & 1).bool()
    sees = (j < 0)[:, None] | (new & ((j >= 0) & (j < n[:, None]))[:, None])  # [S, rows, keys]
    sees = (sees & there[..., None])[:, None, :, None].expand(seqs, kv, most, group, keys).reshape(
        seqs * kv, most * group, keys)
    s = torch.bmm(q, k) * st["scale"]
    s = torch.where(sees, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.where(sees, torch.exp(s - torch.where(top == -math.inf, 0.0, top)), 0.0)
    w = (p / p.sum(-1, keepdim=True).clamp(min=1e-30)).sum(1).view(seqs, kv, keys)
    score = st["score"][0, :, :, :keys]
    had = torch.where((j < 0)[:, None], score * case["decay"], 0.0)
    score.copy_(torch.where((j < n[:, None])[:, None], had + w, score))


def _evict(st):
    case = st["case"]
    page, keep, most = case["page"], case["keep"], st["max_keys"]
    key = torch.arange(most, device=DEV)
    lens = st["len"].long()
    full = lens > keep
    first = min(case["first"], keep)
    last = min(case["last"], keep - first)
    # the order that keys stay in: those that stay whatever they weigh, the others
    # by weight (of two alike the earlier), those that are not there
    held = (key < first) | (key >= (lens - last)[:, None])
    rank = torch.where(key >= lens[:, None], 2, torch.where(held, 0, 1))[None, :, None]
    score = st["score"][..., :most]
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices
    order = order.gather(-1, torch.sort(rank.expand_as(score).gather(-1, order), dim=-1, stable=True).indices)
    kept = order[..., :keep].sort(-1).values
    kept = torch.where(full[None, :, None, None], torch.nn.functional.pad(kept, (0, keep - kept.shape[-1])), -1)
    st["kept"], st["new_len"] = kept.int(), torch.where(full, keep, lens).int()
    there = kept >= 0
    moved = st["score"].gather(-1, kept.clamp(min=0))
    st["new_score"][..., :keep] = torch.where(there, moved, st["new_score"][..., :keep])
    lyr, seq, head, to = there.nonzero(as_tuple=True)
    of = kept[there]
    table = st["table"].long()
    a, b = table[seq, of // page], table[seq, to // page]
    for pool in (st["k"], st["v"]):
        pool[lyr, b, head, to % page] = pool[lyr, a, head, of % page]


# ------------------------------------------------------------------ 64 bits

def exact(case, seed):
    kind = case["kind"]
    if kind == "verify":  # whole numbers alone
        return None
    st = prepare(case, seed)
    page, cu, lens = case["page"], st["cu"].tolist(), st["len"].tolist()
    table = st["table"].cpu()

    def slots(s, keys):
        return (table[s, keys // page].long() * page + keys % page).to(DEV)

    if kind == "weigh":
        dim, group = case["dim"], case["group"]
        parent = st["parent"].tolist()
        score = st["score"].double()
        for s in range(case["seqs"]):
            rows, ctx = cu[s + 1] - cu[s], lens[s]
            begin = rows - _watching(rows, case)
            of = slots(s, torch.arange(ctx + rows))
            hide = torch.ones(rows, ctx + rows, dtype=torch.bool)
            hide[:, :ctx] = False
            if case["tree"]:
                for i in range(rows):
                    j = i
                    while j >= 0:
                        hide[i, ctx + j] = False
                        j = parent[cu[s] + j]
            else:
                hide[:, ctx:] = torch.ones(rows, rows).triu(1).bool()
            hide = hide[begin:].to(DEV)
            for h in range(case["kv"]):
                k = st["k"][0, of // page, h, of % page].double()
                total = torch.zeros(ctx + rows, dtype=torch.float64, device=DEV)
                for x in range(h * group, (h + 1) * group):
                    q = st["q"][cu[s] + begin:cu[s + 1], x * dim:(x + 1) * dim].double()
                    total += torch.softmax((q @ k.T * st["scale"]).masked_fill(hide, -math.inf), -1).sum(0)
                score[0, s, h, :ctx] *= case["decay"]
                score[0, s, h, ctx:ctx + rows] = 0.0
                score[0, s, h, :ctx + rows] += total
        return {"score": score}
    keep = case["keep"]
    k, v, new = st["k"].double(), st["v"].double(), st["new_score"].double()
    first = min(case["first"], keep)
    last = min(case["last"], keep - first)
    for s, m in enumerate(lens):
        if m <= keep:
            continue
        to = slots(s, torch.arange(keep))
        for lyr in range(case["layers"]):
            for h in range(case["kv"]):
                x = st["score"][lyr, s, h, :m].double()
                x[:first] = math.inf
                x[m - last:] = math.inf
                at = torch.sort(x, descending=True, stable=True).indices[:keep].sort().values
                of = slots(s, at.cpu())
                new[lyr, s, h, :keep] = st["score"][lyr, s, h, at].double()
                k[lyr, to // page, h, to % page] = st["k"][lyr, of // page, h, of % page].double()
                v[lyr, to // page, h, to % page] = st["v"][lyr, of // page, h, of % page].double()
    return {"k": k, "v": v, "kept": None, "new_score": new, "new_len": None}
