"""Operators of serving from a paged cache, as cases that can be timed.

A serving loop with drafted tokens runs five operators around the quantized
linears, all over one paged KV cache [layers][pages][kv heads][page][head dim]
and its table of pages [sequences][pages of a sequence]:

 * plan:   positions, cache slots and ancestor masks of a tree of drafted rows;
 * append: RMS norm of every query and key head, the position rotation, and the
           keys and values written into their pages;
 * attend: attention of the new rows (one token, a tree, a prompt) over the
           cached keys and over each other;
 * commit: the walk down the tree by the model's own tokens, and the accepted
           rows' keys and values moved behind the context in every layer;
 * copy:   pages copied in every layer (forks, copy on write, compaction).

`run` computes each in its plain form (torch operations in 32 bits), or, where
`own` is true, through `plugins_amd.paged`.  Shapes are those of the decoder
that this repository times (32 query and 8 kv heads of 128, 36 layers), of its
tests (8 and 2 heads), and others of the same ranges.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # The tree of one sequence: 60 drafted rows behind a context of 2048.
        {"name": "plan_1", "kind": "plan", "seqs": 1, "rows": 60, "ctx": 2048, "page": 64},
        # Trees of a full serving batch.
        {"name": "plan_128", "kind": "plan", "seqs": 128, "rows": 64, "ctx": 8192, "page": 16},
        # One new token for each of 8 sequences.
        {"name": "append_8", "kind": "append", "seqs": 8, "rows": 1, "ctx": 2048, "kv": 8,
         "group": 4, "dim": 128, "page": 64, "dtype": "f16"},
        # Three ragged prompts, the longest of 2048 tokens, the last far into its context.
        {"name": "append_prompt", "kind": "append", "seqs": 3, "rows": 2048, "ctx": 100000,
         "kv": 8, "group": 4, "dim": 128, "page": 64, "dtype": "bf16"},
        # The next token of one sequence: the smallest attention, all latency.
        {"name": "attend_1", "kind": "attend", "seqs": 1, "rows": 1, "ctx": 2048, "kv": 8,
         "group": 4, "dim": 128, "page": 64, "dtype": "f16", "tree": False},
        # Trees of up to 64 drafted rows over 16 ragged contexts.
        {"name": "attend_tree_16", "kind": "attend", "seqs": 16, "rows": 64, "ctx": 8192, "kv": 8,
         "group": 4, "dim": 128, "page": 64, "dtype": "bf16", "tree": True},
        # Small trees over long contexts: the cache's bytes are what counts.
        {"name": "attend_long_4", "kind": "attend", "seqs": 4, "rows": 8, "ctx": 65536, "kv": 8,
         "group": 4, "dim": 128, "page": 64, "dtype": "f16", "tree": True},
        # Ragged prompts in one pass, some with a cached prefix: the largest product.
        {"name": "attend_prompt", "kind": "attend", "seqs": 3, "rows": 2048, "ctx": 2048, "kv": 8,
         "group": 4, "dim": 128, "page": 64, "dtype": "bf16", "tree": False},
        # One sequence's tree verified: 4 accepted rows moved in 36 layers.
        {"name": "commit_1", "kind": "commit", "seqs": 1, "rows": 24, "accept": 4, "ctx": 512,
         "layers": 36, "kv": 8, "dim": 128, "page": 64, "dtype": "f16"},
        # A batch's trees verified.
        {"name": "commit_32", "kind": "commit", "seqs": 32, "rows": 64, "accept": 8, "ctx": 256,
         "layers": 36, "kv": 8, "dim": 128, "page": 64, "dtype": "bf16"},
        # A fork's one partial page, copied in 36 layers.
        {"name": "copy_1", "kind": "copy", "count": 1, "pages": 24, "layers": 36, "kv": 8,
         "dim": 128, "page": 64, "dtype": "f16"},
        # A compaction of the pool: 200 pages move.
        {"name": "copy_200", "kind": "copy", "count": 200, "pages": 512, "layers": 8, "kv": 8,
         "dim": 128, "page": 64, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["plan", "append", "append", "attend", "attend", "attend", "attend",
                       "commit", "copy"])
    page = rng.choice([16, 32, 64, 64, 128, 256])
    dtype = rng.choice(["f16", "bf16"])
    dim = rng.choice([64, 128, 128])
    if kind == "plan":
        return {"kind": kind, "seqs": _log_int(rng, 1, 128), "rows": _log_int(rng, 1, 200),
                "ctx": _log_int(rng, 1, 8192), "page": page}
    if kind == "append":
        return {"kind": kind, "seqs": _log_int(rng, 1, 4), "rows": _log_int(rng, 1, 1024),
                "ctx": _log_int(rng, 1, 60000), "kv": rng.choice([1, 2, 4, 8]),
                "group": rng.choice([1, 2, 3, 4, 5, 8]), "dim": dim, "page": page, "dtype": dtype}
    if kind == "attend":
        kv, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 4, 5, 8])
        if rng.random() < 0.65:  # trees, and single tokens
            tree = rng.random() < 0.7
            rows = _log_int(rng, 1, 130) if tree else 1
            seqs = _log_int(rng, 1, 24)
            return {"kind": kind, "seqs": seqs, "rows": rows,
                    "ctx": _log_int(rng, 1, min(60000, 100000 // seqs)), "kv": kv, "group": group,
                    "dim": dim, "page": page, "dtype": dtype, "tree": tree}
        return {"kind": kind, "seqs": rng.randint(1, 3), "rows": _log_int(rng, 30, 1500),
                "ctx": _log_int(rng, 1, 1500), "kv": kv, "group": min(group, 4), "dim": dim,
                "page": page, "dtype": dtype, "tree": False}
    if kind == "commit":
        rows = _log_int(rng, 1, 100)
        return {"kind": kind, "seqs": _log_int(rng, 1, 32), "rows": rows,
                "accept": rng.randint(1, min(rows, 10)), "ctx": _log_int(rng, 1, 256),
                "layers": rng.randint(1, 36), "kv": rng.choice([1, 2, 4, 8]), "dim": dim,
                "page": rng.choice([16, 32, 64]), "dtype": dtype}
    count = _log_int(rng, 1, 200)
    return {"kind": kind, "count": count, "pages": 2 * count + rng.randint(1, 60),
            "layers": rng.randint(1, 8), "kv": rng.choice([1, 2, 4, 8]), "dim": dim,
            "page": rng.choice([16, 32, 64]), "dtype": dtype}


# ------------------------------------------------------------------ their sizes

def _sizes(case):
    """(rows, context) of each sequence: the first has the most rows over the
    longest context, the others are ragged, by the case alone."""
    rng = random.Random("%d %d %d" % (case["seqs"], case["rows"], case["ctx"]))
    n = [case["rows"]] + [rng.randint(1, case["rows"]) for _ in range(case["seqs"] - 1)]
    c = [case["ctx"]] + [rng.randint(0, case["ctx"]) for _ in range(case["seqs"] - 1)]
    return n, c


def _visible(case):
    """Pairs of a row and a key that it sees: a prompt's rows see those before
    them; a tree's row its ancestors, counted as the logarithm of the tree."""
    n, c = _sizes(case)
    pairs = 0.0
    for rows, ctx in zip(n, c):
        pairs += rows * ctx
        pairs += rows * (math.log2(rows) + 1) if case["tree"] else rows * (rows + 1) / 2
    return pairs


def work(case):
    kind = case["kind"]
    if kind == "copy":
        return {"bytes": 2 * case["count"] * case["layers"] * 2 * case["kv"] * case["page"]
                * case["dim"] * 2, "flops": 0}
    n, c = _sizes(case)
    total, seqs = sum(n), case["seqs"]
    if kind == "plan":
        words = -(-max(n) // 64)
        pages = sum(-(-rows // case["page"]) for rows in n)
        return {"bytes": 4 * (2 * seqs + 1) + 4 * pages + total * (4 + 4 + 4 + 8 * words),
                "flops": 0}
    if kind == "append":
        heads = case["kv"] * (case["group"] + 2)
        return {"bytes": total * (2 * heads * case["dim"] * 2 + 8), "flops": 0}
    if kind == "attend":
        keys = sum(rows + ctx for rows, ctx in zip(n, c))
        heads = case["kv"] * case["group"]
        words = -(-max(n) // 64) if case["tree"] else 0
        return {"bytes": 2 * keys * case["kv"] * case["dim"] * 2
                + total * (2 * heads * case["dim"] * 2 + 8 * words),
                "flops": 4 * case["dim"] * heads * _visible(case)}
    moved = sum(min(case["accept"], rows) - 1 for rows in n)
    return {"bytes": 2 * moved * case["layers"] * 2 * case["kv"] * case["dim"] * 2
            + total * 12 + seqs * 20, "flops": 0}


# ------------------------------------------------------------------ inputs

def _trees(n, rng):
    """A parent of each row (an index into its own sequence's rows, -1 for the
    root): recent rows have more children, as drafts that go deep have."""
    out = []
    for rows in n:
        out += [-1] + [int(i * math.sqrt(rng.random())) for i in range(1, rows)]
    return out


def _batch(case, seed):
    """Rows and pages of the sequences: cu, len, and a table whose pages lie in
    the pool in a random order, with pages of others between them."""
    n, c = _sizes(case)
    rng = random.Random("%d" % seed)
    page = case["page"]
    need = [-(-(rows + ctx) // page) for rows, ctx in zip(n, c)]
    pages = sum(need) + 3
    order = list(range(pages))
    rng.shuffle(order)
    most = max(need)
    table = torch.full((len(n), most), -1, dtype=torch.int32)
    at = 0
    for s, k in enumerate(need):
        table[s, :k] = torch.tensor(order[at:at + k], dtype=torch.int32)
        at += k
    cu = [0]
    for rows in n:
        cu.append(cu[-1] + rows)
    i32 = {"dtype": torch.int32, "device": DEV}
    return n, c, rng, pages, {
        "cu": torch.tensor(cu, **i32), "len": torch.tensor(c, **i32), "table": table.to(DEV),
        "max_rows": max(n), "max_keys": max(r + k for r, k in zip(n, c)), "total": cu[-1]}


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(shape, dtype, g):
    return torch.randn(shape, generator=g, device=DEV, dtype=dtype)


def prepare(case, seed):
    kind, g = case["kind"], _gen(seed)
    st = {"kind": kind, "case": case}
    i32 = {"dtype": torch.int32, "device": DEV}
    if kind == "copy":
        dt = DTYPES[case["dtype"]]
        shape = (case["layers"], case["pages"], case["kv"], case["page"], case["dim"])
        st["k"], st["v"] = _randn(shape, dt, g), _randn(shape, dt, g)
        order = list(range(case["pages"]))
        random.Random("%d" % seed).shuffle(order)
        st["src"], st["dst"] = order[:case["count"]], order[case["count"]:2 * case["count"]]
        st["table"] = torch.full((1, 1), -1, **i32)
    else:
        n, c, rng, pages, more = _batch(case, seed)
        st.update(more)
        total, page = st["total"], case["page"]
        st["parent"] = torch.tensor(_trees(n, rng), **i32)
        if kind == "plan":
            words = -(-max(n) // 64)
            shape = (1, pages, 1, page, 64)
            st["k"] = torch.empty(shape, dtype=torch.float16, device=DEV)
            st["v"] = torch.empty_like(st["k"])
            st["pos"], st["slot"] = torch.zeros(total, **i32), torch.zeros(total, **i32)
            st["mask"] = torch.zeros(total, words, dtype=torch.int64, device=DEV)
        else:
            dt, kv, dim = DTYPES[case["dtype"]], case["kv"], case["dim"]
            layers = case.get("layers", 1)
            shape = (layers, pages, kv, page, dim)
            st["k"], st["v"] = _randn(shape, dt, g), _randn(shape, dt, g)
        if kind == "append":
            heads = kv * case["group"]
            # keys and queries of a projection, not of unit size
            st["q"] = 2 * _randn((total, heads * dim), dt, g)
            st["new_k"] = 2 * _randn((total, kv * dim), dt, g)
            st["new_v"] = _randn((total, kv * dim), dt, g)
            st["q_norm"] = (1 + 0.1 * torch.randn(dim, generator=g, device=DEV)).to(dt)
            st["k_norm"] = (1 + 0.1 * torch.randn(dim, generator=g, device=DEV)).to(dt)
            st["pos"], st["slot"], _ = _plan(st, chain=True)
            st["out"] = torch.empty_like(st["q"])
            st["eps"], st["theta"] = 1e-6, 1e6
        elif kind == "attend":
            heads = kv * case["group"]
            st["q"] = _randn((total, heads * dim), dt, g)
            st["out"] = torch.empty_like(st["q"])
            st["mask"] = _plan(st)[2] if case["tree"] else None
            st["scale"] = 1.0 / math.sqrt(dim)
        elif kind == "commit":
            _verified(st, case, n, g, rng)
            shape = (case["seqs"],)
            st["path"] = torch.empty(case["seqs"], max(n), **i32)
            st["count"], st["next"] = torch.empty(shape, **i32), torch.empty(shape, **i32)
            st["new_len"] = torch.empty(shape, **i32)
    if own:  # the handles that a program keeps over the tensors it has
        from plugins_amd import paged as P
        st["cache"] = P.PagedCache.over(st["k"], st["v"], st["table"])
        if kind != "copy":
            st["rows"] = P.Rows(st["cu"], st["len"], st["total"], st["max_rows"])
    return st


def _verified(st, case, n, g, rng):
    """Drafted tokens and the model's own after each row: a path of the case's
    length is what the model would have said, spread over the tree."""
    ids = torch.randint(0, 50000, (st["total"],), generator=g, device=DEV, dtype=torch.int32)
    target = torch.randint(50000, 100000, (st["total"],), generator=g, device=DEV,
                           dtype=torch.int32)
    parent, at = st["parent"].tolist(), 0
    for rows in n:
        take = min(case["accept"], rows)
        path = [0] + sorted(rng.sample(range(1, rows), take - 1))
        for a, b in zip(path, path[1:]):
            parent[at + b] = a
            target[at + a] = ids[at + b]
        at += rows
    st["parent"] = torch.tensor(parent, dtype=torch.int32, device=DEV)
    st["ids"], st["target"] = ids, target


# ------------------------------------------------------------------ one pass

def run(state):
    kind = state["kind"]
    if own:
        from plugins_amd import paged as P
        if kind == "plan":
            P.tree_plan(state["cache"], state["rows"], state["parent"], state["pos"],
                        state["slot"], state["mask"])
        elif kind == "append":
            P.qkv_append(state["cache"], 0, state["q"], state["new_k"], state["new_v"],
                         state["q_norm"], state["k_norm"], state["pos"], state["slot"],
                         state["out"], state["eps"], state["theta"])
        elif kind == "attend":
            P.attend(state["cache"], 0, state["rows"], state["q"], state["out"],
                     mask=state["mask"], scale=state["scale"])
        elif kind == "commit":
            P.commit(state["cache"], state["rows"], state["parent"], state["ids"],
                     state["target"], state["path"], state["count"], state["next"],
                     state["new_len"])
        else:
            P.copy_pages(state["cache"], state["src"], state["dst"])
    elif kind == "plan":
        state["pos"], state["slot"], state["mask"] = _plan(state)
    elif kind == "append":
        _append(state)
    elif kind == "attend":
        _attend(state)
    elif kind == "commit":
        _commit(state)
    else:
        state["k"][:, state["dst"]] = state["k"][:, state["src"]]
        state["v"][:, state["dst"]] = state["v"][:, state["src"]]
    return {x: state[x] for x in _OUTPUTS[kind]}


_OUTPUTS = {"plan": ("pos", "slot", "mask"), "append": ("out", "k", "v"), "attend": ("out",),
            "commit": ("path", "count", "next", "new_len", "k", "v"), "copy": ("k", "v")}


# ------------------------------------------------------------------ plain forms

def _padded(st):
    """Row numbers [S, most rows] and which of them are there."""
    n = (st["cu"][1:] - st["cu"][:-1]).long()
    i = torch.arange(st["max_rows"], device=DEV)
    there = i[None] < n[:, None]
    return n, torch.where(there, st["cu"][:-1, None].long() + i, 0), there


def _slots(st, keys):
    """Pool slots of key numbers [S, any]; -1 where the table has no page."""
    page = st["case"]["page"]
    at = (keys // page).clamp(0, st["table"].shape[1] - 1)
    of = st["table"].gather(1, at).long()
    return torch.where(of < 0, -1, of * page + keys % page)


def _plan(st, chain=False):
    n, row, there = _padded(st)
    most = st["max_rows"]
    i = torch.arange(most, device=DEV)
    up = i - 1 if chain else torch.where(there, st["parent"][row].long(), -1)
    up = up.expand(len(n), most)
    if chain:
        depth, mask = i.expand(len(n), most), None
    else:
        # powers of (I + the parent relation): every ancestor after log2 steps
        sees = torch.eye(most, device=DEV).expand(len(n), most, most).clone()
        sees.scatter_add_(2, up.clamp(min=0)[..., None], (up >= 0).float()[..., None])
        for _ in range(max(0, (most - 1).bit_length())):
            sees = (torch.bmm(sees, sees) > 0).float()
        depth = sees.sum(-1).long() - 1
        words = -(-most // 64)
        bits = torch.zeros(len(n), most, words * 64, dtype=torch.int64, device=DEV)
        bits[..., :most] = sees.long()
        weight = torch.ones(64, dtype=torch.int64, device=DEV) << torch.arange(64, device=DEV)
        mask = (bits.view(len(n), most, words, 64) * weight).sum(-1)[there]
    pos = (st["len"][:, None].long() + depth)[there].int()
    return pos, _slots(st, st["len"][:, None].long() + i)[there].int(), mask


def _turn(x, w, pos, eps, theta):
    """[T, heads, D] in 32 bits: RMS norm, then the rotation of its halves."""
    dim = x.shape[-1]
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w.float()
    rate = theta ** (torch.arange(dim // 2, device=DEV, dtype=torch.float64) * (-2.0 / dim))
    angle = pos.double()[:, None, None] * rate
    c, s = torch.cos(angle).float(), torch.sin(angle).float()
    a, b = x[..., :dim // 2], x[..., dim // 2:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _append(st):
    case, total = st["case"], st["total"]
    kv, dim, page = case["kv"], case["dim"], case["page"]
    dt = st["q"].dtype
    st["out"] = _turn(st["q"].view(total, -1, dim), st["q_norm"], st["pos"], st["eps"],
                      st["theta"]).to(dt).view(total, -1)
    k = _turn(st["new_k"].view(total, kv, dim), st["k_norm"], st["pos"], st["eps"], st["theta"])
    slot = st["slot"].long()
    st["k"][0, slot // page, :, slot % page] = k.to(dt)
    st["v"][0, slot // page, :, slot % page] = st["new_v"].view(total, kv, dim)


def _attend(st):
    case = st["case"]
    kv, group, dim, page = case["kv"], case["group"], case["dim"], case["page"]
    n, row, there = _padded(st)
    seqs, most, keys = len(n), st["max_rows"], st["max_keys"]
    key = torch.arange(keys, device=DEV).expand(seqs, keys)
    slot = _slots(st, key).clamp(min=0)
    k = st["k"][0, slot // page, :, slot % page].float()  # [S, keys, kv, D]
    v = st["v"][0, slot // page, :, slot % page].float()
    q = st["q"][row].float().view(seqs, most, kv, group, dim)
    q = q.permute(0, 2, 1, 3, 4).reshape(seqs * kv, most * group, dim)
    k = k.permute(0, 2, 3, 1).reshape(seqs * kv, dim, keys).contiguous()
    v = v.permute(0, 2, 1, 3).reshape(seqs * kv, keys, dim).contiguous()
    j = key - st["len"][:, None].long()  # a key's row among the new ones
    if st["mask"] is None:
        new = j[:, None] <= torch.arange(most, device=DEV)[:, None]
    else:
        word = st["mask"][row].gather(2, (j.clamp(min=0, max=most - 1) // 64)[:, None]
                                      .expand(seqs, most, keys))
        new = ((word >> (j.clamp(min=0) % 64)[:, None]) & 1).bool()
    sees = (j < 0)[:, None] | (new & ((j >= 0) & (j < n[:, None]))[:, None])  # [S, rows, keys]
    sees = sees[:, None, :, None].expand(seqs, kv, most, group, keys).reshape(
        seqs * kv, most * group, keys)
    s = torch.bmm(q, k) * st["scale"]
    s = torch.where(sees, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.where(sees, torch.exp(s - torch.where(top == -math.inf, 0.0, top)), 0.0)
    o = torch.bmm(p, v) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    o = o.view(seqs, kv, most, group, dim).permute(0, 2, 1, 3, 4).reshape(seqs, most, -1)
    st["out"][row[there]] = o[there].to(st["out"].dtype)


def _commit(st):
    page = st["case"]["page"]
    n, row, there = _padded(st)
    seqs, most = len(n), st["max_rows"]
    up = torch.where(there, st["parent"][row].long(), -2)
    ids, target = st["ids"][row], st["target"][row]
    here = torch.zeros(seqs, dtype=torch.long, device=DEV)
    live = n > 0
    path = torch.full((seqs, most), -1, dtype=torch.long, device=DEV)
    path[:, 0] = torch.where(live, 0, -1)
    said = target.gather(1, here[:, None])[:, 0]
    for step in range(1, most):
        fits = (up == here[:, None]) & (ids == said[:, None]) & live[:, None]
        live = fits.any(-1)
        here = torch.where(live, fits.int().argmax(-1), here)
        path[:, step] = torch.where(live, here, -1)
        said = torch.where(live, target.gather(1, here[:, None])[:, 0], said)
    count = (path >= 0).sum(-1)
    st["path"], st["count"] = path.int(), count.int()
    st["next"] = torch.where(n > 0, said, -1).int()
    st["new_len"] = (st["len"] + count).int()
    moved = path >= 0
    base = st["len"][:, None].long()
    src = _slots(st, base + path.clamp(min=0))[moved]
    dst = _slots(st, base + torch.arange(most, device=DEV))[moved]
    st["k"][:, dst // page, :, dst % page] = st["k"][:, src // page, :, src % page]
    st["v"][:, dst // page, :, dst % page] = st["v"][:, src // page, :, src % page]


# ------------------------------------------------------------------ 64 bits

def exact(case, seed):
    kind = case["kind"]
    if kind == "plan":  # whole numbers alone
        return None
    st = prepare(case, seed)
    if kind == "copy":
        k, v = st["k"].double(), st["v"].double()
        for a, b in zip(st["src"], st["dst"]):
            k[:, b], v[:, b] = st["k"][:, a].double(), st["v"][:, a].double()
        return {"k": k, "v": v}
    page, cu, lens = case["page"], st["cu"].tolist(), st["len"].tolist()
    table = st["table"].tolist()

    def slot(s, key):
        return table[s][key // page] * page + key % page

    if kind == "append":
        dim, kv = case["dim"], case["kv"]
        at = [lens[s] + i for s in range(case["seqs"]) for i in range(cu[s + 1] - cu[s])]
        to = torch.tensor([slot(s, lens[s] + i) for s in range(case["seqs"])
                           for i in range(cu[s + 1] - cu[s])], device=DEV)
        half = torch.arange(dim // 2, device=DEV, dtype=torch.float64)
        angle = torch.outer(torch.tensor(at, device=DEV, dtype=torch.float64),
                            torch.exp(-2.0 * half / dim * math.log(st["theta"])))
        turn = torch.polar(torch.ones_like(angle), angle)[:, None]

        def heads(x, w):
            x = x.double().view(len(at), -1, dim)
            x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / dim + st["eps"]) * w.double()
            z = torch.complex(x[..., :dim // 2].contiguous(), x[..., dim // 2:].contiguous()) * turn
            return torch.cat([z.real, z.imag], -1)

        k, v = st["k"].double(), st["v"].double()
        k[0, to // page, :, to % page] = heads(st["new_k"], st["k_norm"])
        v[0, to // page, :, to % page] = st["new_v"].double().view(len(at), kv, dim)
        return {"out": heads(st["q"], st["q_norm"]).reshape(len(at), -1), "k": k, "v": v}
    if kind == "attend":
        dim, kv, group = case["dim"], case["kv"], case["group"]
        out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
        parent = st["parent"].tolist()
        for s in range(case["seqs"]):
            rows, ctx = cu[s + 1] - cu[s], lens[s]
            of = torch.tensor([slot(s, x) for x in range(ctx + rows)], device=DEV)
            hide = torch.zeros(rows, ctx + rows, dtype=torch.bool)
            if case["tree"]:
                hide[:, ctx:] = True
                for i in range(rows):
                    j = i
                    while j >= 0:
                        hide[i, ctx + j] = False
                        j = parent[cu[s] + j]
            else:
                hide[:, ctx:] = torch.ones(rows, rows).triu(1).bool()
            hide = hide.to(DEV)
            for h in range(kv * group):
                k = st["k"][0, of // page, h // group, of % page].double()
                v = st["v"][0, of // page, h // group, of % page].double()
                q = st["q"][cu[s]:cu[s + 1], h * dim:(h + 1) * dim].double()
                p = torch.softmax((q @ k.T * st["scale"]).masked_fill(hide, -math.inf), -1)
                out[cu[s]:cu[s + 1], h * dim:(h + 1) * dim] = p @ v
        return {"out": out}
    k, v = st["k"].double(), st["v"].double()
    parent, ids, target = st["parent"].tolist(), st["ids"].tolist(), st["target"].tolist()
    for s in range(case["seqs"]):
        path = [0]
        while True:
            said = target[cu[s] + path[-1]]
            to = [j for j in range(cu[s + 1] - cu[s])
                  if parent[cu[s] + j] == path[-1] and ids[cu[s] + j] == said]
            if not to:
                break
            path.append(to[0])
        for j, i in enumerate(path):
            a, b = slot(s, lens[s] + i), slot(s, lens[s] + j)
            k[:, b // page, :, b % page] = st["k"][:, a // page, :, a % page].double()
            v[:, b // page, :, b % page] = st["v"][:, a // page, :, a % page].double()
    return {"path": None, "count": None, "next": None, "new_len": None, "k": k, "v": v}
