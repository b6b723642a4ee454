"""A Qwen3-8B-shaped decoder decode step around the EXL3 linears.

36 layers, hidden 4096, 32 query / 8 KV heads of 128,
SwiGLU intermediate 12288, vocab 151936; RMSNorm (with per-head q/k norm),
rotate-half RoPE, f16 attention over an f16 KV cache, EXL3 K=4 mul1 weights for
every linear including lm_head; random-initialised weights and caches (no
checkpoints here).  The reference's model plugin runs the same step on MLX
(turboexl3_qwen38/src/direct/attn.zig:133-141, attn_core.zig, linear.zig:65-85,
model.zig; paths relative to /root/reference/plugins/), its linears through the
quant table this library exports.

Every operation runs in libexl3_mi355x.so: the linears through exl3d_linears
(the EXL3 GEMV with the step's norms, SwiGLU and residual adds fused into its
prepare and finish), embedding and attention through the other exl3d_*
harness entries (include/exl3_decoder.h).  PyTorch only allocates the
buffers and supplies the stream.
"""
from __future__ import annotations

import ctypes
import math
from ctypes import c_float, c_int, c_size_t, c_void_p
from dataclasses import dataclass

from . import exl3 as X

HEAD_DIM = 128


@dataclass
class Qwen3Config:
    layers: int = 36
    hidden: int = 4096
    heads: int = 32
    kv_heads: int = 8
    inter: int = 12288
    vocab: int = 151936
    eps: float = 1e-6
    theta: float = 1e6
    k_bits: int = 4

    @property
    def q_dim(self) -> int:
        return self.heads * HEAD_DIM

    @property
    def kv_dim(self) -> int:
        return self.kv_heads * HEAD_DIM


_DEC_SIGS = {
    "exl3d_embed": (c_int, [c_void_p, c_int, c_void_p, c_int, c_void_p, c_void_p, c_void_p]),
    "exl3d_linears": (c_int, [c_void_p, c_int, c_void_p, c_int, c_void_p, c_void_p, c_float, c_void_p,
                              c_void_p, c_void_p, c_void_p, c_void_p]),
    "exl3d_add_rmsnorm": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int, c_float,
                                  c_void_p]),
    "exl3d_qk_norm_rope": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int,
                                   c_int, c_int, c_float, c_float, c_void_p, c_void_p, c_void_p,
                                   c_int, c_void_p]),
    "exl3d_attn_scratch_bytes": (c_size_t, [c_int, c_int, c_int, c_int]),
    "exl3d_attn_decode": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_int,
                                  c_float, c_void_p, c_void_p, c_size_t, c_void_p]),
    "exl3d_attn_decode_rope": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p,
                                       c_int, c_int, c_int, c_float, c_float, c_void_p, c_void_p,
                                       c_int, c_float, c_void_p, c_void_p, c_size_t, c_void_p]),
    "exl3d_attn_splits": (c_int, [c_int, c_int, c_int]),
    "exl3d_attn_heads_per_kv": (c_int, []),
    "exl3d_attn_o": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int,
                             c_int, c_float, c_float, c_void_p, c_void_p, c_int, c_float, c_void_p,
                             c_void_p, c_void_p, c_void_p, c_void_p, c_size_t, c_void_p]),
    "exl3d_silu_mul": (c_int, [c_void_p, c_void_p, c_void_p, c_size_t, c_void_p]),
}
_dec = None


def dec_lib():
    """libexl3_mi355x.so with the exl3d_* signatures set."""
    global _dec
    if _dec is None:
        L = X.lib()
        for name, (res, args) in _DEC_SIGS.items():
            fn = getattr(L, name)
            fn.restype = res
            fn.argtypes = args
        _dec = L
    return _dec


def _ck(rc: int, what: str) -> None:
    if rc != 0:
        raise RuntimeError(f"{what}: HIP error {rc}")


def _p(t) -> int:
    return t.data_ptr()


# ------------------------------------------------------------------ ops

def embed(ids, table, h, ssq=None, stream=None):
    B, H = h.shape
    _ck(dec_lib().exl3d_embed(_p(ids), B, _p(table), H, _p(h), _p(ssq) if ssq is not None else None,
                              X.stream_handle(stream)), "embed")


def linears(ws, x, outs=None, norm_w=None, nssq=None, eps=0.0, up=None, res=None, res_ssq=None,
            stream=None):
    """exl3d_linears: the EXL3 linears ws on x with the decode step's fusions
    (RMSNorm of an f32 residual x, SwiGLU with up, residual finish into res)."""
    n = len(ws)
    wp = (ctypes.POINTER(X.Weight) * n)(*[ctypes.pointer(w) for w in ws])
    op = (c_void_p * n)(*[_p(t) for t in outs]) if outs is not None else None
    opt = lambda t: _p(t) if t is not None else None  # noqa: E731
    rc = dec_lib().exl3d_linears(ctypes.cast(wp, c_void_p), n, _p(x), x.shape[0], opt(norm_w),
                                 opt(nssq), eps, opt(up), opt(res), opt(res_ssq),
                                 ctypes.cast(op, c_void_p) if op is not None else None,
                                 X.stream_handle(stream))
    if rc == -1:
        raise RuntimeError("linears: weights or shapes refused")
    _ck(rc, "linears")


def add_rmsnorm(h, add, w, out, eps, stream=None):
    B, H = h.shape
    _ck(dec_lib().exl3d_add_rmsnorm(_p(h), _p(add) if add is not None else None, _p(w), _p(out), B, H,
                                    eps, X.stream_handle(stream)), "add_rmsnorm")


def qk_norm_rope(q, k, v, qn, kn, pos, qout, kcache, vcache, eps, theta, stream=None):
    B = q.shape[0]
    nq, nkv, tmax = q.shape[1] // HEAD_DIM, k.shape[1] // HEAD_DIM, kcache.shape[2]
    _ck(dec_lib().exl3d_qk_norm_rope(_p(q), _p(k), _p(v), _p(qn), _p(kn), _p(pos), B, nq, nkv, eps,
                                     theta, _p(qout), _p(kcache), _p(vcache), tmax,
                                     X.stream_handle(stream)), "qk_norm_rope")


def attn_scratch_bytes(B, nq, nkv, tmax) -> int:
    return int(dec_lib().exl3d_attn_scratch_bytes(B, nq, nkv, tmax))


def attn_decode(q, kcache, vcache, pos, out, scratch, stream=None):
    B = q.shape[0]
    nq, nkv, tmax = q.shape[1] // HEAD_DIM, kcache.shape[1], kcache.shape[2]
    _ck(dec_lib().exl3d_attn_decode(_p(q), _p(kcache), _p(vcache), _p(pos), B, nq, nkv, tmax,
                                    1.0 / math.sqrt(HEAD_DIM), _p(out), _p(scratch),
                                    scratch.numel() * scratch.element_size(),
                                    X.stream_handle(stream)), "attn_decode")


def attn_decode_rope(q, k, v, qn, kn, pos, kcache, vcache, out, scratch, eps, theta, stream=None):
    """q/k norm + RoPE + KV append + attention in one launch (raw q, k, v)."""
    B = q.shape[0]
    nq, nkv, tmax = q.shape[1] // HEAD_DIM, kcache.shape[1], kcache.shape[2]
    _ck(dec_lib().exl3d_attn_decode_rope(_p(q), _p(k), _p(v), _p(qn), _p(kn), _p(pos), B, nq, nkv,
                                         eps, theta, _p(kcache), _p(vcache), tmax,
                                         1.0 / math.sqrt(HEAD_DIM), _p(out), _p(scratch),
                                         scratch.numel() * scratch.element_size(),
                                         X.stream_handle(stream)), "attn_decode_rope")


def attn_o(q, k, v, qn, kn, pos, kcache, vcache, o, res, res_ssq, att, scratch, eps, theta,
           stream=None):
    """exl3d_attn_o: attn_decode_rope, then res += att @ o^T (residual finish,
    res_ssq its sums of squares per 128 columns); at rows that fit one
    prepare batch o's prepare combines the attention's splits (att is then
    not written)."""
    B = q.shape[0]
    nq, nkv, tmax = q.shape[1] // HEAD_DIM, kcache.shape[1], kcache.shape[2]
    rc = dec_lib().exl3d_attn_o(_p(q), _p(k), _p(v), _p(qn), _p(kn), _p(pos), B, nq, nkv, eps, theta,
                                _p(kcache), _p(vcache), tmax, 1.0 / math.sqrt(HEAD_DIM),
                                ctypes.byref(o), _p(res), _p(res_ssq), _p(att), _p(scratch),
                                scratch.numel() * scratch.element_size(), X.stream_handle(stream))
    if rc == -1:
        raise RuntimeError("attn_o: weight or shapes refused")
    _ck(rc, "attn_o")


def silu_mul(g, u, out, stream=None):
    _ck(dec_lib().exl3d_silu_mul(_p(g), _p(u), _p(out), out.numel(), X.stream_handle(stream)),
        "silu_mul")


# ------------------------------------------------------------------ model

def random_linear(torch, i: int, o: int, k_bits: int, gen):
    """An EXL3 linear with uniform-random trellis words, suh +-1 and
    svh f16(+-U[0.5, 1.5] * 0.02) (BASELINE's synthetic packing)."""
    n = 16 * k_bits
    t = torch.randint(-32768, 32768, (i // 16, o // 16, n), dtype=torch.int32, device="cuda",
                      generator=gen).to(torch.int16)
    suh = (torch.randint(0, 2, (i,), device="cuda", generator=gen) * 2 - 1).to(torch.float16)
    sgn = torch.randint(0, 2, (o,), device="cuda", generator=gen) * 2 - 1
    mag = torch.rand(o, device="cuda", generator=gen) + 0.5
    svh = (sgn * mag * 0.02).to(torch.float16)
    return X.Linear(t, suh, svh)


class Qwen3Decoder:
    """Weights, KV caches and step buffers for `batch` sequences whose caches
    hold `ctx` random positions; step() decodes one token per sequence."""

    def __init__(self, cfg: Qwen3Config, batch: int, ctx: int, seed: int = 0, max_new: int = 16):
        import torch
        self.torch = torch
        self.cfg, self.B = cfg, batch
        self.tmax = ctx + max_new
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        H, dev = cfg.hidden, "cuda"

        def norm_w(n):
            return (1.0 + 0.1 * torch.randn(n, device=dev, generator=g)).to(torch.float16)

        self.embed_table = (torch.randn(cfg.vocab, H, device=dev, generator=g)).to(torch.float16)
        self.layers = []
        for _ in range(cfg.layers):
            L = {
                "q": random_linear(torch, H, cfg.q_dim, cfg.k_bits, g),
                "k": random_linear(torch, H, cfg.kv_dim, cfg.k_bits, g),
                "v": random_linear(torch, H, cfg.kv_dim, cfg.k_bits, g),
                "o": random_linear(torch, cfg.q_dim, H, cfg.k_bits, g),
                "gate": random_linear(torch, H, cfg.inter, cfg.k_bits, g),
                "up": random_linear(torch, H, cfg.inter, cfg.k_bits, g),
                "down": random_linear(torch, cfg.inter, H, cfg.k_bits, g),
                "in_norm": norm_w(H), "post_norm": norm_w(H),
                "q_norm": norm_w(HEAD_DIM), "k_norm": norm_w(HEAD_DIM),
                "kc": torch.randn(batch, cfg.kv_heads, self.tmax, HEAD_DIM, device=dev,
                                  generator=g).to(torch.float16),
                "vc": torch.randn(batch, cfg.kv_heads, self.tmax, HEAD_DIM, device=dev,
                                  generator=g).to(torch.float16),
            }
            self.layers.append(L)
        self.final_norm = norm_w(H)
        self.lm_head = random_linear(torch, H, cfg.vocab, cfg.k_bits, g)
        B = batch
        f16 = torch.float16
        self.h = torch.empty(B, H, dtype=torch.float32, device=dev)
        self.ssq = torch.empty(B, H // 128, dtype=torch.float32, device=dev)
        self.g = torch.empty(B, cfg.inter, dtype=f16, device=dev)
        self.u = torch.empty(B, cfg.inter, dtype=f16, device=dev)
        self.q = torch.empty(B, cfg.q_dim, dtype=f16, device=dev)
        self.k = torch.empty(B, cfg.kv_dim, dtype=f16, device=dev)
        self.v = torch.empty(B, cfg.kv_dim, dtype=f16, device=dev)
        self.att = torch.empty(B, cfg.q_dim, dtype=f16, device=dev)
        self.logits = torch.empty(B, cfg.vocab, dtype=f16, device=dev)
        nbytes = attn_scratch_bytes(B, cfg.heads, cfg.kv_heads, self.tmax)
        # zeroed once: the attention leaves its arrival tickets zero
        self.scratch = torch.zeros((nbytes + 3) // 4, dtype=torch.float32, device=dev)
        self.ids = torch.zeros(B, dtype=torch.int32, device=dev)
        self.pos = torch.full((B,), ctx, dtype=torch.int32, device=dev)

    def weight_bytes(self) -> int:
        """Packed EXL3 bytes one step reads (every linear once)."""
        c = self.cfg
        per = (c.hidden * (c.q_dim + 2 * c.kv_dim) + c.q_dim * c.hidden + 3 * c.hidden * c.inter)
        return (c.layers * per + c.hidden * c.vocab) * c.k_bits // 8

    def kv_bytes(self) -> int:
        """KV cache bytes one step's attention reads (keys 0 .. pos per row)."""
        c = self.cfg
        rows = int(self.pos.sum().item()) + self.B
        return c.layers * 2 * c.kv_heads * HEAD_DIM * 2 * rows

    def step(self, stream=None):
        """One decode step: logits [B, vocab] for tokens self.ids at positions
        self.pos (the caches take their k, v at row pos).

        Five launches a layer: q+k+v with the input RMSNorm of the residual h
        in their prepare; attention with q/k norm, RoPE and the KV append;
        o, whose prepare combines the attention's key splits and whose
        finish adds into h (and leaves h's sums of squares per 128 columns
        for the next norm); gate+up with the post-attention RMSNorm in their
        prepare; down with the SwiGLU in its prepare and its finish adding
        into h.  Rows beyond one prepare batch (batch 16) add the
        attention's combine launch and norm / SwiGLU launches."""
        c = self.cfg
        embed(self.ids, self.embed_table, self.h, self.ssq, stream)
        for L in self.layers:
            linears([L["q"].weight, L["k"].weight, L["v"].weight], self.h,
                    outs=[self.q, self.k, self.v], norm_w=L["in_norm"], nssq=self.ssq, eps=c.eps,
                    stream=stream)
            attn_o(self.q, self.k, self.v, L["q_norm"], L["k_norm"], self.pos, L["kc"], L["vc"],
                   L["o"].weight, self.h, self.ssq, self.att, self.scratch, c.eps, c.theta,
                   stream)
            linears([L["gate"].weight, L["up"].weight], self.h, outs=[self.g, self.u],
                    norm_w=L["post_norm"], nssq=self.ssq, eps=c.eps, stream=stream)
            linears([L["down"].weight], self.g, up=self.u, res=self.h, res_ssq=self.ssq,
                    stream=stream)
        linears([self.lm_head.weight], self.h, outs=[self.logits], norm_w=self.final_norm,
                nssq=self.ssq, eps=c.eps, stream=stream)
        return self.logits


class PagedDecoder:
    """A Qwen3Decoder's weights over a paged cache (plugins_amd.paged): one pass
    takes any rows of any sequences -- prompts, single tokens, trees of drafted
    tokens -- and `verify` keeps what the model's own tokens accept.

    The reference's counterpart is its drafter and verify step on MLX
    (turboexl3_qwen38/src/spec/drafter.zig); its verify rows take the decode
    chain of the quant table, as these linears do up to 16 rows.

    With `window` (0: all rows, else the last ones of each sequence's step) every key
    keeps the attention weight that it has had, `decay` times what it had a step before,
    and `evict` brings sequences down to the heaviest; `fork` and `restart` are then the
    decoder's, not the cache's.  Rows go on behind a sequence's keys, at the place that its
    text has there: one that is to go on from earlier is forked there, or started again."""

    window, decay = None, 1.0
    score = gone = None  # with a window: the keys' weights, and how many each sequence has evicted
    # ... and of each sequence two key numbers: up to the first its keys are the text's first
    # ones, from the second on they are the text's `gone` places further.  Those between are
    # other ones in every layer and head.
    even = None

    def __init__(self, model: Qwen3Decoder, seqs: int, pages: int, max_pages: int, page: int = 64,
                 window: int | None = None, decay: float = 1.0):
        from . import paged as P
        self.P, self.m, self.cfg, self.torch = P, model, model.cfg, model.torch
        c = model.cfg
        self.cache = P.PagedCache(c.layers, pages, c.kv_heads, seqs, max_pages, page, HEAD_DIM,
                                  self.torch.float16, model.embed_table.device)
        if window is not None:
            self.window, self.decay = window, decay
            dev = model.embed_table.device
            self.score = self.torch.zeros(c.layers, seqs, c.kv_heads, max_pages * page, device=dev)
            self.gone = self.torch.zeros(seqs, dtype=self.torch.int32, device=dev)
            self.even = [(max_pages * page, 0)] * seqs

    def _row_of(self, cu, n: int):
        """Of rows 0 .. n - 1 of a step: their sequences (the last one's for rows
        behind it) and their places in them."""
        t = self.torch.arange(n, dtype=self.torch.int32, device=cu.device)
        s = self.torch.searchsorted(cu[1:], t, right=True).clamp(max=cu.numel() - 2)
        return s, t - cu[s]

    def _weigh(self, layer: int, rows, q, mask) -> None:
        self.P.weigh(self.cache, layer, rows, q, self.score[layer, :rows.seqs], mask, None, self.window,
                     self.decay)

    def forward(self, rows, ids, parent=None, only=None, stream=None, queries=None):
        """Logits [rows, vocab] of the step's rows (of the rows numbered by `only`,
        int64, if given), whose keys and values go into the cache behind each
        sequence's `rows.len`; the pages are there (cache.reserve).  ids int32
        [rows], one outside the vocabulary (in rows that pad the step, say) taken
        as the nearest in it; parent: the trees (None: each sequence's rows in a
        line).  queries: a list that gets each layer's, whose weights of the keys are
        then not taken here."""
        torch, P, m, c, cache = self.torch, self.P, self.m, self.cfg, self.cache
        if stream is not None:
            with P._on(cache, stream):
                return self.forward(rows, ids, parent, only, queries=queries)
        T = rows.rows
        P._ints(ids, "ids", cache, T)  # embed reads as many as there are rows
        if cache.index != P._device():  # the linears and norms go to the current one
            with torch.cuda.device(cache.index):
                return self.forward(rows, ids, parent, only, queries=queries)
        f16 = {"dtype": torch.float16, "device": ids.device}
        if T == 0:
            if only is not None and only.numel() > 0:
                raise IndexError("only: the step has no rows")
            return torch.empty(0, c.vocab, **f16)
        h = torch.empty(T, c.hidden, dtype=torch.float32, device=ids.device)
        x, att = torch.empty(T, c.hidden, **f16), torch.empty(T, c.q_dim, **f16)
        pos, slot, mask = P.plan(cache, rows, parent)
        if self.gone is not None and rows.seqs:
            pos += self.gone[self._row_of(rows.cu, T)[0]]
        embed(ids.clamp(0, c.vocab - 1), m.embed_table, h)
        add = None
        for li, L in enumerate(m.layers):
            add_rmsnorm(h, add, L["in_norm"], x, c.eps)
            q, k, v = X.matmul_shared([L["q"].weight, L["k"].weight, L["v"].weight], x)
            P.qkv_append(cache, li, q, k, v, L["q_norm"], L["k_norm"], pos, slot, q, c.eps, c.theta)
            P.attend(cache, li, rows, q, att, mask)
            if queries is not None:
                queries.append(q)
            elif self.score is not None:
                self._weigh(li, rows, q, mask)
            add_rmsnorm(h, X.matmul(L["o"].weight, att), L["post_norm"], x, c.eps)
            add = X.swiglu(L["gate"].weight, L["up"].weight, L["down"].weight, x)
        add_rmsnorm(h, add, m.final_norm, x, c.eps)
        return X.matmul(m.lm_head.weight, x if only is None else x[only])

    def verify(self, rows, ids, parent=None, most: int | None = None, stream=None,
               temperature=None, draft=None, distinct: bool = False, u=None):
        """One verification: the rows' logits, then the walk down each sequence's tree
        (row 0 is a token that is certain already) by the model's most likely tokens,
        or, with `temperature` float32 [sequences], by ones sampled: draft [rows,
        vocab] are the probabilities that drafted tokens were drawn with (None: they
        were chosen), distinct says that siblings were drawn without replacement, u
        float64 [rows] are the random numbers (None: of torch's generator).  Returns
        path, count, next and new_len (int32 on the device); the cache holds each
        sequence's first new_len keys, and the pages behind them are the caller's to
        trim once the lengths are on the host.  Keys get their weights from the
        accepted rows alone."""
        torch, P = self.torch, self.P
        if stream is not None:
            with P._on(self.cache, stream):
                return self.verify(rows, ids, parent, most, None, temperature, draft, distinct, u)
        if temperature is None and (draft is not None or u is not None or distinct):
            raise ValueError("draft, distinct and u are of a sampled verification: give a temperature")
        queries = None if self.score is None else []
        logits = self.forward(rows, ids, parent, queries=queries)
        i32 = {"dtype": torch.int32, "device": ids.device}
        if temperature is None:
            target = logits.float().argmax(-1).int()
        else:
            target = torch.empty(rows.rows, **i32)
            if u is None:
                u = torch.rand(rows.rows, dtype=torch.float64, device=ids.device)
            P.verify(rows, parent, ids, logits, u, target, draft, temperature, distinct)
        path = torch.empty(rows.seqs, max(1, rows.max_rows) if most is None else most, **i32)
        count, after, new_len = (torch.empty(rows.seqs, **i32) for _ in range(3))
        P.commit(self.cache, rows, parent, ids, target, path, count, after, new_len)
        if queries and rows.seqs:
            # the accepted rows, now in a line behind the keys they followed
            cu = torch.zeros_like(rows.cu)
            torch.cumsum(count, 0, dtype=torch.int32, out=cu[1:])
            n, longest = rows.rows, min(rows.max_rows, path.shape[1])
            line = P.Rows(cu, rows.len, n, longest)
            s, i = self._row_of(cu, n)
            at = rows.cu[s] + path[s, i.clamp(max=path.shape[1] - 1)].clamp(min=0)
            at.clamp_(0, n - 1)
            for li, q in enumerate(queries):
                self._weigh(li, line, q[at], None)
        return path, count, after, new_len

    def fork(self, src: int, dst: int, keys: int, stream=None) -> None:
        """Sequence dst starts with src's first `keys` keys, pages shared, and their
        weights.  Where src has evicted keys these are the first ones of the text, up to the
        least `first` that evictions had, or reach the last ones that they left; a number between,
        up to which every head kept other keys of the text, is refused."""
        whole = True
        if self.score is not None and 0 <= src < len(self.even):
            below, behind = self.even[src]
            whole = keys <= below
            if not whole and keys < behind:
                raise ValueError(f"sequence {src} has evicted keys: it forks at up to {below} or from {behind} on, "
                                 f"not at {keys}")
        with self.P._on(self.cache, stream):
            self.cache.fork(src, dst, keys)
            if self.score is not None:
                self.score[:, dst, :, :keys].copy_(self.score[:, src, :, :keys])
                if whole:
                    self.gone[dst:dst + 1].zero_()
                else:
                    self.gone[dst:dst + 1].copy_(self.gone[src:src + 1])
                self.even[dst] = (self.score.shape[3], 0) if whole else self.even[src]

    def restart(self, seq: int, stream=None) -> None:
        """Gives back a sequence's pages: it holds no keys, and none are gone."""
        with self.P._on(self.cache, stream):
            self.cache.trim(seq, 0)
            if self.gone is not None:
                self.gone[seq:seq + 1].zero_()
                self.even[seq] = (self.score.shape[3], 0)

    def evict(self, lens, keep: int, first: int = 0, last: int = 0, stream=None):
        """Of each sequence's lens[s] keys (a host list, a length for each sequence of
        the cache) at most `keep` stay, in every layer and kv head: the first `first`,
        the last `last` and those of the highest weights.  The pages behind them are
        given back.  Returns the new lengths and `kept` int32 [layers, sequences, kv
        heads, keep] (the numbers that the kept keys had; -1 throughout where none went)."""
        torch, P, cache = self.torch, self.P, self.cache
        if self.score is None:
            raise RuntimeError("a decoder without `window` keeps no weights")
        lens = [int(n) for n in lens]
        if len(lens) != self.score.shape[1] or keep < 1:
            raise ValueError("a length for each sequence, and at least one key to keep")
        if stream is not None:
            with P._on(cache, stream):
                return self.evict(lens, keep, first, last)
        book, page = cache._book(), cache.page
        over = [s for s, n in enumerate(lens) if n > keep]
        for s in over:
            if lens[s] > book.held(s) * page:
                raise ValueError(f"sequence {s} holds pages of {book.held(s) * page} keys, not of {lens[s]}")
        table = book.table()
        for s in over:  # the pages that are written: no other sequence's
            for i in range((keep + page - 1) // page):
                if book.shared(int(table[s, i])) > 1:
                    cache.reserve(s, i * page + 1, (i + 1) * page)
        i32 = {"dtype": torch.int32, "device": self.score.device}
        before = torch.tensor(lens, **i32)
        new_len, kept = torch.empty_like(before), torch.empty(*self.score.shape[:3], keep, **i32)
        P.evict(cache, before, self.score, kept, self.score, new_len, None, first, last)
        self.gone += before - new_len
        head = min(first, keep)
        tail = min(last, keep - head)
        for s in over:
            below, behind = self.even[s]
            self.even[s] = min(below, head), max(keep - tail, behind - (lens[s] - keep))
            cache.trim(s, keep)
        return [min(n, keep) for n in lens], kept
