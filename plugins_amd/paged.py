"""A paged KV cache and the operators that serve drafted tokens from it
(include/exl3_paged.h): the host mirror in Python.

A cache is two tensors [layers][pages][kv heads][page][head dim] (keys and
values, float16 or bfloat16) and a table [sequences][pages of a sequence] of
page numbers on the device.  A step brings `Rows`: a token, a prompt's rows or a
tree of drafted tokens for each of several sequences.

    cache = PagedCache(layers=36, pages=4096, kv_heads=8, seqs=32, max_pages=512)
    cache.reserve(seq, have, have + n)         # pages for n new rows
    rows = Rows.of([n], [have], cache.device)
    pos, slot, mask = plan(cache, rows, parent)
    for layer in ...:
        qkv_append(cache, layer, q, k, v, q_norm, k_norm, pos, slot, q)
        attend(cache, layer, rows, q, out, mask=mask)
    commit(cache, rows, parent, ids, target, path, count, next, new_len)
    cache.trim(seq, new_len)

Every operator runs in libexl3_mi355x.so on the current stream (or the one
given); PyTorch allocates and supplies the stream.  A refused call raises
`exl3.Exl3Error` with the refusal's name.
"""
from __future__ import annotations

import ctypes
import math
from ctypes import POINTER, Structure, c_double, c_float, c_int32, c_int64, c_size_t, c_uint32, c_void_p

from . import exl3 as X

TREE_MAX = 1024  # EXL3P_TREE_MAX

_torch = None  # the module, from the first cache or rows on
_int32 = _device = _raw_stream = None


def _t():
    global _torch, _int32, _device, _raw_stream
    if _torch is None:
        _torch = X._torch()
        _int32 = _torch.int32
        # torch.cuda.current_device() and current_stream(i).cuda_stream without what
        # surrounds them (0.2 and 2 us a call)
        _device, _raw_stream = _torch._C._cuda_getDevice, _torch._C._cuda_getCurrentRawStream
    return _torch


class CacheDesc(Structure):
    """exl3p_cache"""
    _fields_ = [("size", c_uint32), ("dtype", c_int32), ("k", c_void_p), ("v", c_void_p),
                ("layers", c_int32), ("pages", c_int32), ("kv_heads", c_int32), ("page", c_int32),
                ("dim", c_int32), ("seqs", c_int32), ("max_pages", c_int32), ("table", c_void_p)]


class RowsDesc(Structure):
    """exl3p_rows"""
    _fields_ = [("size", c_uint32), ("seqs", c_int32), ("rows", c_int32), ("max_rows", c_int32),
                ("cu", c_void_p), ("len", c_void_p)]


_V = X.Verdict
_P = c_void_p
_SIGS = {
    "exl3p_tree_plan": (_V, [_P, _P, _P, _P, _P, _P, c_int32, _P]),
    "exl3p_qkv_append": (_V, [_P, c_int32, c_int32, c_int32, _P, c_int64, _P, c_int64, _P, c_int64,
                              _P, _P, _P, _P, _P, c_int64, c_float, c_double, _P]),
    "exl3p_attend_scratch_bytes": (c_size_t, [_P, _P, c_int32]),
    "exl3p_attend": (_V, [_P, c_int32, _P, c_int32, _P, c_int64, _P, c_int32, c_float, _P, c_int64,
                          _P, c_size_t, _P]),
    "exl3p_commit": (_V, [_P, _P, _P, _P, _P, _P, c_int32, _P, _P, _P, _P]),
    "exl3p_copy_pages": (_V, [_P, _P, _P, c_int32, _P]),
    "exl3p_book_open": (_P, [c_int32, c_int32, c_int32, c_int32, POINTER(_V)]),
    "exl3p_book_close": (None, [_P]),
    "exl3p_book_reserve": (_V, [_P, c_int32, c_int32, c_int32, _P, _P, c_int32, POINTER(c_int32)]),
    "exl3p_book_fork": (_V, [_P, c_int32, c_int32, c_int32]),
    "exl3p_book_trim": (_V, [_P, c_int32, c_int32]),
    "exl3p_book_compact": (_V, [_P, _P, _P, c_int32, POINTER(c_int32)]),
    "exl3p_book_table": (_P, [_P]),
    "exl3p_book_free_pages": (c_int32, [_P]),
    "exl3p_book_held": (c_int32, [_P, c_int32]),
    "exl3p_book_shared": (c_int32, [_P, c_int32]),
}
_paged = None


def paged_lib():
    """libexl3_mi355x.so with the exl3p_* signatures set."""
    global _paged
    if _paged is None:
        L = X.lib()
        for name, (res, args) in _SIGS.items():
            fn = getattr(L, name)
            fn.restype = res
            fn.argtypes = args
        _paged = L
    return _paged


def _c_int(x: int) -> int:
    """x, refused where a C int32 would hold another number (ctypes takes the low bits)."""
    if not -(1 << 31) <= x < 1 << 31:
        raise OverflowError(f"{x} is no 32-bit integer")
    return x


class Book:
    """exl3p_book: which pages are whose (host memory only)."""

    def __init__(self, pages: int, page: int, seqs: int, max_pages: int):
        v = X.Verdict()
        self.pages, self.page, self.seqs, self.max_pages = pages, page, seqs, max_pages
        self._b = None
        self._b = paged_lib().exl3p_book_open(*map(_c_int, (pages, page, seqs, max_pages)),
                                              ctypes.byref(v))
        X.check(v, "book")

    def _pairs(self, fn, *args, room):
        src, dst, n = (c_int32 * max(1, room))(), (c_int32 * max(1, room))(), c_int32(0)
        X.check(fn(self._b, *map(_c_int, args), src, dst, _c_int(room), ctypes.byref(n)), "book")
        return list(src[:n.value]), list(dst[:n.value])

    def reserve(self, seq: int, start: int, stop: int):
        """Pages for keys up to `stop`, keys start .. stop - 1 writable (pages held
        behind them stay, shared ones shared); the pairs (src, dst) that have to be
        copied first."""
        return self._pairs(paged_lib().exl3p_book_reserve, seq, start, stop, room=1)

    def fork(self, src: int, dst: int, keys: int) -> None:
        X.check(paged_lib().exl3p_book_fork(self._b, *map(_c_int, (src, dst, keys))), "book")

    def trim(self, seq: int, keys: int) -> None:
        X.check(paged_lib().exl3p_book_trim(self._b, _c_int(seq), _c_int(keys)), "book")

    def compact(self, room: int | None = None):
        return self._pairs(paged_lib().exl3p_book_compact,
                           room=self.pages if room is None else room)

    def table(self):
        """A numpy view [seqs][max_pages] of the book's own table, which keeps the
        book open (but for close())."""
        import numpy as np
        p = paged_lib().exl3p_book_table(self._b)
        if p is None:
            raise ValueError("the book is closed")
        t = (c_int32 * self.max_pages * self.seqs).from_address(p)
        t.book = self
        return np.ctypeslib.as_array(t)

    def free_pages(self) -> int:
        return paged_lib().exl3p_book_free_pages(self._b)

    def held(self, seq: int) -> int:
        return paged_lib().exl3p_book_held(self._b, seq)

    def shared(self, page: int) -> int:
        return paged_lib().exl3p_book_shared(self._b, page)

    def close(self) -> None:
        if self._b:
            paged_lib().exl3p_book_close(self._b)
            self._b = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class PagedCache:
    """Keys, values, table and book of a cache."""

    def __init__(self, layers: int, pages: int, kv_heads: int, seqs: int, max_pages: int,
                 page: int = 64, head_dim: int = 128, dtype=None, device="cuda"):
        torch = _t()
        book = Book(pages, page, seqs, max_pages)
        shape = (layers, pages, kv_heads, page, head_dim)
        dtype = torch.float16 if dtype is None else dtype
        k = torch.zeros(shape, dtype=dtype, device=device)
        self._over(k, torch.zeros_like(k),
                   torch.full((seqs, max_pages), -1, dtype=torch.int32, device=device))
        self.book = book

    @classmethod
    def over(cls, k, v, table) -> "PagedCache":
        """A cache over tensors in hand: k, v [layers][pages][kv heads][page][dim],
        table int32 [sequences][pages]; its pages are the caller's to keep (no book)."""
        c = cls.__new__(cls)
        c.book = None
        c._over(k, v, table)
        return c

    def _over(self, k, v, table) -> None:
        torch = _t()
        if k.device.type != "cuda":
            raise ValueError("a cache lies on a GPU")
        if k.dim() != 5 or v.shape != k.shape or v.dtype != k.dtype or table.dim() != 2:
            raise ValueError("k and v are alike, [layers][pages][kv heads][page][dim]; table has 2 dims")
        if table.dtype != torch.int32:
            raise TypeError("the table is int32")
        for t in (k, v, table):
            if not t.is_contiguous() or t.device != k.device:
                raise ValueError("k, v and table are dense and on one device")
        self.k, self.v, self.table = k, v, table
        self.device, self.index = k.device, k.device.index
        self.dtype = k.dtype
        layers, pages, kv_heads, page, dim = k.shape
        self.desc = CacheDesc(ctypes.sizeof(CacheDesc), X.dtype_of(k), k.data_ptr(), v.data_ptr(),
                              layers, pages, kv_heads, page, dim, table.shape[0], table.shape[1],
                              table.data_ptr())
        self._ref = ctypes.addressof(self.desc)
        self.layers, self.pages, self.kv_heads, self.page, self.head_dim = layers, pages, kv_heads, page, dim

    # ---- the book, and what it asks of the device

    # What the book has changed and the device does not have yet: pairs of pages to
    # copy and the sequence (None: all) whose row of the table changed.  It stays
    # where a copy failed, and is done before the book changes again: until then
    # the device's table and the pages in it are those of before, whole.
    _owed = None

    def _book(self) -> Book:
        if self.book is None:
            raise RuntimeError("a cache over given tensors has no book")
        return self.book

    def _sync(self, seq: int | None = None, stream=None) -> None:
        """The book's table, or a sequence's row of it, to the device."""
        torch = _t()
        t = torch.from_numpy(self._book().table())
        with _on(self, stream):
            if seq is None:
                self.table.copy_(t)
            else:
                self.table[seq].copy_(t[seq])

    def _settle(self, stream) -> Book:
        """The book, with nothing owed to the device."""
        book = self._book()
        if self._owed is not None:
            src, dst, seq = self._owed
            if src:
                copy_pages(self, src, dst, stream)
            self._sync(seq, stream)
            self._owed = None
        return book

    def reserve(self, seq: int, start: int, stop: int, stream=None) -> None:
        """Pages for a sequence's keys up to `stop`, keys start .. stop - 1 its own
        to write: shared pages among them are replaced, the one that holds earlier
        keys too by a copy.  Pages behind them that the sequence holds stay as they
        are, shared ones shared: trim(seq, start) first to be rid of them.

        Here, in fork, trim and compact: where the copy to the device fails, the
        book keeps the change, and the next of these calls copies first."""
        self._owed = (*self._settle(stream).reserve(seq, start, stop), seq)
        self._settle(stream)

    def fork(self, src: int, dst: int, keys: int, stream=None) -> None:
        """Sequence dst starts with src's first `keys` keys, their pages shared."""
        self._settle(stream).fork(src, dst, keys)
        self._owed = ([], [], dst)
        self._settle(stream)

    def trim(self, seq: int, keys: int, stream=None) -> None:
        """Gives back the pages behind the sequence's first `keys` keys (0: all)."""
        self._settle(stream).trim(seq, keys)
        self._owed = ([], [], seq)
        self._settle(stream)

    def compact(self, stream=None) -> int:
        """Moves the pages in use to the lowest numbers; how many moved."""
        src, dst = self._settle(stream).compact()
        if src:
            self._owed = (src, dst, None)
            self._settle(stream)
        return len(src)


class Rows:
    """A step's rows: cu int32 [sequences + 1], len int32 [sequences] (keys cached
    before them), both on the device; `rows` of the step's tensors, at most
    `max_rows` of a sequence."""

    def __init__(self, cu, len, rows: int, max_rows: int):
        torch = _t()
        _c_int(rows), _c_int(max_rows)
        if cu.dtype != torch.int32 or len.dtype != torch.int32:
            raise TypeError("cu and len are int32")
        if cu.dim() != 1 or len.dim() != 1 or cu.numel() != len.numel() + 1 or cu.device != len.device:
            raise ValueError("cu has one element more than len, on one device")
        if not cu.is_contiguous() or not len.is_contiguous():
            raise ValueError("cu and len are dense")
        self.cu, self.len = cu, len
        self.rows, self.max_rows, self.seqs = rows, max_rows, len.numel()
        if cu.device.type != "cuda":
            raise ValueError("a step's rows lie on a GPU")
        self.device, self.index = cu.device, cu.device.index
        self.desc = RowsDesc(ctypes.sizeof(RowsDesc), self.seqs, rows, max_rows, cu.data_ptr(),
                             len.data_ptr())
        self._ref = ctypes.addressof(self.desc)

    @classmethod
    def of(cls, counts, lens, device="cuda") -> "Rows":
        """Rows from host lists: counts[s] rows behind lens[s] cached keys."""
        torch = _t()
        if len(counts) != len(lens):
            raise ValueError("a count and a length for each sequence")
        cu = [0]
        for n in counts:
            cu.append(cu[-1] + int(n))
        return cls(torch.tensor(cu, dtype=torch.int32, device=device),
                   torch.tensor([int(x) for x in lens], dtype=torch.int32, device=device), cu[-1],
                   max([int(n) for n in counts], default=0))


class _on:
    """The cache's device, and the stream given, as torch's current ones."""

    def __init__(self, cache, stream):
        torch = _t()
        self.held = []
        if stream is not None:
            _stream(cache, stream)
        if cache.index != torch.cuda.current_device():
            self.held.append(torch.cuda.device(cache.index))
        if stream is not None:
            self.held.append(torch.cuda.stream(stream))

    def __enter__(self):
        for h in self.held:
            h.__enter__()

    def __exit__(self, *e):
        for h in reversed(self.held):
            h.__exit__(*e)


def _matrix(t, what: str, cache, rows: int, width: int):
    """Base and row stride of a step's tensor [rows, ...] of `width` a row."""
    if t.dtype is not cache.dtype:
        raise TypeError(f"{what} is {t.dtype}, the cache {cache.dtype}")
    if t.get_device() != cache.index:
        raise ValueError(f"{what} is on {t.device}, the cache on {cache.device}")
    shape, stride = t.shape, t.stride()
    if len(shape) == 2:
        ok = shape[1] == width and stride[1] == 1
    else:
        ok = (len(shape) == 3 and shape[1] * shape[2] == width and
              shape[2] == cache.head_dim and stride[2] == 1 and
              (stride[1] == shape[2] or shape[1] == 1))
    if not ok or shape[0] != rows:
        raise ValueError(f"{what}: [{rows}, {width}] (or heads apart), elements side by side, not "
                         f"{tuple(shape)} with strides {tuple(stride)}")
    return t.data_ptr(), stride[0] if rows > 1 else width


def _ints(t, what: str, cache, n: int):
    if t.dtype is _int32 and t.numel() == n and t.get_device() == cache.index and t.is_contiguous():
        return t.data_ptr()
    if t.dtype is not _int32:
        raise TypeError(f"{what} is int32")
    raise ValueError(f"{what}: {n} dense elements on {cache.device}")


def _stream(cache, stream):
    if stream is not None:
        on = getattr(stream, "device_index", cache.index)  # (others' streams may not say)
        if on != cache.index:
            raise ValueError(f"the stream is on device {on}, the cache on {cache.device}")
        return stream.cuda_stream
    return _raw_stream(cache.index)


def _call(cache, fn, what, *args):
    if cache.index == _device():
        v = fn(*args)
    else:
        with _torch.cuda.device(cache.index):
            v = fn(*args)
    if v.code != X.OK:
        raise X.Exl3Error(v, what)


def _of(cache, rows) -> None:
    if rows.index != cache.index:
        raise ValueError(f"the rows are on {rows.device}, the cache on {cache.device}")


def _mask(mask, cache, rows):
    """Address and words of ancestor masks int64 [rows, words]."""
    if mask is None:
        return None, 0
    if mask.dtype is not _torch.int64:
        raise TypeError("a mask is int64")
    shape = mask.shape
    if len(shape) != 2 or shape[0] != rows.rows or not mask.is_contiguous() or \
            mask.get_device() != cache.index or (shape[1] == 0 and rows.max_rows > 0):
        raise ValueError(f"a mask is dense [{rows.rows}, words] on {cache.device}")
    return mask.data_ptr(), shape[1]


def _heads(q, cache) -> int:
    return q.shape[1] if q.dim() == 3 else q.shape[1] // cache.head_dim


# ------------------------------------------------------------------ operators

def tree_plan(cache, rows, parent, pos, slot, mask=None, stream=None) -> None:
    """exl3p_tree_plan into pos, slot int32 [rows] and mask int64 [rows, words]."""
    _of(cache, rows)
    n = rows.rows
    mp, words = _mask(mask, cache, rows)
    _call(cache, paged_lib().exl3p_tree_plan, "tree_plan", cache._ref, rows._ref,
          None if parent is None else _ints(parent, "parent", cache, n), _ints(pos, "pos", cache, n),
          _ints(slot, "slot", cache, n), mp, words, _stream(cache, stream))


def plan(cache, rows, parent=None, stream=None):
    """tree_plan into new tensors: pos, slot, mask (None without a parent: rows
    in a line see those before them)."""
    torch = _torch
    with _on(cache, stream):
        pos = torch.empty(rows.rows, dtype=torch.int32, device=cache.device)
        slot = torch.empty_like(pos)
        mask = None if parent is None else torch.empty(
            rows.rows, max(1, -(-rows.max_rows // 64)), dtype=torch.int64, device=cache.device)
        tree_plan(cache, rows, parent, pos, slot, mask, stream)
    return pos, slot, mask


def qkv_append(cache, layer: int, q, k, v, q_norm, k_norm, pos, slot, q_out, eps: float = 1e-6,
               theta: float = 1e6, stream=None) -> None:
    """exl3p_qkv_append: q [rows, heads * dim] normalized and rotated to q_out,
    k and v into the layer's pages.  q_norm, k_norm [dim], or None: no norm."""
    n, dim = q.shape[0], cache.head_dim
    heads = _heads(q, cache)
    qp, qs = _matrix(q, "q", cache, n, heads * dim)
    kp, ks = _matrix(k, "k", cache, n, cache.kv_heads * dim)
    vp, vs = _matrix(v, "v", cache, n, cache.kv_heads * dim)
    op, os_ = _matrix(q_out, "q_out", cache, n, heads * dim)
    norms = []
    for w in (q_norm, k_norm):
        if w is not None and (w.dtype is not cache.dtype or w.get_device() != cache.index or
                              w.numel() != dim or not w.is_contiguous()):
            raise ValueError(f"a norm's weights are [{dim}], of the cache's type and device")
        norms.append(None if w is None else w.data_ptr())
    _call(cache, paged_lib().exl3p_qkv_append, "qkv_append", cache._ref, _c_int(layer), n,
          heads, qp, qs, kp, ks, vp, vs, norms[0], norms[1], _ints(pos, "pos", cache, n),
          _ints(slot, "slot", cache, n), op, os_, eps, theta, _stream(cache, stream))


def attend(cache, layer: int, rows, q, out=None, mask=None, scale: float | None = None,
           scratch=None, stream=None):
    """exl3p_attend: out [rows, heads * dim] = softmax(q k^T scale) v over the
    cache's keys and, by their masks, the rows'.  out may be q.  scratch: a byte tensor of at
    least attend_scratch_bytes() that no overlapping call uses (None: taken from
    torch's allocator for this call)."""
    torch = _torch
    _of(cache, rows)
    L = paged_lib()
    n, dim = rows.rows, cache.head_dim
    heads = _heads(q, cache)
    if out is None:
        with _on(cache, stream):
            out = torch.empty(n, heads * dim, dtype=cache.dtype, device=cache.device)
    qp, qs = _matrix(q, "q", cache, n, heads * dim)
    op, os_ = _matrix(out, "out", cache, n, heads * dim)
    mp, words = _mask(mask, cache, rows)
    if scratch is None:
        need = attend_scratch_bytes(cache, rows, heads)
        if stream is None:
            scratch = torch.empty(need, dtype=torch.uint8, device=cache.device)
        else:
            with _on(cache, stream):
                scratch = torch.empty(need, dtype=torch.uint8, device=cache.device)
    elif scratch.get_device() != cache.index or not scratch.is_contiguous():
        raise ValueError(f"scratch is dense, on {cache.device}")
    _call(cache, L.exl3p_attend, "attend", cache._ref, _c_int(layer), rows._ref, heads,
          qp, qs, mp, words, 1.0 / math.sqrt(dim) if scale is None else scale, op, os_,
          scratch.data_ptr(), scratch.numel() * scratch.element_size(), _stream(cache, stream))
    return out


def attend_scratch_bytes(cache, rows, heads: int) -> int:
    """exl3p_attend_scratch_bytes on the cache's device."""
    if cache.index == _device():
        return paged_lib().exl3p_attend_scratch_bytes(cache._ref, rows._ref, heads)
    with _torch.cuda.device(cache.index):
        return paged_lib().exl3p_attend_scratch_bytes(cache._ref, rows._ref, heads)


def commit(cache, rows, parent, ids, target, path, count, next, new_len, stream=None) -> None:
    """exl3p_commit: path int32 [sequences, most], count, next, new_len int32
    [sequences]; the accepted rows' keys and values move in every layer."""
    _of(cache, rows)
    n, s = rows.rows, rows.seqs
    if path.dim() != 2 or path.shape[0] != s:
        raise ValueError(f"path is [{s}, most rows accepted]")
    _call(cache, paged_lib().exl3p_commit, "commit", cache._ref, rows._ref,
          None if parent is None else _ints(parent, "parent", cache, n), _ints(ids, "ids", cache, n),
          _ints(target, "target", cache, n), _ints(path, "path", cache, path.numel()), path.shape[1],
          _ints(count, "count", cache, s), _ints(next, "next", cache, s),
          _ints(new_len, "new_len", cache, s), _stream(cache, stream))


def copy_pages(cache, src, dst, stream=None) -> None:
    """exl3p_copy_pages: page dst[i] = page src[i] in every layer (host lists)."""
    n = len(src)
    if len(dst) != n:
        raise ValueError("as many pages to write as to read")
    arr = c_int32 * max(1, n)
    src, dst = map(_c_int, src), map(_c_int, dst)
    _call(cache, paged_lib().exl3p_copy_pages, "copy_pages", cache._ref, arr(*src), arr(*dst), n,
          _stream(cache, stream))
