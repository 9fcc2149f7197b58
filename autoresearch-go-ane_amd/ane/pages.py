"""The pages of ``KVCache8`` caches (``include/ane_serve.h``): which sequence
holds which, and which of a long context a query attends to.

``KVPages`` is a pool of page ids that the caches of all layers share: ``Fork``
takes a table of sequences to their next step (beams that go on from others,
sequences that end, pages for new tokens, copies of pages that several hold),
``Compact`` brings the pages in use together, ``Copy`` copies pages within a
pool or into another.  ``KVBounds`` keeps bounds on the keys of each page of a
cache: ``Update`` after an append, ``Select`` for the pages that
``KVCache8.Attend(blocks=...)`` then reads.

As in ``serve.py``: torch tensors on one GPU, torch's current stream, no
waiting, capturable, ``EngineError`` on what the host can see to be wrong; no
CPU fallback and no counterpart in the reference, which evaluates whole windows
only (ane/engine.go:954-1038).
"""
from __future__ import annotations

import ctypes as C

from . import _lib
from .serve import _check, _fail, _stream_getter, _tensor, _torch, _whole


class KVBounds:
    """Bounds on the keys of a cache's pages: box int8 [pages, kv_heads, 2,
    head_dim] (the largest key of each dimension, then the smallest, in whole
    numbers of 2**unit, rounded outwards), unit int8 [pages, kv_heads].  The
    caller owns them; they need no initial contents."""

    def __init__(self, cache, box, unit):
        op = "kv8 bound"
        torch = _torch()
        i8 = (torch.int8,)
        bp = _whole(op, "box", box, i8, cache.device, shape=(cache.pages, cache.kv_heads, 2, cache.head_dim))
        up = _whole(op, "unit", unit, i8, cache.device, shape=(cache.pages, cache.kv_heads))
        self.cache, self.box, self.unit = cache, box, unit
        self._lib, self._i32, self._empty, self._u8 = cache._lib, torch.int32, torch.empty, torch.uint8
        self._c = _lib.Kv8Bounds(bp, up)
        self._at = C.addressof(self._c)
        self._bound, self._select = (_lib.plain(self._lib, "ane_kv8_" + n) for n in ("bound", "select"))

    @classmethod
    def Empty(cls, cache):
        """Bounds of zeros."""
        new = _torch().zeros
        return cls(cache, new((cache.pages, cache.kv_heads, 2, cache.head_dim), dtype=_torch().int8, device=cache.device),
                   new((cache.pages, cache.kv_heads), dtype=_torch().int8, device=cache.device))

    def Update(self, batch):
        """The bounds of the pages that the batch's new tokens were appended
        to."""
        c = self.cache
        c._batch("kv8 bound", batch)
        rc = self._bound(c._at, self._at, batch._at, c._stream(c._index))
        if rc:
            _check(self._lib, rc)

    def Select(self, batch, q, count, first=1, recent=1, blocks=None):
        """For each row of q (fp16 [rows, heads, head_dim], rotated) and
        key/value head the ``count`` pages of its sequence whose keys can match
        it best, the first ``first`` and the last ``recent`` pages always among
        them: blocks int32 [rows, kv_heads, count] (new if None: rows of no
        sequence are then undefined), places in the table, rising, then -1.
        Bounds of a row's own page are of later tokens of the batch too: with
        recent 0 a chunk may choose otherwise than token by token."""
        op = "kv8 select"
        c = self.cache
        c._batch(op, batch)
        qp, qr, qh = c._rows(op, "q", q, batch)
        heads = q.shape[1]
        if not (0 < count <= 65536 and 0 <= first <= 65536 and 0 <= recent <= 65536):
            _fail(op, f"count={count} first={first} recent={recent}")
        if blocks is None:
            blocks = self._empty((batch.rows, c.kv_heads, count), dtype=self._i32, device=c.device)
            bp = blocks.data_ptr()
        else:
            bp, n = c._blocks(op, blocks, batch)
            if n != count:
                _fail(op, f"blocks has shape {tuple(blocks.shape)}, want ({batch.rows}, {c.kv_heads}, {count})")
        key = ("select", c.kv_heads, c.page_tokens, c.head_dim, heads, count)
        n = batch._ws.get(key)
        if n is None:
            n = batch._ws[key] = _check(self._lib,
                                        self._lib.ane_kv8_select_workspace(c._c, batch._c, heads, count))
        ws = self._empty(n, dtype=self._u8, device=c.device) if n else None
        a = _lib.pack_select(qp, bp, qr, qh, heads, count, first, recent, 0 if ws is None else ws.data_ptr(), n)
        rc = self._select(c._at, self._at, batch._at, a, c._stream(c._index))
        if rc:
            _check(self._lib, rc)
        return blocks


class KVPages:
    """The pool of the pages of ``caches`` (one ``KVCache8`` a layer, all of
    the same sizes): page id i is page i of each.  refs int32 [pages]: how many
    entries of tables name a page, not above 0: free.  bounds: the layers'
    ``KVBounds`` (None for a layer without), which move with the pages."""

    def __init__(self, caches, refs, bounds=None):
        self._op = op = "kv8 pages"
        torch = _torch()
        self.caches = list(caches)
        if not self.caches:
            _fail(op, "no caches")
        c = self.caches[0]
        for x in self.caches:
            if (x.pages, x.page_tokens, x.kv_heads, x.head_dim, x.device) != (
                    c.pages, c.page_tokens, c.kv_heads, c.head_dim, c.device):
                _fail(op, "caches differ in their sizes or their device")
        self.bounds = list(bounds) if bounds is not None else None
        if self.bounds is not None and (len(self.bounds) != len(self.caches) or any(
                b is not None and b.cache is not x for b, x in zip(self.bounds, self.caches))):
            _fail(op, "bounds are not those of the caches")
        self._i32 = (torch.int32,)
        self.device, self.pages, self.page_tokens = c.device, c.pages, c.page_tokens
        rp = _whole(op, "refs", refs, self._i32, self.device, shape=(self.pages,))
        self.refs = refs
        self._lib, self._index = c._lib, c._index
        n = len(self.caches)
        self._layers = (_lib.Kv8Cache * n)(*(x._c for x in self.caches))
        self._bounds = None
        if self.bounds is not None:
            self._bounds = (_lib.Kv8Bounds * n)(*(_lib.Kv8Bounds() if b is None else b._c for b in self.bounds))
        self._c = _lib.Kv8Pool(self._layers, self._bounds, rp, n)
        self._at = C.addressof(self._c)
        self._empty, self._u8, self._stream = torch.empty, torch.uint8, _stream_getter()
        self._fork, self._compact, self._copy = (_lib.plain(self._lib, "ane_kv8_" + n)
                                                 for n in ("fork", "compact", "copy"))
        self._bytes = {}  # of a fork's workspace, by the table's size
        self._compact_bytes = _check(self._lib, self._lib.ane_kv8_compact_workspace(self._c))

    @classmethod
    def Empty(cls, caches, bounds=None):
        """A pool whose pages are all free."""
        caches = list(caches)
        if not caches:
            _fail("kv8 pages", "no caches")
        return cls(caches, _torch().zeros(caches[0].pages, dtype=_torch().int32, device=caches[0].device), bounds)

    def _table(self, op, t):
        """(address, stride, pages, sequences)."""
        try:
            n, w = t.shape
            sn, sw = t.stride()
            if t.dtype in self._i32 and t.get_device() == self._index and (sw == 1 or w == 1) and 0 < w <= sn < 1 << 31:
                return t.data_ptr(), sn, w, n
        except (AttributeError, ValueError):
            pass
        p = _tensor(op, "table", t, self._i32, self.device, dims=2)
        n, w = (int(x) for x in t.shape)
        if w < 1:
            _fail(op, "table has no pages")
        stride = int(t.stride(0)) if n > 1 else max(int(t.stride(0)), w)
        if stride >= 1 << 31:
            _fail(op, f"table's rows are {stride} apart")
        return p, stride, w, n

    def _vector(self, op, name, t, n):
        try:
            if t.dtype in self._i32 and t.get_device() == self._index and t.shape == (n,) and t.is_contiguous():
                return t.data_ptr()
        except AttributeError:
            pass
        return _whole(op, name, t, self._i32, self.device, shape=(n,))

    def Fork(self, table, start, parents=None, new=1, missing=None):
        """Takes table int32 [nseq, pages] and start int32 [nseq] (the tokens
        that the sequences hold) to their next step, in place: sequence i goes
        on from parents[i] (int32 [nseq]; None: itself; -1: it ends) and gets
        pages for ``new`` tokens (a number, or int32 [nseq]).  A page that is
        written next and that others hold too is copied first, in all layers.
        A smaller start cuts a sequence off, 0 frees it; refs follow.  Returns
        missing int32 [1] (new if None): the entries for which the pool had no
        page, which are -1."""
        op = "kv8 fork"
        tp, stride, width, nseq = self._table(op, table)
        sp = self._vector(op, "start", start, nseq)
        pp = 0 if parents is None else self._vector(op, "parents", parents, nseq)
        each = np_ = 0
        if hasattr(new, "data_ptr"):
            np_ = self._vector(op, "new", new, nseq)
        else:
            each = int(new)
            if not 0 <= each < 1 << 31:
                _fail(op, f"new={new}")
        if missing is None:
            missing = self._empty(1, dtype=self._i32[0], device=self.device)
            mp = missing.data_ptr()
        else:
            mp = self._vector(op, "missing", missing, 1)
        n = self._bytes.get((nseq, width))
        if n is None:
            n = self._bytes[nseq, width] = _check(self._lib, self._lib.ane_kv8_fork_workspace(self._c, nseq, width))
        ws = self._empty(n, dtype=self._u8, device=self.device)
        a = _lib.pack_fork(tp, sp, pp, np_, mp, stride, width, nseq, each, ws.data_ptr(), n)
        rc = self._fork(self._at, a, self._stream(self._index))
        if rc:
            _check(self._lib, rc)
        return missing

    def Compact(self, table=None, moved=None):
        """Brings the pages that are held to the lowest ids, in all layers;
        refs and the entries of table (int32 [nseq, pages]) follow.  Returns
        moved int32 [pages] (new if None): where each page is now, -1 if it was
        free."""
        op = "kv8 compact"
        tp = stride = width = nseq = 0
        if table is not None:
            tp, stride, width, nseq = self._table(op, table)
        if moved is None:
            moved = self._empty(self.pages, dtype=self._i32[0], device=self.device)
            mp = moved.data_ptr()
        else:
            mp = self._vector(op, "moved", moved, self.pages)
        n = self._compact_bytes
        ws = self._empty(n, dtype=self._u8, device=self.device)
        a = _lib.pack_compact(tp, mp, stride, width, nseq, ws.data_ptr(), n)
        rc = self._compact(self._at, a, self._stream(self._index))
        if rc:
            _check(self._lib, rc)
        return moved

    def Copy(self, src, dst, tokens=None, into=None):
        """Copies the pages src[i] to the pages dst[i] (int32 [n]) of ``into``
        (another pool of like layers; None: this one), in all layers: the
        16-token units of their first tokens[i] tokens (None: all).  Ids
        outside the pools are passed over; refs stay as they are.  n is at
        most 2**24."""
        op = "kv8 copy"
        to = self if into is None else into
        n = int(src.shape[0]) if hasattr(src, "shape") and src.dim() == 1 else 0
        sp = self._vector(op, "src", src, n)
        dp = self._vector(op, "dst", dst, n)
        kp = 0 if tokens is None else self._vector(op, "tokens", tokens, n)
        rc = self._copy(self._at, to._at, _lib.pack_copy(sp, dp, kp, n), self._stream(self._index))
        if rc:
            _check(self._lib, rc)
