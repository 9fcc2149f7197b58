"""Serving operators on device tensors (``include/ane_serve.h``).

``KVCache8`` is a paged key/value cache held in 8 bits: ``Append`` rotates a
batch's new queries and keys and writes its keys and values, ``Attend`` is the
causal attention of its queries over the cache, for prompts, chunks of prompts
and single tokens.  ``LogitControls`` changes logits by the requests'
penalties, biases and masks and picks the next tokens.

All tensors are torch tensors on one GPU.  Calls run on torch's current stream
of that GPU, wait for nothing and can be captured into a graph.  What they need
in between comes from torch's allocator, so calls on several streams, and
several captured graphs, share nothing.  Errors follow the engine's convention
(``EngineError`` with the library's message); there is no CPU fallback.  The
reference evaluates whole windows only (ane/engine.go:954-1038) and has no
counterpart.
"""
from __future__ import annotations

import ctypes as C

from . import _lib
from .engine import EngineError

NO_TOKEN = 65535  # tokens[r] of a row that allows none

E_MIN, E_MAX = -15, 8  # range of the cache's exponents


def _torch():
    import torch
    return torch


def _fail(op, msg):
    raise EngineError(_lib.ANE_ERR_ARG, f"storiesane {op}: {msg}")


def _tensor(op, name, t, dtypes, device, dims=None, shape=None):
    """The address of a tensor of one of ``dtypes`` on ``device``, its last
    dimension (if it has more than one element) contiguous."""
    if not hasattr(t, "data_ptr"):
        _fail(op, f"{name} is not a tensor")
    if t.dtype not in dtypes:
        _fail(op, f"{name} is {t.dtype}, want {' or '.join(str(d) for d in dtypes)}")
    if t.device != device:
        _fail(op, f"{name} is on {t.device}, want {device}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        _fail(op, f"{name} has shape {tuple(t.shape)}, want {tuple(shape)}")
    if dims is not None and t.dim() != dims:
        _fail(op, f"{name} has {t.dim()} dimensions, want {dims}")
    if t.dim() and t.shape[-1] > 1 and t.stride(-1) != 1 and t.numel():
        _fail(op, f"{name} is not contiguous along its last dimension")
    return t.data_ptr()


def _whole(op, name, t, dtypes, device, dims=None, shape=None):
    p = _tensor(op, name, t, dtypes, device, dims, shape)
    if not t.is_contiguous():
        _fail(op, f"{name} is not contiguous")
    return p


def _on_gpu(op, t):
    if not hasattr(t, "device") or t.device.type != "cuda":
        _fail(op, "tensors must be on a GPU")
    return t.device


def _stream_getter():
    """device index -> its current stream's handle.  torch's own getter of the
    bare handle where it has one: 0.2 us against 3 for the Stream object, in
    calls that take 10."""
    torch = _torch()
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return raw if raw is not None else lambda index: torch.cuda.current_stream(index).cuda_stream


def _check(lib, rc):
    if rc < 0:
        raise EngineError(rc, lib.ane_op_last_error().decode())
    return rc


class KVBatch:
    """The new tokens of one step, shared by the calls of all layers.

    table int32 [nseq, table_pages], start int32 [nseq] (tokens held before),
    offsets int32 [nseq + 1] (rows of each sequence in the step's tensors),
    rows (rows of those tensors).  The tensors are read when the kernels run:
    a captured step is replayed with what they then hold.  max_len and
    max_new, where known on the host, choose the launch sizes; wrong ones cost
    time.  An append's bits do not depend on them; attention adds its sums up
    in as many parts as they make, so that last bits may."""

    def __init__(self, table, start, offsets, rows, max_len=0, max_new=0):
        op = "kv8 batch"
        dev = _on_gpu(op, table)
        i32 = (_torch().int32,)
        t = _tensor(op, "table", table, i32, dev, dims=2)
        nseq = int(table.shape[0])
        s = _whole(op, "start", start, i32, dev, shape=(nseq,))
        o = _whole(op, "offsets", offsets, i32, dev, shape=(nseq + 1,))
        if table.shape[1] < 1:
            _fail(op, "table has no pages")
        stride = int(table.stride(0)) if nseq > 1 else max(int(table.stride(0)), int(table.shape[1]))
        if stride >= 1 << 31 or not all(0 <= int(v) < 1 << 31 for v in (rows, max_len, max_new)):
            _fail(op, f"rows={rows} max_len={max_len} max_new={max_new}")
        self._keep = (table, start, offsets)
        self.device, self.nseq, self.rows = dev, nseq, int(rows)
        self._c = _lib.Kv8Batch(t, s, o, stride, int(table.shape[1]), nseq, int(rows), int(max_len), int(max_new))
        self._at = C.addressof(self._c)
        self._ws = {}  # workspace bytes by (kv_heads, page_tokens, head_dim, heads)


class KVCache8:
    """The cache's pages: k float8_e4m3fn [pages, kv_heads, page_tokens,
    head_dim], v float8_e4m3fn [pages, kv_heads, page_tokens/16, 4, 16,
    head_dim/16, 4] (token s, dimension d at [s//16, s%16//4, d%16, d//16,
    s%4]), k_exp and v_exp int8 [pages, kv_heads]: value = code * 2**exp.
    The caller owns them; a page needs no initial contents."""

    def __init__(self, k, v, k_exp, v_exp):
        op = "kv8 cache"
        torch = _torch()
        dev = _on_gpu(op, k)
        f8, i8 = (torch.float8_e4m3fn, torch.uint8), (torch.int8,)
        kp = _whole(op, "k", k, f8, dev, dims=4)
        pages, kvh, page, dh = (int(x) for x in k.shape)
        if page % 16 or dh % 16:
            _fail(op, f"page_tokens={page} and head_dim={dh} must be multiples of 16")
        vp = _whole(op, "v", v, f8, dev, shape=(pages, kvh, page // 16, 4, 16, dh // 16, 4))
        ke = _whole(op, "k_exp", k_exp, i8, dev, shape=(pages, kvh))
        ve = _whole(op, "v_exp", v_exp, i8, dev, shape=(pages, kvh))
        self._lib = _lib.load()
        self.k, self.v, self.k_exp, self.v_exp = k, v, k_exp, v_exp
        self.device, self.kv_heads, self.head_dim = dev, kvh, dh
        self.pages, self.page_tokens = pages, page
        self._half, self._f32 = torch.float16, (torch.float32,)
        self._index = dev.index
        self._empty, self._u8, self._stream = torch.empty, torch.uint8, _stream_getter()
        self._c = _lib.Kv8Cache(kp, vp, ke, ve, pages, page, kvh, dh, dev.index)
        self._at = C.addressof(self._c)
        self._append, self._attend = (_lib.plain(self._lib, "ane_kv8_" + n) for n in ("append", "attend"))

    @classmethod
    def Empty(cls, pages, kv_heads, head_dim=64, page_tokens=64, device="cuda"):
        """A cache of zeros on ``device``."""
        torch = _torch()
        k = torch.zeros((pages, kv_heads, page_tokens, head_dim), dtype=torch.uint8, device=device)
        v = torch.zeros((pages, kv_heads, page_tokens // 16, 4, 16, head_dim // 16, 4), dtype=torch.uint8,
                        device=device)
        e = torch.zeros((2, pages, kv_heads), dtype=torch.int8, device=device)
        return cls(k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn), e[0], e[1])

    def _rows(self, op, name, t, batch, heads=None):
        """(address, stride of rows, stride of heads) of fp16 [rows, heads,
        head_dim]; a dimension of one element has no stride that matters."""
        try:
            r, h, d = t.shape
            sr, sh, sd = t.stride()
            if (t.dtype is self._half and t.get_device() == self._index and r == batch.rows and d == self.head_dim
                    and sd == 1 and (heads is None or h == heads)):
                return t.data_ptr(), sr if r > 1 else 0, sh if h > 1 else 0
        except (AttributeError, ValueError):
            pass
        _tensor(op, name, t, (self._half,), self.device, dims=3)  # says what is wrong with it
        _fail(op, f"{name} has shape {tuple(t.shape)}, want ({batch.rows}, {heads or 'heads'}, {self.head_dim})")

    def _new(self, batch, heads):
        return self._empty((batch.rows, heads, self.head_dim), dtype=self._half, device=self.device)

    def _batch(self, op, batch):
        if batch.device != self.device:
            _fail(op, f"batch is on {batch.device}, the cache on {self.device}")

    def _angles(self, op, name, t):
        if not (t.dtype is self._f32[0] and t.get_device() == self._index and t.dim() == 2 and t.is_contiguous()
                and t.shape[1] * 2 == self.head_dim):
            _whole(op, name, t, self._f32, self.device, dims=2)
            _fail(op, f"{name} has shape {tuple(t.shape)}, want (positions, {self.head_dim // 2})")
        return t.data_ptr()

    def Append(self, batch, q, k, v, cos, sin, q_out=None):
        """Rotates q and k (fp16 [rows, heads or kv_heads, head_dim], any
        strides that are multiples of 8) by their positions, writes the
        queries to q_out (new if None; may be q) and appends keys and values.
        q None: keys and values only.  cos, sin: fp32 [positions, head_dim/2].
        Returns q_out."""
        op = "kv8 append"
        self._batch(op, batch)
        kp, kr, kh = self._rows(op, "k", k, batch, self.kv_heads)
        vp, vr, vh = self._rows(op, "v", v, batch, self.kv_heads)
        heads = qp = qr = qh = op_ = or_ = oh = 0
        if q is not None:
            qp, qr, qh = self._rows(op, "q", q, batch)
            heads = q.shape[1]
            if q_out is None:
                q_out = self._new(batch, heads)
            op_, or_, oh = self._rows(op, "q_out", q_out, batch, heads)
        elif q_out is not None:
            _fail(op, "q_out without q")
        cp, sp = self._angles(op, "cos", cos), self._angles(op, "sin", sin)
        n = cos.shape[0]
        if sin.shape[0] != n:
            _fail(op, f"cos has {n} positions, sin {sin.shape[0]}")
        a = _lib.pack_append(qp, kp, vp, op_, cp, sp, qr, qh, kr, kh, vr, vh, or_, oh, heads, n)
        rc = self._append(self._at, batch._at, a, self._stream(self._index))
        if rc:
            _check(self._lib, rc)
        return q_out

    def Attend(self, batch, q, out=None, scale=None):
        """Causal attention of q (fp16 [rows, heads, head_dim], rotated) over
        the cache; the batch's tokens have been appended.  scale: default
        head_dim ** -0.5.  Returns out (new if None: rows of no sequence are
        then undefined; may be q)."""
        op = "kv8 attend"
        self._batch(op, batch)
        qp, qr, qh = self._rows(op, "q", q, batch)
        heads = q.shape[1]
        if out is None:
            out = self._new(batch, heads)
        yp, yr, yh = self._rows(op, "out", out, batch, heads)
        key = (self.kv_heads, self.page_tokens, self.head_dim, heads)
        n = batch._ws.get(key)
        if n is None:
            n = batch._ws[key] = _check(self._lib, self._lib.ane_kv8_attend_workspace(self._c, batch._c, heads))
        ws = self._empty(n, dtype=self._u8, device=self.device) if n else None
        try:
            a = _lib.pack_attend(qp, yp, qr, qh, yr, yh, heads, self.head_dim ** -0.5 if scale is None else scale,
                                 0 if ws is None else ws.data_ptr(), n)
        except (OverflowError, _lib.struct.error):
            _fail(op, f"scale={scale} is no fp32 number")
        rc = self._attend(self._at, batch._at, a, self._stream(self._index))
        if rc:
            _check(self._lib, rc)
        return out


class LogitControls:
    """The requests' parameters: repetition (> 0 meant; 1 changes nothing),
    frequency and presence penalties fp32 [rows], bias fp32 [vocab] or [rows,
    vocab], mask int32 words [ceil(vocab/32)] or [rows, ceil(vocab/32)] (bit
    v % 32 of word v // 32 set: token v allowed).  None: not used.  The
    tensors are read when the kernels run, so their contents may change from
    step to step."""

    def __init__(self, vocab, repetition=None, frequency=None, presence=None, bias=None, mask=None):
        self._op = op = "control logits"
        torch = _torch()
        self.vocab = int(vocab)
        self._keep = given = [t for t in (repetition, frequency, presence, bias, mask) if t is not None]
        self.device = _on_gpu(op, given[0]) if given else None
        self.rows = None
        a = _lib.LogitsArgs()
        f32 = (torch.float32,)
        for name, t in (("repetition", repetition), ("frequency", frequency), ("presence", presence)):
            if t is not None:
                setattr(a, name, _whole(op, name, t, f32, self.device, dims=1))
                self._same_rows(name, t.shape[0])
        for name, t, types, width in (("bias", bias, f32, self.vocab),
                                      ("mask", mask, (torch.int32, torch.uint32), (self.vocab + 31) // 32)):
            if t is None:
                continue
            if t.dim() not in (1, 2) or t.shape[-1] != width:
                _fail(op, f"{name} has shape {tuple(t.shape)}, want ([rows,] {width})")
            setattr(a, name, _tensor(op, name, t, types, self.device))
            if t.dim() == 2:
                self._same_rows(name, t.shape[0])
                setattr(a, name + "_row", self._row(t))
        self.penalties = any(t is not None for t in (repetition, frequency, presence))
        self._f32, self._i32 = f32, (torch.int32,)
        self._u16 = (torch.uint16, torch.int16)
        self._empty, self._u8, self._stream = torch.empty, torch.uint8, _stream_getter()
        self._index = self.device.index if self.device is not None else None
        self._params = (a.repetition or 0, a.frequency or 0, a.presence or 0, a.bias or 0, a.mask or 0, a.bias_row,
                        a.mask_row)
        self._bytes = {}  # of the workspace, by rows
        self._lib = _lib.load()
        self._control = _lib.plain(self._lib, "ane_control_logits")

    def _same_rows(self, name, n):
        if self.rows is not None and self.rows != n:
            _fail(self._op, f"{name} has {n} rows, others have {self.rows}")
        self.rows = int(n)

    @staticmethod
    def _row(t):
        """Stride between rows; one row has none that matters."""
        return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])

    def Apply(self, logits, history=None, lengths=None, prompts=None, out=None, tokens=None):
        """logits fp32 [rows, vocab] -> (out, tokens): the changed logits (new
        if None; may be logits) and the greedy choice int32 [rows] (new if
        None; NO_TOKEN where nothing is allowed).  history uint16 or int16
        bits [rows, n], of which lengths int32 [rows] are tokens, the first
        prompts int32 [rows] (None: 0) of them the prompt's."""
        op = self._op
        index = logits.get_device() if hasattr(logits, "get_device") else -1
        if index < 0:
            _on_gpu(op, logits)
        if self._index is not None and index != self._index:
            _fail(op, f"logits are on {logits.device}, the controls on {self.device}")
        lp, lr, rows, vocab = self._matrix("logits", logits, self._f32, index)
        if vocab != self.vocab or (self.rows is not None and rows != self.rows):
            _fail(op, f"logits have shape {tuple(logits.shape)}, want ({self.rows or 'rows'}, {self.vocab})")
        if out is None:
            out = self._empty((rows, vocab), dtype=logits.dtype, device=logits.device)
        yp, yr, yn, yv = self._matrix("out", out, self._f32, index)
        if yn != rows or yv != vocab:
            _fail(op, f"out has shape {tuple(out.shape)}, want ({rows}, {vocab})")
        if tokens is None:
            tokens = self._empty(rows, dtype=self._i32[0], device=logits.device)
        tp = self._vector("tokens", tokens, index, rows)
        hp = hr = np_ = pp = most = 0
        if history is not None:
            hp, hr, hn, most = self._matrix("history", history, self._u16, index)
            if hn != rows:
                _fail(op, f"history has {hn} rows, want {rows}")
            if lengths is None:
                _fail(op, "history without lengths")
            np_ = self._vector("lengths", lengths, index, rows)
            if prompts is not None:
                pp = self._vector("prompts", prompts, index, rows)
        elif self.penalties:
            _fail(op, "penalties without a history")
        elif lengths is not None or prompts is not None:
            _fail(op, "lengths without a history")
        n = self._bytes.get(rows)
        if n is None:
            n = self._bytes[rows] = _check(self._lib, self._lib.ane_control_logits_workspace(rows, vocab))
        ws = self._empty(n, dtype=self._u8, device=logits.device) if n else None
        rep, freq, pres, bias, mask, bias_row, mask_row = self._params
        a = _lib.pack_logits(lp, yp, hp, np_, pp, rep, freq, pres, bias, mask, tp, lr, yr, hr, bias_row, mask_row,
                             rows, vocab, most, index, 0 if ws is None else ws.data_ptr(), n)
        rc = self._control(a, self._stream(index))
        if rc:
            _check(self._lib, rc)
        return out, tokens

    def _matrix(self, name, t, dtypes, index):
        """(address, stride of rows, rows, columns)."""
        try:
            n, w = t.shape
            sn, sw = t.stride()
            if t.dtype in dtypes and t.get_device() == index and (sw == 1 or w <= 1 or n == 0):
                return t.data_ptr(), sn if n > 1 else max(sn, w), n, w
        except (AttributeError, ValueError):
            pass
        _tensor(self._op, name, t, dtypes, _torch().device("cuda", index), dims=2)  # says what is wrong with it
        _fail(self._op, f"{name} is not a matrix of rows")

    def _vector(self, name, t, index, rows):
        if t.dtype is self._i32[0] and t.get_device() == index and t.shape == (rows,) and t.is_contiguous():
            return t.data_ptr()
        return _whole(self._op, name, t, self._i32, _torch().device("cuda", index), shape=(rows,))
