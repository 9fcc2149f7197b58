"""The serving operators without a GPU: what they refuse, and the index
arithmetic of the cache kernels walked on the host (the kernels call the same
functions), for good batches and for device arrays that hold nonsense."""
import ctypes as C

import numpy as np
import pytest

from ane import _lib

lib = _lib.load()
P16 = 0x10000   # an aligned address that is never followed: every call below is refused, or has no rows


def cache(**kw):
    f = dict(k=P16, v=P16, k_exp=P16, v_exp=P16, pages=4, page_tokens=64, kv_heads=2, head_dim=64, device=0)
    f.update(kw)
    return _lib.Kv8Cache(**f)


def batch(**kw):
    f = dict(table=P16, start=P16, offsets=P16, table_stride=3, table_pages=3, nseq=2, rows=5, max_len=0, max_new=0)
    f.update(kw)
    return _lib.Kv8Batch(**f)


def append_args(**kw):
    f = dict(q=P16, k=P16, v=P16, q_out=2 * P16, cos=P16, sin=P16, q_row=256, q_head=64, k_row=128, k_head=64,
             v_row=128, v_head=64, q_out_row=256, q_out_head=64, heads=4, positions=192)
    f.update(kw)
    return _lib.Kv8AppendArgs(**f)


def attend_args(**kw):
    f = dict(q=P16, out=P16, q_row=256, q_head=64, out_row=256, out_head=64, heads=4, scale=0.125, ws=P16,
             ws_bytes=1 << 40)
    f.update(kw)
    return _lib.Kv8AttendArgs(**f)


def logits_args(**kw):
    f = dict(logits=P16, out=P16, history=P16, lengths=P16, prompts=P16, repetition=P16, frequency=P16, presence=P16,
             bias=P16, mask=P16, tokens=P16, logits_row=100, out_row=100, history_row=9, bias_row=0, mask_row=4,
             rows=2, vocab=100, history_max=9, device=0, ws=P16, ws_bytes=1 << 30)
    f.update(kw)
    return _lib.LogitsArgs(**f)


def append(c=None, b=None, a=None):
    return lib.ane_kv8_append(c or cache(), b or batch(), a or append_args(), None)


def attend(c=None, b=None, a=None):
    return lib.ane_kv8_attend(c or cache(), b or batch(), a or attend_args(), None)


def refused(rc, *words):
    assert rc == _lib.ANE_ERR_ARG
    msg = lib.ane_op_last_error().decode()
    assert msg.startswith("storiesane "), msg
    for w in words:
        assert w in msg, msg


CACHES = [(dict(k=None), "null cache"), (dict(v_exp=None), "null cache"), (dict(k=P16 + 8), "aligned"),
          (dict(page_tokens=48), "page_tokens=48"), (dict(page_tokens=8), "page_tokens=8"),
          (dict(page_tokens=512), "page_tokens=512"), (dict(head_dim=96), "head_dim=96"), (dict(pages=0), "pages=0"),
          (dict(kv_heads=0), "kv_heads=0")]
BATCHES = [(dict(table=None), "null batch"), (dict(offsets=None), "null batch"), (dict(nseq=-1), "nseq=-1"),
           (dict(nseq=70000), "nseq=70000"), (dict(rows=-1), "rows=-1"), (dict(rows=(1 << 30) + 1), "rows="),
           (dict(table_pages=0), "table_pages=0"), (dict(table_pages=4), "table_pages=4"),
           (dict(table_pages=1 << 25, table_stride=1 << 25), "table_pages="), (dict(max_len=-1), "max_len=-1")]


@pytest.mark.parametrize("kw,word", CACHES)
def test_cache_refusals(kw, word):
    refused(append(c=cache(**kw)), word)
    refused(attend(c=cache(**kw)), word)
    assert lib.ane_kv8_attend_workspace(cache(**kw), batch(), 4) == _lib.ANE_ERR_ARG


@pytest.mark.parametrize("kw,word", BATCHES)
def test_batch_refusals(kw, word):
    refused(append(b=batch(**kw)), word)
    refused(attend(b=batch(**kw)), word)


@pytest.mark.parametrize("kw,word", [
    (dict(k=None), "null"), (dict(cos=None), "null"), (dict(q=None), "null"), (dict(q_out=None), "null"),
    (dict(heads=-1), "null"), (dict(k_row=4), "stride 4"), (dict(v_head=-8), "stride -8"), (dict(q_row=20), "stride"),
    (dict(v=P16 + 2), "aligned"), (dict(q=P16 + 2), "aligned"), (dict(sin=P16 + 4), "aligned"),
    (dict(positions=191), "positions=191"), (dict(q_out_row=0), "overlap"), (dict(q_out_head=0), "overlap"),
    (dict(q_out_row=192), "overlap"), (dict(q_out=P16, q_out_row=512), "other strides")])
def test_append_refusals(kw, word):
    refused(append(a=append_args(**kw)), word)


@pytest.mark.parametrize("kw,word", [
    (dict(q=None), "null"), (dict(out=None), "null"), (dict(q_head=4), "stride 4"), (dict(out=P16 + 8), "aligned"),
    (dict(ws=P16 + 4), "aligned"), (dict(scale=0.0), "scale=0"), (dict(scale=-1.0), "scale=-1"),
    (dict(scale=float("nan")), "scale=nan"), (dict(scale=float("inf")), "scale=inf"), (dict(heads=3), "heads=3"),
    (dict(heads=0), "heads=0"), (dict(heads=66), "heads=66"), (dict(out_row=128), "overlap"),
    (dict(ws=None), "workspace of 0"), (dict(ws_bytes=16), "workspace of 16")])
def test_attend_refusals(kw, word):
    b = batch(table_pages=1024, table_stride=1024)   # long enough for a split, which needs the workspace
    refused(attend(b=b, a=attend_args(**kw)), word)


@pytest.mark.parametrize("kw,word", [
    (dict(logits=None), "null"), (dict(rows=-1), "rows=-1"), (dict(rows=65536), "rows=65536"),
    (dict(vocab=0), "vocab=0"), (dict(vocab=65536), "vocab=65536"), (dict(out=None, tokens=None), "neither"),
    (dict(lengths=None), "lengths"), (dict(history_max=-1), "history_max=-1"), (dict(history_max=10), "history_max=10"),
    (dict(history=None), "history_max=9"),
    (dict(history=None, history_max=0, lengths=None), "penalties without"), (dict(logits_row=99), "stride"), (dict(out_row=99), "stride"),
    (dict(bias_row=99), "stride"), (dict(mask_row=3), "stride"), (dict(out_row=101), "in place"),
    (dict(ws=P16 + 8), "workspace"),
    (dict(vocab=60000, logits_row=60000, out_row=60000, mask_row=1875, ws=None), "workspace of 0"),
    (dict(vocab=60000, logits_row=60000, out_row=60000, mask_row=1875, ws_bytes=8), "workspace of 8")])
def test_control_refusals(kw, word):
    refused(lib.ane_control_logits(logits_args(**kw), None), word)


def test_calls_without_rows_do_nothing():
    for b in (batch(nseq=0, table=None, start=None, offsets=None), batch(rows=0)):
        assert append(b=b) == _lib.ANE_OK
        assert attend(b=b) == _lib.ANE_OK
        assert lib.ane_kv8_attend_workspace(cache(), b, 4) == 0
    assert append(b=batch(rows=0), a=append_args(q=None, k=None, v=None)) == _lib.ANE_OK
    assert attend(b=batch(rows=0), a=attend_args(q=None, out=None)) == _lib.ANE_OK
    assert lib.ane_control_logits(logits_args(rows=0, logits=None), None) == _lib.ANE_OK
    refused(lib.ane_kv8_append(None, batch(), append_args(), None), "no cache")
    refused(lib.ane_kv8_attend(cache(), batch(), None, None), "null")


@pytest.mark.parametrize("cls,pack", [(_lib.Kv8AppendArgs, _lib.pack_append), (_lib.Kv8AttendArgs, _lib.pack_attend),
                                      (_lib.LogitsArgs, _lib.pack_logits)])
def test_packed_arguments_are_the_structs(cls, pack):
    values = [7 * i + 1 for i in range(len(cls._fields_))]
    data = pack(*values)
    assert len(data) == C.sizeof(cls)
    a = cls.from_buffer_copy(data)
    assert [getattr(a, n) for n, _ in cls._fields_] == values


class Host:
    """A batch whose arrays are host memory, for the index walk."""

    def __init__(self, table, start, offsets, rows, page, pages):
        self.arrays = [np.ascontiguousarray(x, dtype=np.int32) for x in (table, start, offsets)]
        t, s, o = (x.ctypes.data for x in self.arrays)
        n, w = self.arrays[0].shape
        self.b = batch(table=t, start=s, offsets=o, table_stride=w, table_pages=w, nseq=n, rows=rows)
        self.c = cache(page_tokens=page, pages=pages)
        self.page, self.pages, self.rows, self.width = page, pages, rows, w

    def items(self, tile, of_pages):
        out = (C.c_int32 * 6)()
        k, n, got = 0, 1, []
        while k < n:
            rc = lib.ane_debug_kv8_item(self.c, self.b, tile, of_pages, k, out)
            if rc == _lib.ANE_ERR_ARG and k == 0:
                return got   # no items at all
            assert rc == _lib.ANE_OK, lib.ane_op_last_error()
            n = out[5]
            got.append(tuple(out[:5]))
            k += 1
        assert lib.ane_debug_kv8_item(self.c, self.b, tile, of_pages, n, out) == _lib.ANE_ERR_ARG
        return got

    def within(self, items):
        for seq, row, n, pos, page in items:
            assert 0 <= seq < self.arrays[0].shape[0] and n >= 0
            assert 0 <= row and row + n <= self.rows
            assert 0 <= pos and pos + n <= self.width * self.page
            assert -1 <= page < self.pages


@pytest.mark.parametrize("nseq", [1, 2, 63, 64, 65, 700, 4097])
@pytest.mark.parametrize("page,tile", [(16, 1), (64, 5), (256, 16), (32, 64)])
def test_every_row_is_in_one_item(nseq, page, tile):
    r = np.random.default_rng(nseq * 1000 + page + tile)
    n = r.integers(0, 4 if nseq > 100 else min(150, 8 * page), nseq)
    n[r.random(nseq) < 0.2] = 0
    n[r.random(nseq) < 0.3] = 1
    width = 8
    start = r.integers(0, width * page - n + 1)
    offsets = np.concatenate([[0], np.cumsum(n)])
    table = r.permutation(nseq * width).reshape(nseq, width)
    h = Host(table, start, offsets, int(offsets[-1]) + 3, page, nseq * width)
    for of_pages in (0, 1, 3):
        items = [i for i in h.items(tile, of_pages) if i[2]]
        h.within(items)
        seen = np.zeros(h.rows, int)
        for seq, row, cnt, pos, pid in items:
            seen[row:row + cnt] += 1
            assert offsets[seq] <= row and row + cnt <= offsets[seq + 1]
            assert pos == start[seq] + row - offsets[seq]
            if of_pages:
                assert pos // page == (pos + cnt - 1) // page and pid == table[seq, pos // page]
            else:
                assert cnt <= tile and (row - offsets[seq]) % tile == 0
        assert (seen[:offsets[-1]] == 1).all() and (seen[offsets[-1]:] == 0).all()


@pytest.mark.parametrize("nseq", [1, 2, 9, 33, 64])
@pytest.mark.parametrize("tile", [1, 5, 16])
def test_longest_contexts_come_first(nseq, tile):
    """The tiles of every sequence, those of the one that ends last first (of
    two that end alike, the first), each one's own from its last on; empty
    items behind them."""
    r = np.random.default_rng(nseq * 100 + tile)
    page, width = 32, 12
    n = r.integers(0, 90, nseq)
    n[r.random(nseq) < 0.2] = 0
    n[0] = 7
    start = r.integers(0, width * page - n + 1)
    if nseq > 2:
        start[2] = start[1] + n[1] - n[2] if start[1] + n[1] >= n[2] else start[2]
    offsets = np.concatenate([[0], np.cumsum(n)])
    table = r.permutation(nseq * width).reshape(nseq, width)
    h = Host(table, start, offsets, int(offsets[-1]) + 3, page, nseq * width)
    items = h.items(tile, 2)
    h.within(items)
    want = []
    for i in sorted(range(nseq), key=lambda i: (-(start[i] + n[i]), i)):
        for t in reversed(range(0, int(n[i]), tile)):
            want.append((i, offsets[i] + t, min(tile, n[i] - t), start[i] + t))
    assert [i[:4] for i in items[:len(want)]] == want
    assert all(i[2] == 0 for i in items[len(want):])


def test_longest_contexts_of_many_sequences_refused():
    h = Host(np.zeros((65, 2), int), np.zeros(65, int), np.arange(66), 65, 16, 2)
    out = (C.c_int32 * 6)()
    refused(lib.ane_debug_kv8_item(h.c, h.b, 4, 2, 0, out), "nseq=65")


@pytest.mark.parametrize("seed", range(40))
def test_nonsense_stays_in_range(seed):
    r = np.random.default_rng(seed)
    nseq = int(r.integers(1, 200))
    page = int(r.choice([16, 64, 256]))
    rows = int(r.integers(1, 2000))
    wild = np.array([-2**31, -5, -1, 0, 1, 7, 2**30, 2**31 - 1])

    def some(shape, hi):
        x = r.integers(-3, hi, shape)
        return np.where(r.random(shape) < 0.2, r.choice(wild, shape), x)

    h = Host(some((nseq, 4), 12), some(nseq, 5 * page), some(nseq + 1, rows + 50), rows, page, 10)
    for tile in (1, 5, 64):
        h.within(h.items(tile, 0))
        if nseq <= 64:
            h.within(h.items(tile, 2))
    h.within(h.items(1, 1))
    h.within(h.items(1, 3))


def test_positions_past_the_table_are_not_taken():
    h = Host([[0, 1], [2, 3]], [30, 40], [0, 10, 20], 20, 16, 4)
    items = [i for i in h.items(64, 0) if i[2]]
    assert items == [(0, 0, 2, 30, -1)]   # positions 30 and 31; sequence 1 starts behind the table's 32
    assert [i for i in h.items(1, 1) if i[2]] == [(0, 0, 2, 30, 1)]
