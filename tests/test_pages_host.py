"""Beam search, the tables of the pages and the choice of pages without a GPU:
what they refuse, and the argument structs."""
import ctypes as C
import struct

import numpy as np
import pytest

import pages_ref as ref
from ane import _lib

lib = _lib.load()
P16 = 0x10000   # an aligned address that is never followed: every call below is refused, or has no rows
FAR = 1 << 24


def refused(rc, *words):
    assert rc == _lib.ANE_ERR_ARG
    msg = lib.ane_op_last_error().decode()
    assert msg.startswith("storiesane "), msg
    for w in words:
        assert w in msg, msg


def cache(**kw):
    f = dict(k=P16, v=P16, k_exp=P16, v_exp=P16, pages=4, page_tokens=64, kv_heads=2, head_dim=64, device=0)
    f.update(kw)
    return _lib.Kv8Cache(**f)


def batch(**kw):
    f = dict(table=P16, start=P16, offsets=P16, table_stride=3, table_pages=3, nseq=2, rows=5, max_len=0, max_new=0)
    f.update(kw)
    return _lib.Kv8Batch(**f)


def beam_args(**kw):
    f = dict(logits=P16, scores=2 * FAR, weights=3 * FAR, finished=4 * FAR, tokens=5 * FAR, parents=6 * FAR,
             scores_out=7 * FAR, finished_out=8 * FAR, history=9 * FAR, lengths=10 * FAR, logits_row=100, history_row=9,
             requests=2, beams=3, vocab=100, eos=7, history_max=9, half=0, device=0, ws=P16, ws_bytes=1 << 30)
    f.update(kw)
    return _lib.BeamArgs(**f)


def beam(**kw):
    return lib.ane_beam_select(beam_args(**kw), None)


@pytest.mark.parametrize("kw, words", [
    (dict(requests=-1), ("requests=-1",)), (dict(beams=0), ("beams=0",)), (dict(beams=33), ("beams=33", "1..32")),
    (dict(vocab=0), ("vocab=0",)), (dict(vocab=65536), ("vocab=65536",)),
    (dict(requests=32768, beams=2), ("65535 rows",)),
    (dict(logits=None), ("null buffer",)), (dict(scores=None), ("null buffer",)), (dict(tokens=None), ("null buffer",)),
    (dict(parents=None), ("null buffer",)), (dict(scores_out=None), ("null buffer",)),
    (dict(finished=None), ("eos=7",)), (dict(finished_out=None), ("go together",)),
    (dict(eos=-1), ("go together",)), (dict(eos=100), ("eos=100",)),
    (dict(finished=None, finished_out=None), ("eos=7",)),
    (dict(history=None), ("history",)), (dict(lengths=None), ("without lengths",)),
    (dict(history_max=-1), ("history_max=-1",)), (dict(history_row=8), ("stride 8",)),
    (dict(history=None, lengths=None), ("history_max=9",)),
    (dict(logits_row=99), ("logits_row=99",)),
    (dict(ws=None), ("workspace of 0",)), (dict(ws=P16 + 8), ("16-byte",)), (dict(ws_bytes=8), ("workspace of 8",)),
    (dict(tokens=6 * FAR + 4), ("overlaps",)), (dict(scores_out=2 * FAR + 4), ("scores_out", "scores")),
    (dict(scores_out=3 * FAR), ("weights",)), (dict(finished_out=4 * FAR + 1), ("finished",)),
    (dict(tokens=P16 + 40), ("logits",)), (dict(lengths=9 * FAR + 10), ("history",)),
    (dict(history=P16 + 100), ("logits",)), (dict(scores_out=4 * FAR - 4), ("finished",)),
])
def test_beam_select_refuses(kw, words):
    refused(beam(**kw), "beam select", *words)


def test_beam_select_of_nothing():
    assert beam(requests=0, logits=None, ws=None) == _lib.ANE_OK
    refused(lib.ane_beam_select(None, None), "null arguments")
    assert lib.ane_beam_select_workspace(0, 4, 1000, 0) >= 0
    assert lib.ane_beam_select_workspace(3, 4, 1000, 1) > 0
    refused(lib.ane_beam_select_workspace(1, 40, 1000, 0), "beams=40")


BOUNDS = dict(box=P16, unit=P16)


def bounds(**kw):
    return _lib.Kv8Bounds(**{**BOUNDS, **kw})


def test_bound_refuses():
    refused(lib.ane_kv8_bound(cache(), bounds(box=None), batch(), None), "kv8 bound", "null bounds")
    refused(lib.ane_kv8_bound(cache(), bounds(unit=None), batch(), None), "null bounds")
    refused(lib.ane_kv8_bound(cache(), bounds(box=P16 + 8), batch(), None), "16-byte")
    refused(lib.ane_kv8_bound(cache(), None, batch(), None), "null bounds")
    refused(lib.ane_kv8_bound(None, bounds(), batch(), None), "no cache")
    refused(lib.ane_kv8_bound(cache(page_tokens=48), bounds(), batch(), None), "page_tokens=48")
    assert lib.ane_kv8_bound(cache(), bounds(), batch(nseq=0, rows=0), None) == _lib.ANE_OK


def select_args(**kw):
    f = dict(q=P16, blocks=FAR, q_row=256, q_head=64, heads=4, count=3, first=1, recent=1, ws=None, ws_bytes=0)
    f.update(kw)
    return _lib.Kv8SelectArgs(**f)


@pytest.mark.parametrize("kw, words", [
    (dict(q=None), ("null buffer",)), (dict(blocks=None), ("null buffer",)), (dict(q=P16 + 2), ("16-byte",)),
    (dict(q_row=260), ("260",)), (dict(q_head=-8), ("-8",)), (dict(heads=3), ("heads=3",)), (dict(heads=0), ("heads=0",)),
    (dict(heads=66), ("heads=66",)), (dict(count=0), ("count=0",)), (dict(count=65537), ("count=65537",)),
    (dict(first=-1), ("first=-1",)), (dict(recent=-1), ("recent=-1",)), (dict(first=2, recent=2), ("first=2 recent=2",)),
    (dict(blocks=P16 + 16), ("overlaps",)),
])
def test_select_refuses(kw, words):
    refused(lib.ane_kv8_select(cache(), bounds(), batch(), select_args(**kw), None), "kv8 select", *words)


def test_select_of_nothing_and_attend_blocks_refuse():
    assert lib.ane_kv8_select(cache(), bounds(), batch(nseq=0, rows=0), select_args(q=None), None) == _lib.ANE_OK
    refused(lib.ane_kv8_select(cache(), bounds(), batch(), None, None), "null arguments")
    refused(lib.ane_kv8_select_workspace(cache(), batch(), 4, 0), "count=0")
    a = _lib.Kv8AttendArgs(q=P16, out=2 * FAR, q_row=256, q_head=64, out_row=256, out_head=64, heads=4, scale=0.125,
                           ws=P16, ws_bytes=1 << 40)
    refused(lib.ane_kv8_attend_blocks(cache(), batch(), a, None, 3, None), "null buffer")
    refused(lib.ane_kv8_attend_blocks(cache(), batch(), a, P16, 0, None), "count=0")
    refused(lib.ane_kv8_attend_blocks(cache(), batch(), a, 2 * FAR + 64, 3, None), "out overlaps blocks")
    refused(lib.ane_kv8_attend_blocks_workspace(cache(), batch(), 4, 70000), "count=70000")
    refused(lib.ane_kv8_attend_blocks_workspace(cache(), batch(), 5, 7), "heads=5")
    assert lib.ane_kv8_attend_blocks_workspace(cache(), batch(), 4, 4) == 0
    assert lib.ane_kv8_attend_blocks_workspace(cache(), batch(), 4, 100) > 0
    assert lib.ane_kv8_attend_blocks(cache(), batch(nseq=0, rows=0), a, None, 3, None) == _lib.ANE_OK


def test_select_of_long_contexts_wants_a_workspace():
    long = batch(table_pages=1024, table_stride=1024)
    assert lib.ane_kv8_select_workspace(cache(), long, 4, 3) == 5 * 2 * 1024 * 4
    assert lib.ane_kv8_select_workspace(cache(), batch(table_pages=1023, table_stride=1023), 4, 3) == 0
    for ws, n in ((None, 1 << 20), (P16, 5 * 2 * 1024 * 4 - 1), (P16 + 8, 1 << 20)):
        refused(lib.ane_kv8_select(cache(), bounds(), long, select_args(ws=ws, ws_bytes=n), None), "workspace of")


def test_more_rows_than_a_launch_takes():
    big = cache(kv_heads=1024)
    wide = dict(q_row=16 * 1024 * 64, heads=1024 * 16, blocks=1 << 50)
    many = batch(rows=1 << 16)
    refused(lib.ane_kv8_select(big, bounds(), many, select_args(**wide), None), "rows=65536 are too many")
    refused(lib.ane_kv8_select_workspace(big, many, 1024 * 16, 7), "rows=65536 are too many")
    assert lib.ane_kv8_select_workspace(big, batch(rows=1 << 15), 1024 * 16, 7) == 0
    a = _lib.Kv8AttendArgs(q=P16, out=1 << 50, q_row=16 * 1024 * 64, q_head=64, out_row=16 * 1024 * 64, out_head=64,
                           heads=1024 * 16, scale=0.125, ws=P16, ws_bytes=1 << 60)
    refused(lib.ane_kv8_attend_blocks(big, batch(rows=1 << 14), a, P16, 30, None), "rows=16384 nseq=2 are too many")
    assert lib.ane_kv8_attend_blocks_workspace(big, batch(rows=1 << 13), 1024 * 16, 3) == 0
    refused(lib.ane_kv8_bound(cache(page_tokens=16), bounds(), batch(nseq=65536, rows=1 << 30), None),
            "rows=1073741824 are too many")


def pool(layers=None, refs=3 * FAR, with_bounds=None):
    layers = layers or [cache(), cache()]
    arr = (_lib.Kv8Cache * len(layers))(*layers)
    bnd = None if with_bounds is None else (_lib.Kv8Bounds * len(layers))(*with_bounds)
    return _lib.Kv8Pool(arr, bnd, refs, len(layers))


def fork_args(**kw):
    f = dict(table=FAR, start=4 * FAR, parents=5 * FAR, news=6 * FAR, missing=7 * FAR, table_stride=5, table_pages=4,
             nseq=3, new_tokens=0, ws=P16, ws_bytes=1 << 30)
    f.update(kw)
    return _lib.Kv8ForkArgs(**f)


@pytest.mark.parametrize("kw, words", [
    (dict(table=None), ("null table",)), (dict(start=None), ("null buffer",)), (dict(missing=None), ("null buffer",)),
    (dict(nseq=-1), ("nseq=-1",)), (dict(nseq=65537), ("nseq=65537",)), (dict(table_pages=0), ("table_pages=0",)),
    (dict(table_pages=6), ("stride 5",)), (dict(table_pages=1 << 25, table_stride=1 << 25), ("tokens",)),
    (dict(nseq=65536, table_pages=1 << 20, table_stride=1 << 20), ("entries",)),
    (dict(news=None, new_tokens=-1), ("new_tokens=-1",)), (dict(ws=None), ("workspace",)), (dict(ws_bytes=16), ("workspace",)),
    (dict(ws=P16 + 4), ("16-byte",)), (dict(parents=4 * FAR), ("parents overlaps start",)),
    (dict(missing=3 * FAR + 4), ("overlaps",)), (dict(start=FAR + 16), ("overlaps",)),
])
def test_fork_refuses(kw, words):
    refused(lib.ane_kv8_fork(pool(), fork_args(**kw), None), "kv8 fork", *words)


def test_pools_refuse():
    for bad, words in ((_lib.Kv8Pool(None, None, P16, 2), "no pool"),
                       (pool([cache(), cache(pages=5)]), "layer 1 differs"),
                       (pool([cache(), cache(device=1)]), "layer 1 differs"),
                       (pool([cache(k=None)]), "null cache buffer"), (pool([cache(kv_heads=0)]), "kv_heads=0"),
                       (pool(with_bounds=[bounds(), bounds(unit=None)]), "box without unit"),
                       (pool(with_bounds=[bounds(box=P16 + 4), bounds()]), "16-byte")):
        refused(lib.ane_kv8_fork(bad, fork_args(), None), words)
        refused(lib.ane_kv8_fork_workspace(bad, 3, 4), words)
        refused(lib.ane_kv8_compact_workspace(bad), words)
        refused(lib.ane_kv8_copy(bad, pool(), _lib.Kv8CopyArgs(P16, P16, None, 1), None), words)
        refused(lib.ane_kv8_copy(pool(), bad, _lib.Kv8CopyArgs(P16, P16, None, 1), None), words)
    refused(lib.ane_kv8_fork(pool(refs=None), fork_args(), None), "null refs")
    refused(lib.ane_kv8_fork(None, fork_args(), None), "no pool")
    refused(lib.ane_kv8_fork(pool(), None, None), "null arguments")
    assert lib.ane_kv8_fork_workspace(pool(with_bounds=[bounds(), _lib.Kv8Bounds()]), 3, 4) > 0


def compact_args(**kw):
    f = dict(table=FAR, moved=2 * FAR, table_stride=5, table_pages=4, nseq=3, ws=P16, ws_bytes=1 << 30)
    f.update(kw)
    return _lib.Kv8CompactArgs(**f)


@pytest.mark.parametrize("kw, words", [
    (dict(moved=None), ("null",)), (dict(table=None), ("null table",)), (dict(table_stride=3), ("stride 3",)),
    (dict(ws_bytes=0), ("workspace",)), (dict(moved=3 * FAR + 4), ("overlaps",)), (dict(moved=FAR + 4), ("overlaps",)),
])
def test_compact_refuses(kw, words):
    refused(lib.ane_kv8_compact(pool(), compact_args(**kw), None), "kv8 compact", *words)


def test_copy_refuses():
    args = _lib.Kv8CopyArgs(P16, P16, None, 2)
    for other in ([cache()], [cache(page_tokens=32)] * 2, [cache(kv_heads=1)] * 2, [cache(head_dim=128)] * 2):
        refused(lib.ane_kv8_copy(pool(), pool(other), args, None), "kv8 copy", "differ")
    refused(lib.ane_kv8_copy(pool(), pool(), None, None), "null arguments")
    refused(lib.ane_kv8_copy(pool(), pool(), _lib.Kv8CopyArgs(None, P16, None, 2), None), "null buffer")
    refused(lib.ane_kv8_copy(pool(), pool(), _lib.Kv8CopyArgs(P16, None, None, 2), None), "null buffer")
    refused(lib.ane_kv8_copy(pool(), pool(), _lib.Kv8CopyArgs(P16, P16, None, -1), None), "n=-1")
    assert lib.ane_kv8_copy(pool(), pool([cache(pages=9)] * 2), _lib.Kv8CopyArgs(None, None, None, 0), None) == _lib.ANE_OK


@pytest.mark.parametrize("cls, fmt", [
    (_lib.BeamArgs, "10P2q7iPq"), (_lib.Kv8SelectArgs, "2P2q4iPq"), (_lib.Kv8ForkArgs, "5P4iPq"),
    (_lib.Kv8CompactArgs, "2P3iPq"), (_lib.Kv8CopyArgs, "3Pi4x")])
def test_packed_arguments_are_the_structs(cls, fmt):
    assert struct.calcsize(fmt) == C.sizeof(cls)
    values = [i + 1 for i in range(len(cls._fields_))]
    packed = cls.from_buffer_copy(struct.pack(fmt, *values))
    assert [getattr(packed, n) for n, _ in cls._fields_] == values


def test_reference_fork_keeps_counts():
    """The plain fork used by the GPU tests: refs are the entries that name a page."""
    r = np.random.default_rng(3)
    P, width, pages, nseq = 16, 6, 60, 8
    table = np.full((nseq, width), -1, np.int32)
    start, refs = np.zeros(nseq, np.int32), np.zeros(pages, np.int32)
    table, start, refs, missing, copies = ref.fork(table, start, refs, P, None, [20] * nseq)
    assert missing == 0 and not copies and (refs[:16] == 1).all()
    start[:] = 20
    for _ in range(20):
        parents = r.integers(-1, nseq, nseq)
        before = (table.copy(), start.copy())
        table, start, refs, missing, copies = ref.fork(table, start, refs, P, parents, [1] * nseq)
        assert missing == 0
        np.testing.assert_array_equal(refs, np.bincount(table[table >= 0], minlength=pages))
        for i in range(nseq):   # nobody else holds the page that is written next
            assert refs[table[i, start[i] // P]] == 1
            if parents[i] >= 0:
                full = before[1][parents[i]] // P
                np.testing.assert_array_equal(table[i, :full], before[0][parents[i], :full])
        start = np.minimum(start + 1, 40).astype(np.int32)
