"""Outputs of the serving operators that overlap an input in part are refused;
those that are the input, or lie between its rows, are not."""
import ctypes as C

import numpy as np
import pytest

from ane import _lib
from test_serve_host import P16, append_args, attend_args, batch, cache, logits_args, refused

lib = _lib.load()


def share(a, b):
    return bool(lib.ane_debug_share_memory((C.c_int64 * 6)(*a), (C.c_int64 * 6)(*b)))


def bytes_of(t):
    at, rows, row, heads, head, width = t
    starts = (at + np.arange(rows)[:, None] * row + np.arange(heads)[None] * head).reshape(-1)
    return set((starts[:, None] + np.arange(width)[None]).reshape(-1).tolist())


@pytest.mark.parametrize("seed", range(30))
def test_shared_memory_is_what_the_bytes_say(seed):
    """Small tensors with strides of all kinds (0 and overlapping ones too), in
    either order, against the set of their bytes."""
    r = np.random.default_rng(seed)
    seen = [0, 0]
    for _ in range(300):
        ts = []
        row = int(r.integers(0, 40))
        for _ in range(2):
            if r.random() < 0.5:
                row = int(r.integers(0, 40))
            ts.append([1000 + int(r.integers(0, 120)), int(r.integers(1, 7)), row, int(r.integers(1, 5)),
                       int(r.integers(0, 90 if r.random() < 0.5 else 12)), int(r.integers(1, 7))])
        want = bool(bytes_of(ts[0]) & bytes_of(ts[1]))
        assert share(*ts) == want and share(ts[1], ts[0]) == want, ts
        seen[want] += 1
    assert min(seen) > 30


def test_large_tensors_through_each_other():
    """Queries and outputs in one buffer: [rows, 2, heads, 64], [rows, heads, 2,
    64], head-major, one behind the other; and one row further on."""
    n, h = 20000, 12
    at = 1 << 40
    for a, b in (((at, n, 4 * h * 64, h, 128, 128), (at + 2 * h * 64, n, 4 * h * 64, h, 128, 128)),
                 ((at, n, 4 * h * 64, h, 256, 128), (at + 128, n, 4 * h * 64, h, 256, 128)),
                 ((at, n, 256, h, n * 256, 128), (at + 128, n, 256, h, n * 256, 128)),
                 ((at, n, h * 128, h, 128, 128), (at + n * h * 128, n, 128, h, n * 128, 128))):
        assert not share(a, b) and not share(b, a)
        moved = (b[0] - 64, *b[1:])
        assert share(a, moved) and share(moved, a)
        assert share(a, a)


def test_append_refuses():
    for kw in (dict(q_out=P16 + 64 * 2), dict(q=P16 + 4096, q_out=P16 + 4096 - 256), dict(q=8 * P16, q_out=P16),
               dict(q=8 * P16, v=9 * P16, q_out=P16 + 16)):
        refused(lib.ane_kv8_append(cache(), batch(), append_args(**kw), None), "q_out overlaps")


def test_attend_refuses():
    for kw in (dict(out=P16 + 128), dict(out=P16 + 5 * 512 - 16), dict(out=P16, out_row=512), dict(q_row=0)):
        refused(lib.ane_kv8_attend(cache(), batch(), attend_args(**kw), None), "out overlaps q")


def test_controls_refuse():
    for kw in (dict(out=P16 + 4), dict(out=P16 + 396), dict(out=P16 - 4), dict(out=P16 + 400, logits_row=200)):
        refused(lib.ane_control_logits(logits_args(**kw), None), "out overlaps logits")
