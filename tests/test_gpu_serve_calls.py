"""Calls of the serving operators that the documentation allows: outputs in
place or between an input's rows, tokens without logits."""
import ctypes as C

import numpy as np
import pytest

import serve_ref as ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import ane  # noqa: E402
from ane import _lib  # noqa: E402
from test_gpu_serve import DEV, Pool, batch_of, dev, layout, rope_tables  # noqa: E402
from test_gpu_serve_pages import FORMS  # noqa: E402


@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("form", FORMS)
def test_attend_in_place_and_between_rows(form, dh):
    """out = q, and queries and outputs side by side in one buffer: the bits of
    a call with a tensor of its own."""
    lens, heads, kvh, hints = FORMS[form]
    r = np.random.default_rng(dh)
    table, start, offsets, pages = layout(r, lens, 32)
    rows = int(offsets[-1])
    c = Pool(r, pages, kvh, 32, dh).cache
    b = batch_of(table, start, offsets, rows, **hints)
    q = dev(r.standard_normal((rows, heads, dh)).astype(np.float16))
    want = c.Attend(b, q)
    both = torch.zeros((rows, 2, heads, dh), dtype=torch.float16, device=DEV)
    both[:, 1] = q
    assert torch.equal(c.Attend(b, both[:, 1], both[:, 0]), want) and torch.equal(both[:, 1], q)
    wide = torch.zeros((rows, heads, 2, dh), dtype=torch.float16, device=DEV)
    wide[:, :, 0] = q
    assert torch.equal(c.Attend(b, wide[:, :, 0], wide[:, :, 1]), want) and torch.equal(wide[:, :, 0], q)
    assert c.Attend(b, q, q) is q and torch.equal(q, want)
    with pytest.raises(ane.EngineError, match="out overlaps q"):
        c.Attend(b, both[:, 1], both.view(rows * 2, heads, dh)[:rows])


def test_append_queries_between_rows():
    r = np.random.default_rng(3)
    lens = [(30, 1), (0, 40), (15, 2), (63, 9)]
    table, start, offsets, pages = layout(r, lens, 32)
    rows = int(offsets[-1])
    cos, sin = (dev(t) for t in rope_tables(table.shape[1] * 32, 64))
    b = batch_of(table, start, offsets, rows)
    x = torch.zeros((rows, 16, 64), dtype=torch.float16, device=DEV)     # q | k | v | rotated q
    x[:, :10] = dev(r.standard_normal((rows, 10, 64)).astype(np.float16))
    c = Pool(r, pages, 2, 32, 64).cache
    y = x.clone()
    want = c.Append(b, x[:, :6], x[:, 6:8], x[:, 8:10], cos, sin)
    c.Append(b, x[:, :6], x[:, 6:8], x[:, 8:10], cos, sin, x[:, 10:])
    assert torch.equal(x[:, 10:], want) and torch.equal(x[:, :10], y[:, :10])
    with pytest.raises(ane.EngineError, match="q_out overlaps"):
        c.Append(b, x[:, :6], x[:, 6:8], x[:, 8:10], cos, sin, x[:, 4:10])


@pytest.mark.parametrize("rows,vocab", [(1, 70), (5, 32000), (200, 9001)])
def test_control_between_rows_and_tokens_alone(rows, vocab):
    r = np.random.default_rng(vocab)
    lg = r.standard_normal((rows, vocab)).astype(np.float32)
    hist = r.integers(0, vocab, (rows, 50)).astype(np.uint16)
    n = r.integers(0, 51, rows).astype(np.int32)
    rep = r.uniform(1, 2, rows).astype(np.float32)
    want, wt = ref.control(lg, hist, n, None, rep, None, None, None, None)
    both = torch.zeros((rows, 2, vocab), device=DEV)
    both[:, 0] = dev(lg)
    ctl = ane.LogitControls(vocab, repetition=dev(rep))
    h, nd, repd = dev(hist.view(np.int16)), dev(n), dev(rep)
    out, tok = ctl.Apply(both[:, 0], h, nd, out=both[:, 1])
    np.testing.assert_array_equal(out.cpu().numpy(), want)
    np.testing.assert_array_equal(tok.cpu().numpy(), wt)
    np.testing.assert_array_equal(both[:, 0].cpu().numpy(), lg)
    with pytest.raises(ane.EngineError, match="out overlaps logits"):
        ctl.Apply(both[:, 0], h, nd, out=both.view(rows, -1)[:, 1:vocab + 1])
    # out NULL: the tokens alone
    lib = _lib.load()
    x = dev(lg)
    tok.fill_(-5)
    size = lib.ane_control_logits_workspace(rows, vocab)
    ws = torch.empty(max(size, 16), dtype=torch.uint8, device=DEV)
    a = _lib.LogitsArgs(logits=x.data_ptr(), out=None, history=h.data_ptr(), lengths=nd.data_ptr(), prompts=None,
                        repetition=repd.data_ptr(), frequency=None, presence=None, bias=None, mask=None,
                        tokens=tok.data_ptr(), logits_row=vocab, out_row=0, history_row=50, bias_row=0, mask_row=0,
                        rows=rows, vocab=vocab, history_max=50, device=0, ws=ws.data_ptr(), ws_bytes=size)
    assert lib.ane_control_logits(C.byref(a), C.c_void_p(torch.cuda.current_stream().cuda_stream)) == _lib.ANE_OK
    np.testing.assert_array_equal(tok.cpu().numpy(), wt)
    assert torch.equal(x, dev(lg))
