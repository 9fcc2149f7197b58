"""A Step or Generate call whose chain fails part of the way is redone with one
launch per GEMM from where it began: over either cache, bit for bit what a call
gives whose chain failed before it had done anything."""
import numpy as np
import pytest

import ane
from test_gpu_decode_serve import setup

pytestmark = pytest.mark.gpu


QUIET, LOUD = 5, 700


def model(before, seed):
    """A model in which the token LOUD alone has an embedding along dimension 0,
    which layer 0's gain makes 200 times larger: its keys and values are some
    hundred times any other token's.  The prompt is without it; controls choose
    QUIET for some 20 steps, by its bias, and then, QUIET repeated so often,
    LOUD."""
    cfg = ane.tiny_decode()
    p, prefix, forced = setup(cfg, 3, 64, before + 3, seed)
    w = ane.views(cfg, p)
    w["embed"][:, 0] = 0
    w["embed"][LOUD, 0] = 1
    w["layers.0.g_att"][0] = 200
    for t in (prefix, forced):
        t[t == LOUD] = QUIET
    bias = np.zeros(cfg.vocab, np.float32)
    bias[QUIET], bias[LOUD] = 200, 180
    return cfg, p, prefix, forced, dict(bias=bias, frequency=np.ones(3, np.float32))


def life(cfg, p, prefix, forced, controls, page, before, fail, steps):
    """Prefill, `before` steps, a Generate whose chain fails at step `fail`
    (None: a decoder without the chain), and steps behind it."""
    dec = ane.Decoder(cfg, p, max_batch=3, max_ctx=256, page_tokens=page)
    try:
        dec.DebugFillCache(0xFF)
        dec.SetControls(**controls)
        dec.Prefill(prefix)
        for i in range(before):
            dec.Step(forced[:, i])
        if fail is not None:
            assert dec.FusedChain() == 1
            dec.DebugFailChain(fail)
        out = [dec.Generate(steps)]
        assert dec.FusedChain() == (0 if fail is None else 2)
        for i in range(before, forced.shape[1]):
            out.append(dec.Step(forced[:, i], want_logits=True)[1])
        return out
    finally:
        dec.Close()


@pytest.mark.parametrize("fail", [1, 59, 119])
@pytest.mark.parametrize("page", [0, 16, 64, 256])
@pytest.mark.parametrize("before", [0, 5])
def test_redone_generate_is_as_if_never_tried(before, page, fail, monkeypatch):
    """120 steps behind a prompt of 64 and `before` steps: by the failing step
    the good ones have raised exponents of the 8-bit cache's pages, and rounded
    rows from before the call again."""
    m = model(before, 81)
    got = life(*m, page, before, fail, 120)
    want = life(*m, page, before, 0, 120)
    first = (got[0] == LOUD).argmax(1)
    assert (got[0] == LOUD).any(1).all() and first.min() > 5 and first.max() < 50, first
    if not before:                    # the same form throughout: also what a decoder without the chain gives
        monkeypatch.setenv("ANE_DEC_TAIL", "0")
        for a, b in zip(want, life(*m, page, before, None, 120)):
            np.testing.assert_array_equal(a, b)
    for a, b in zip(got, want):
        np.testing.assert_array_equal(a, b)


def test_redone_step_and_a_generate_that_does_not_reach_the_failure():
    cfg = ane.tiny_decode()
    p, prefix, forced = setup(cfg, 2, 64, 2, 82)
    dec = ane.Decoder(cfg, p, max_batch=2, max_ctx=256, page_tokens=16)
    try:
        dec.Prefill(prefix)
        dec.DebugFailChain(9)
        dec.Generate(5)
        dec.Generate(20)              # the request was for the call before
        assert dec.FusedChain() == 1
        dec.DebugFailChain(0)
        _, lg = dec.Step(forced[:, 0], want_logits=True)
        assert dec.FusedChain() == 2 and np.isfinite(lg).all() and dec.Position() == 64 + 26
    finally:
        dec.Close()
