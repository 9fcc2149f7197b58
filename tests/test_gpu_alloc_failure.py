"""Device memory that runs out: what the call promises holds, and calls behind it
do not report the failure again (it would stay the thread's last HIP error,
which every launch looks at)."""
import numpy as np
import pytest

import ane
from ane import _lib
from ane.moe import MoeConfig, MoeLayer, moe_param_count
from test_gpu_decode_serve import run, setup

pytestmark = pytest.mark.gpu


@pytest.fixture
def fail():
    lib = _lib.load()
    yield lib.ane_decode_debug_allocs
    lib.ane_decode_debug_allocs(0, 0)


@pytest.mark.parametrize("first", range(11))
@pytest.mark.parametrize("a,b", [(0, 32), (32, 0), (64, 16)])
def test_set_cache_goes_back_to_what_was_there(a, b, first, fail):
    cfg = ane.tiny_decode()
    p, prefix, forced = setup(cfg, 2, 64, 2, 91)
    dec = ane.Decoder(cfg, p, max_batch=2, max_ctx=128, page_tokens=a)
    try:
        want = run(dec, prefix, forced)
        fail(first, 1)
        try:
            dec.SetCache(b)
            fail(0, 0)
            assert first >= (10 if b else 2)     # there are not that many
            dec.SetCache(a)
        except ane.EngineError as e:
            assert "out of memory" in str(e) and first < (10 if b else 2)
        np.testing.assert_array_equal(run(dec, prefix, forced), want)
        dec.SetCache(b)
        assert np.isfinite(run(dec, prefix, forced)).all()
    finally:
        dec.Close()


@pytest.mark.parametrize("a,b", [(0, 32), (32, 0)])
def test_no_memory_for_either_cache_closes_the_decoder_alone(a, b, fail):
    cfg = ane.tiny_decode()
    p, prefix, forced = setup(cfg, 2, 64, 1, 92)
    dec, other = (ane.Decoder(cfg, p, max_batch=2, max_ctx=128, page_tokens=a) for _ in range(2))
    try:
        want = run(other, prefix, forced)
        fail(0, 2)
        with pytest.raises(ane.EngineError, match="no memory for either"):
            dec.SetCache(b)
        with pytest.raises(ane.EngineError):
            dec.Prefill(prefix)
        np.testing.assert_array_equal(run(other, prefix, forced), want)
    finally:
        dec.Close()
        other.Close()


def test_workspace_that_cannot_be_had(fail):
    """The attention's workspace is allocated by the first call that needs it."""
    cfg = ane.tiny_decode()
    p, prefix, forced = setup(cfg, 2, 64, 1, 93)
    dec = ane.Decoder(cfg, p, max_batch=2, max_ctx=4200, page_tokens=64)
    try:
        dec.Prefill(prefix)
        fail(0, 1)
        with pytest.raises(ane.EngineError, match="out of memory"):
            dec.Step(forced[:, 0])
        lg = dec.Step(forced[:, 0], want_logits=True)[1]
        np.testing.assert_array_equal(lg, run(dec, prefix, forced)[:, 1])
    finally:
        dec.Close()


@pytest.mark.parametrize("first", [0, 5, 12, 30])
def test_open_that_fails(first, fail):
    cfg = ane.tiny_decode()
    p, prefix, forced = setup(cfg, 2, 64, 1, 94)
    fail(first, 1)
    with pytest.raises(ane.EngineError, match="out of memory"):
        ane.Decoder(cfg, p, max_batch=2, max_ctx=128)
    dec = ane.Decoder(cfg, p, max_batch=2, max_ctx=128)
    try:
        assert np.isfinite(run(dec, prefix, forced)).all()
    finally:
        dec.Close()


def test_moe_layer_too_large_to_open():
    """4 TB of activations: refused by the allocator; a small layer opens and
    runs behind it."""
    c = _lib.MoeCfg(1 << 20, 64, 2, 2, 1 << 20, 0)
    lib = _lib.load()
    h = _lib.C.c_void_p()
    assert lib.ane_moe_open(_lib.C.byref(c), _lib.C.byref(h)) == _lib.ANE_ERR_HIP
    assert b"out of memory" in lib.ane_moe_last_error(h)
    lib.ane_moe_destroy(h)
    cfg = MoeConfig(dim=64, hidden=64, experts=2)
    r = np.random.default_rng(95)
    m = MoeLayer(cfg, (r.standard_normal(moe_param_count(cfg)) * 0.05).astype(np.float32), max_tokens=64)
    try:
        m.Load(r.standard_normal((64, 64)).astype(np.float32))
        m.Run()
    finally:
        m.Close()


@pytest.mark.parametrize("first", range(8))
def test_controls_that_cannot_be_had_leave_nothing_behind(first, fail):
    """However often setting them fails, what was allocated for them is used by
    the call that succeeds."""
    cfg = ane.tiny_decode(vocab=4096)
    p, prefix, forced = setup(cfg, 2, 64, 1, 96)
    bias = np.zeros(cfg.vocab, np.float32)
    bias[77] = 1000
    dec, other = (ane.Decoder(cfg, p, max_batch=2, max_ctx=128) for _ in range(2))
    try:
        fail(0, 0)
        other.SetControls(bias=bias)
        want = fail(0, 0)
        got = 0
        for _ in range(3):
            fail(first, 1)
            with pytest.raises(ane.EngineError, match="out of memory"):
                dec.SetControls(bias=bias)
            got += fail(0, 0)
            first = 0
        dec.SetControls(bias=bias)
        assert got + fail(0, 0) == want
        assert (dec.Prefill(prefix)[0] == 77).all()
    finally:
        dec.Close()
        other.Close()


@pytest.mark.parametrize("which", ["forward", "backward", "offload"])
def test_seam_object_too_large_to_open(which):
    """Weights of 412 GB (dim 2^18) or an embedding of 4 TB: refused by
    the allocator; a small object opens behind it."""
    lib = _lib.load()
    C = _lib.C

    def open_(dim, hidden, heads, seq, vocab, w):
        h = C.c_void_p()
        p = w.ctypes.data_as(C.POINTER(C.c_float))
        if which == "offload":
            rc = lib.ane_offload_open(vocab, dim, seq, p, 0, C.byref(h))
        else:
            lw = _lib.LayerWeights(*[p] * 6)
            rc = getattr(lib, f"ane_layer_{which}_open")(dim, hidden, heads, seq, C.byref(lw), C.byref(h))
        return rc, h
    w = np.zeros(1 << 16, np.float32)      # never read by the first call
    rc, h = open_(1 << 18, 64, 1 << 12, 64, 1 << 23, w)
    assert rc == _lib.ANE_ERR_NOMEM and not h.value, lib.ane_seam_last_error()
    rc, h = open_(64, 64, 1, 64, 512, w)
    assert rc == _lib.ANE_OK, lib.ane_seam_last_error()
    getattr(lib, "ane_offload_destroy" if which == "offload" else f"ane_layer_{which}_destroy")(h)
