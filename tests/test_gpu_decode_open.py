"""What a decoder allocates for its cache when it opens."""
import ctypes as C

import numpy as np
import pytest

import ane
from ane import _lib
from test_gpu_decode_serve import run, setup


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 64, 256])
def test_open_with_the_8_bit_cache_never_holds_the_fp16_one(page):
    """The 8-bit cache takes half the fp16 one's bytes, and for each page of
    codes (kv_heads * page * 64 bytes a side) an exponent a head and side, four
    bytes of table, and once per sequence a page kept by a call; the rest of
    an open decoder is the same."""
    cfg = ane.tiny_decode()
    L, B, KV, ctx = cfg.layers, 8, cfg.kv_heads, 16384
    p, prefix, forced = setup(cfg, B, 64, 1, 97)
    lib = _lib.load()
    took = []
    for page_tokens in (0, page):
        lib.ane_decode_debug_allocs(0, 0)
        dec = ane.Decoder(cfg, p, max_batch=B, max_ctx=ctx, page_tokens=page_tokens)
        try:
            took.append(lib.ane_decode_debug_allocs(0, 0))
            assert np.isfinite(run(dec, prefix, forced)).all()
        finally:
            dec.Close()
    fp16 = L * B * KV * ctx * 64 * 2 * 2
    pages = L * B * ctx // page
    eight = pages * KV * (page * 64 + 1) * 2
    more = pages * 4 + L * B * KV * (page * 64 + 1) * 2 + (1 << 20)   # table, kept pages; rows of a step
    assert took[0] - fp16 + eight <= took[1] <= took[0] - fp16 + eight + more


@pytest.mark.gpu
def test_opened_with_a_cache_or_switched_to_it_is_the_same():
    cfg = ane.tiny_decode()
    p, prefix, forced = setup(cfg, 2, 64, 3, 98)
    got = []
    for opened, switched in ((32, None), (0, 32), (64, 32), (32, 0), (0, None)):
        dec = ane.Decoder(cfg, p, max_batch=2, max_ctx=100, page_tokens=opened)
        try:
            if switched is not None:
                dec.SetCache(switched)
            got.append(run(dec, prefix, forced))
        finally:
            dec.Close()
    for i, j in ((0, 1), (0, 2), (3, 4)):
        np.testing.assert_array_equal(got[i], got[j])


@pytest.mark.parametrize("page", [-1, 8, 48, 512])
def test_open_refuses_other_page_sizes(page):
    """Before anything is done on a GPU."""
    cfg = ane.tiny_decode()
    lib = _lib.load()
    c = _lib.DecodeCfg(cfg.dim, cfg.hidden, cfg.heads, cfg.kv_heads, cfg.layers, cfg.vocab, 2, 128, 10000.0, 0)
    h = C.c_void_p()
    assert lib.ane_decode_open_cache(C.byref(c), page, C.byref(h)) == _lib.ANE_ERR_ARG
    assert f"page_tokens={page}".encode() in lib.ane_decode_last_error(h)
    lib.ane_decode_destroy(h)
    with pytest.raises(ane.EngineError, match=f"page_tokens={page}"):
        ane.Decoder(cfg, np.zeros(1, np.float32), page_tokens=page)
