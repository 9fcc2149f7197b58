"""Scales of the attention that cannot be used are refused in the operator's own
manner, whatever kind of number they are."""
import ctypes as C
import types

import pytest

import ane
from ane import _lib, serve
from test_serve_host import attend_args, batch, cache, refused

lib = _lib.load()


@pytest.mark.parametrize("scale", [3e38, -3e38, 2.4e38])
def test_scale_whose_exponent_base_2_is_infinite(scale):
    """scale * log2(e) multiplies the scores: past fp32 it would make NaN of
    scores of 0."""
    refused(lib.ane_kv8_attend(cache(), batch(), attend_args(q=1 << 24, scale=scale), None), "scale=")


class FakeTensor:
    """What the checks ask of a tensor; never followed."""

    def __init__(self, *shape):
        self.shape = shape

    def stride(self):
        return (self.shape[1] * self.shape[2], self.shape[2], 1)

    def data_ptr(self):
        return 1 << 20


@pytest.mark.parametrize("scale", [1e39, -1e300, "0.1", 10**400], ids=["large", "below", "text", "whole"])
def test_scale_that_is_no_fp32_number(scale):
    c = serve.KVCache8.__new__(serve.KVCache8)
    c._lib, c.device, c.kv_heads, c.page_tokens, c.head_dim = lib, "cuda:0", 2, 16, 64
    c._rows = lambda op, name, t, batch, heads=None: (t.data_ptr(), *t.stride()[:2])
    held = cache(), batch()
    c._at, c._attend, c._stream, c._index = C.addressof(held[0]), _lib.plain(lib, "ane_kv8_attend"), lambda i: None, 0
    b = types.SimpleNamespace(device="cuda:0", rows=5, _ws={(2, 16, 64, 4): 0}, _at=C.addressof(held[1]))
    t = FakeTensor(5, 4, 64)
    with pytest.raises(ane.EngineError, match="scale="):
        c.Attend(b, t, t, scale)
