"""Attention over the paged 8-bit cache where one key takes most of the weight
and tens of thousands share the rest."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import ane  # noqa: E402
from test_gpu_serve import DEV, batch_of  # noqa: E402


@pytest.mark.parametrize("top", [0, 7, -1])
@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("n,new,hints", [(60000, 1, {}), (60000, 1, dict(max_len=1000, max_new=1)), (777, 1, {}),
                                         (20000, 40, {}), (9000, 700, {})])
def test_small_weights_of_many_keys_count(n, new, hints, dh, top):
    """Key `top` scores s above all others, whose weights are e^-s of its own:
    a row of m others has m e^-s / (1 + m e^-s) of their value (the top key's
    is 0).  For every s in steps of 0.5 up to 20 (weights down to 2^-28).

    Weights are fp16 with the largest at 2^7 or more: each off by 2^-11 of
    itself, or, where it is below 2^-14 (2^-21 of the largest), by 2^-25, 2^-32
    of the largest.  Then the sums over m keys in fp32 (2^-24 each), a score off
    by 2^-24 times dh + 2 roundings of s, and the output's rounding."""
    P, kvh, heads = 256, 1, 4
    pages = (n + new + P - 1) // P
    top = top % n
    cache = ane.KVCache8.Empty(pages, kvh, dh, P, DEV)
    k = cache.k.view(torch.uint8)
    # every value 1 (code 0x38) but the top key's; every key 0 but the top one, all of it 1
    cache.v.view(torch.uint8).fill_(0x38)
    cache.v.view(torch.uint8)[top // P, :, top % P // 16, top % 16 // 4, :, :, top % 4] = 0
    k[top // P, :, top % P] = 0x38
    table = np.arange(pages)[None]
    b = batch_of(table, np.array([n]), np.array([0, new]), new, **hints)
    for first in np.arange(0.5, 20, 2.0):
        s = first + 0.5 * np.arange(heads)          # a score for each head
        x = np.float16(s * 8 / dh)                  # q . k = dh x, scale 1 / 8
        q = torch.from_numpy(np.repeat(x[None, :, None], dh, -1).repeat(new, 0)).to(DEV)
        got = cache.Attend(b, q, scale=0.125).double().cpu().numpy()
        s = x.astype(np.float64) * dh / 8
        m = n + np.arange(new)[:, None] * 1.0   # keys but the top one, of each row
        w = np.exp(-s)[None]
        want = (m * w / (1 + m * w))[:, :, None]
        ds = (dh + 2) * 2.0 ** -24 * s + 2.0 ** -23
        tail = (m * 2.0 ** -32 / (1 + m * w))[:, :, None]
        tol = want * ((2 * ds)[None, :, None] + 2 * 2.0 ** -11 + m[:, :, None] * 2.0 ** -23 + 2.0 ** -11) + tail + 2.0 ** -25
        err = np.abs(got - want)
        print(n, new, dh, "s", s, "worst error over tolerance", (err / tol).max(), "value", want[-1, :, 0])
        assert (err <= tol).all()
