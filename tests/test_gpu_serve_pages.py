"""Attention over the paged 8-bit cache where pages are not what their
neighbours suggest: pages that nothing was written to."""
import numpy as np
import pytest

import serve_ref as ref

torch = pytest.importorskip("torch")
pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore:overflow encountered", "ignore:invalid value")]

from test_gpu_serve import DEV, Pool, batch_of, dev, layout  # noqa: E402

FORMS = {
    # single tokens, whole and in parts; chunks; one long chunk in 48-row tiles; many prompts, a wave a tile
    "tokens": ([(776, 1), (0, 1), (15, 1), (100, 1)], 12, 4, dict(max_new=1, max_len=777)),
    "parts": ([(5000, 1), (16, 1)], 6, 2, dict(max_new=1, max_len=5001)),
    "chunks": ([(250, 23), (5, 33), (0, 1)], 6, 2, dict(max_new=33, max_len=273)),
    "long-chunk": ([(4090, 530)], 12, 4, dict(max_new=530, max_len=4620)),
    "many": ([(i % 7 * 9, 1 + i * 37 % 90) for i in range(60)], 16, 16, dict(max_new=90, max_len=144)),
}


@pytest.mark.parametrize("e", [-128, -127, 127])
@pytest.mark.parametrize("P", [16, 64])
@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("form", FORMS)
def test_unwritten_pages_take_no_part(form, dh, P, e):
    """Pages that no table names, the pool's first and last among them, hold
    NaN codes and exponents far outside the range; one page is missing.  The
    last step of 32 keys ends behind a sequence's last page.  Bit for bit what
    the same call gives where those pages hold zeros."""
    lens, heads, kvh, hints = FORMS[form]
    r = np.random.default_rng(P + dh)
    table, start, offsets, pages = layout(r, lens, P)
    table[table >= 0] += 1
    pages += 1
    table[0, 0] = pages + 3
    named = np.zeros(pages, bool)
    named[table[(table >= 0) & (table < pages)]] = True
    assert not named[0]
    q = dev(r.standard_normal((int(offsets[-1]), heads, dh)).astype(np.float16))
    got = []
    for code, exps in ((0, 0), (0x7f, e)):
        pool = Pool(np.random.default_rng(1), pages, kvh, P, dh)
        for x, fill in ((pool.kb, code), (pool.vb, code), (pool.ke, exps), (pool.ve, exps)):
            x[~named] = fill
        pool.load()
        out = torch.full((int(offsets[-1]), heads, dh), 7.0, dtype=torch.float16, device=DEV)
        pool.cache.Attend(batch_of(table, start, offsets, int(offsets[-1]), **hints), q, out)
        torch.cuda.synchronize()
        got.append(out.cpu().numpy())
        if form != "many" and form != "long-chunk":
            want, tol = ref.attend(*pool.held(), table, start, offsets, q.cpu().numpy(), dh ** -0.5)
            assert (np.abs(got[-1] - want) <= tol).all()
    np.testing.assert_array_equal(got[0].view(np.uint16), got[1].view(np.uint16))
