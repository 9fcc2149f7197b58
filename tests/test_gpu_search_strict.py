"""What other tests of the search ask only in part: the entries of a sequence
whose last page is not there, and every step of a search within one bound."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore:overflow encountered", "ignore:invalid value")]

import ane  # noqa: E402
import test_gpu_search_run as run  # noqa: E402

DEV = "cuda"


def ids(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("other, pages", [(0, 12), (3, 21000)])   # by one block, and in a large pool
def test_page_that_is_not_there_stays_so(other, pages):
    """Its tokens are lost and count as missing; the ones behind them get a
    page."""
    cache = ane.KVCache8.Empty(pages, 1, 64, 16)
    pool = ane.KVPages(([cache]), torch.zeros(pages, dtype=torch.int32, device=DEV))
    pool.refs[4] = 1
    pool.refs[:other] = 1
    table, start = ids([[4, -1, -1]]), ids([20])
    missing = pool.Fork(table, start, new=30)
    assert missing.tolist() == [1]
    assert table.tolist() == [[4, -1, other]]
    assert start.tolist() == [20]
    want = torch.zeros(pages, dtype=torch.int32, device=DEV)
    want[4] = want[other] = 1
    want[:other] = 1
    assert torch.equal(pool.refs, want)


@pytest.mark.parametrize("seed, beams, compact", [(0, 4, False), (1, 3, True), (2, 6, True)])
def test_no_error_adds_up_over_a_search(monkeypatch, seed, beams, compact):
    """Each step of the plain search starts from the scores and sequences of the
    GPU's, so the first step's bound holds for all."""
    real, steps = np.testing.assert_allclose, []

    def close(a, b, atol):
        steps.append(np.nanmax(np.abs(np.where(np.isfinite(b), a - b, 0))))
        real(a, b, atol=min(atol, 2e-2))
    monkeypatch.setattr(run.np.testing, "assert_allclose", close)
    run.test_search(seed, beams, compact)
    print("largest differences of a step:", " ".join(f"{x:.1e}" for x in steps))
    assert len(steps) == 12


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("rows, vocab", [(256, 1000), (64, 32000), (300, 32000), (40, 60011), (3, 17)])
def test_log_sums(rows, vocab, half):
    """Scores that leave only the log sum's error, of rows of one beam each: s = scores + (max - lse) is about 0,
    and what fp32 then rounds away is 2^-24 of it.

    The bound, in half steps of fp32 (2^-24): the exponent is off by its difference's rounding, the constant's and the
    product's, 3 |x - max|; each of two powers of two (a part's, and its factor) by 2; 15 additions of a lane."""
    g = torch.Generator(device=DEV).manual_seed(vocab)
    for scale in (0.3, 1.0, 3.0, 10.0):
        x = torch.randn((rows, vocab), device=DEV, generator=g) * scale
        x = x.half() if half else x
        y = x.double()
        top, lse = y.amax(1), torch.logsumexp(y, 1)
        scores = (lse - top).float()
        _, _, out = ane.BeamSearch(vocab, 1).Select(x, scores)
        want = scores.double() + (top - lse)
        p = torch.exp(y - lse[:, None])
        bound = (19 + 3 * (p * (top[:, None] - y)).sum(1)) * 2.0 ** -24
        assert ((out.double() - want).abs() <= bound + want.abs() * 2.0 ** -24).all()


def choices_of_a_chunk(recent, count=3):
    """Of 90 tokens on 200, in one batch and token by token, over the same codes."""
    P, held, new = 16, 200, 90
    g = torch.Generator(device=DEV).manual_seed(recent)
    cache = ane.KVCache8.Empty(30, 2, 64, P)
    cache.k.view(torch.uint8).copy_(torch.randint(0, 0x70, cache.k.shape, dtype=torch.uint8, device=DEV, generator=g)
                                    + 128 * torch.randint(0, 2, cache.k.shape, dtype=torch.uint8, device=DEV, generator=g))
    cache.k_exp.fill_(-6)
    table = torch.randperm(30, device=DEV, generator=g)[None, :20].int()
    q = torch.randn((new, 4, 64), device=DEV, generator=g).half()
    out = []
    for whole in (True, False):
        bounds = ane.KVBounds.Empty(cache)
        bounds.Update(ane.KVBatch(table, ids([0]), ids([0, held]), held))
        rows = []
        for t in [0] if whole else range(new):
            n = new if whole else 1
            batch = ane.KVBatch(table, ids([held + t]), ids([0, n]), n)
            bounds.Update(batch)
            rows.append(bounds.Select(batch, q[t:t + n], count, first=0, recent=recent))
        out.append(torch.cat(rows))
    return out


@pytest.mark.parametrize("recent", [1, 2])
def test_rows_of_a_chunk_choose_as_token_by_token(recent):
    whole, single = choices_of_a_chunk(recent)
    assert torch.equal(whole, single)


def test_rows_of_a_chunk_without_recent_pages_differ_by_their_own_page():
    """Its bounds are of the chunk's later tokens too; of the other pages nothing
    differs but what takes its place."""
    whole, single = choices_of_a_chunk(0, count=1)
    own = (200 + torch.arange(90, device=DEV))[:, None, None] // 16
    differ = whole != single
    assert differ.any()
    # bounds that hold more keys promise no less: where the choices differ, the chunk's is the own page
    assert (whole == own)[differ].all()
