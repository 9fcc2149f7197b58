"""Forms of beam search's step that large batches and long histories take, against
a plain 64-bit implementation."""
import numpy as np
import pytest

import search_forms as forms

torch = pytest.importorskip("torch")
pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore:overflow encountered", "ignore:invalid value")]

import ane  # noqa: E402
from test_gpu_beams import Case  # noqa: E402

DEV = "cuda"


@pytest.mark.parametrize("beams, most, held", [(32, 1 << 29, (1 << 29) - 3), (32, 1 << 29, 1 << 29), (3, 1 << 30, (1 << 30) - 9)])
def test_histories_of_more_words_than_31_bits_count(beams, most, held):
    """All beams go on from one whose history is long; in the others there is
    anything."""
    at = beams - 2
    history = torch.empty((beams, most), dtype=torch.int16, device=DEV)
    for c in range(0, most, 1 << 28):
        n = min(1 << 28, most - c)
        history[at, c:c + n] = torch.arange(n, device=DEV, dtype=torch.int32).add_(c >> 3).to(torch.int16)
    keep = history[at, :held].clone()
    behind = history[:, -2:].clone()
    lengths = torch.full((beams,), 5, dtype=torch.int32, device=DEV)
    lengths[at] = held
    scores = torch.full((beams,), -1e4, device=DEV)
    scores[at] = 0
    logits = -torch.arange(50, device=DEV, dtype=torch.float32).repeat(beams, 1)
    tokens, parents, _ = ane.BeamSearch(50, beams).Select(logits, scores, history=history, lengths=lengths)
    assert tokens.tolist() == list(range(beams)) and (parents == at).all()
    assert (lengths == min(held + 1, most)).all()
    for r in range(beams):
        assert torch.equal(history[r, :held], keep), r
    if held < most:
        assert history[:, held].tolist() == list(range(beams))
        if held + 1 <= most - 2:
            assert torch.equal(history[:, -2:], behind)   # behind the new length


@pytest.mark.parametrize("most", [(1 << 30) + 1, 1 << 31])
def test_longer_histories_are_refused(most):
    history = torch.empty((1, most), dtype=torch.int16, device=DEV)
    lengths = torch.zeros(1, dtype=torch.int32, device=DEV)
    with pytest.raises(ane.EngineError, match="at most 1073741824"):
        ane.BeamSearch(50, 1).Select(torch.zeros((1, 50), device=DEV), torch.zeros(1, device=DEV), history=history,
                                     lengths=lengths)


@pytest.mark.parametrize("case", forms.BEAMS, ids=str)
def test_beam_step(case):
    size, form = case
    assert forms.beam_form(**size) == form
    c = Case(np.random.default_rng(size["vocab"]), **size)
    c.check(offset=1 if size.get("wide") else 0)
    if size["hist"] is None:     # the last entries of a row, behind its last whole turn, are the best
        c.logits[:, -1] = c.logits.max(1) + 2
        got = c.check()
        assert (got["tokens"] == size["vocab"] - 1).any()
