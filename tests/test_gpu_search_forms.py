"""Forms of beam search, of the pages' copies and of the choice of pages that
large batches take, against plain implementations."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore:overflow encountered", "ignore:invalid value")]

import ane  # noqa: E402

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
