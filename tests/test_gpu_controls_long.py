"""Controls on logits over histories as long as a length can say."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import ane  # noqa: E402

DEV = "cuda"


@pytest.mark.parametrize("held", [(1 << 31) - 1, (1 << 31) - 5, (1 << 31) - 2048, (1 << 31) - 2049])
def test_history_of_nearly_2_to_the_31_ids(held):
    """Its last ids count, and nothing behind or in front of it does."""
    vocab, most, before = 100, (1 << 31) - 1, 1 << 16
    room = torch.full((1, before + most), 7, dtype=torch.int16, device=DEV)   # 7 counts
    history = room[:, before:]
    history[0, :held] = 30000                                                 # passed over: not of the vocabulary
    history[0, 0] = 2
    history[0, held - 3:held] = 3
    lengths = torch.tensor([held], dtype=torch.int32, device=DEV)
    prompts = torch.tensor([held - 2], dtype=torch.int32, device=DEV)
    each = lambda x: torch.tensor([x], device=DEV)  # noqa: E731
    controls = ane.LogitControls(vocab, repetition=each(2.0), frequency=each(0.25), presence=each(0.5))
    logits = torch.full((1, vocab), 8.0, device=DEV)
    out, tokens = controls.Apply(logits, history, lengths, prompts)
    want = torch.full((vocab,), 8.0)
    want[2] = 4.0
    want[3] = 4.0 - 2 * 0.25 - 0.5
    assert torch.equal(out[0].cpu(), want)
    assert int(tokens) == 0


def test_longer_history_is_refused():
    history = torch.empty((1, 1 << 31), dtype=torch.int16, device=DEV)
    controls = ane.LogitControls(100, repetition=torch.ones(1, device=DEV))
    with pytest.raises(ane.EngineError, match="2147483648 places"):
        controls.Apply(torch.zeros((1, 100), device=DEV), history, torch.zeros(1, dtype=torch.int32, device=DEV))
