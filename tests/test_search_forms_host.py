"""Limits of beam search and of the pages' operators at their largest sizes, and
the forms that calls take, without a GPU."""
import pytest

from ane import _lib
from test_pages_host import beam, refused

lib = _lib.load()


@pytest.mark.parametrize("most", [(1 << 30) + 1, 2**31 - 9, 2**31 - 1])
@pytest.mark.parametrize("beams", [1, 3, 32])
def test_longer_histories_than_places_have_bits_for(most, beams):
    """Their words' places, times 8, would pass 31 bits."""
    refused(beam(history_max=most, history_row=most, requests=1, beams=beams, history=1 << 45), "beam select",
            f"history_max={most}")


def test_long_histories_that_overlap_an_input():
    """2^30 ids are 2^31 bytes: they reach into what lies behind them."""
    most = 1 << 30
    at = 1 << 45
    for other in ("logits", "scores", "weights"):
        refused(beam(history_max=most, history_row=most, requests=1, beams=1, history=at, **{other: at + 2 * most - 400}),
                "overlaps")
