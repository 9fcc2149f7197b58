"""Limits of beam search and of the pages' operators at their largest sizes, and
the forms that calls take, without a GPU."""
import ctypes as C

import pytest

import search_forms as forms
from ane import _lib
from test_pages_host import batch, beam, cache, pool, refused

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


@pytest.mark.parametrize("case", forms.SELECT, ids=forms.name_of)
def test_shapes_take_the_forms_of_the_choice_that_they_are_for(case):
    shape, want, scores = case
    got = forms.select_form(**shape)
    assert got[:4] == want
    assert forms.where_scores_are(shape, got) == scores


def test_forms_refuse_what_the_calls_refuse():
    out = (C.c_int32 * 6)()
    refused(lib.ane_debug_kv8_select_form(cache(), batch(), 3, out), "heads=3")
    refused(lib.ane_debug_kv8_select_form(cache(page_tokens=48), batch(), 4, out), "page_tokens=48")
    refused(lib.ane_debug_kv8_select_form(cache(), batch(), 4, None), "null")
    refused(lib.ane_debug_kv8_attend_form(cache(), batch(), 5, 7, out), "heads=5")
    refused(lib.ane_debug_kv8_attend_form(cache(), batch(), 4, 70000, out), "count=70000")
    refused(lib.ane_debug_kv8_attend_form(cache(), batch(), 4, 7, None), "null")
    refused(lib.ane_debug_kv8_copy_form(pool([cache(), cache(pages=5)]), 4, out), "layer 1 differs")
    refused(lib.ane_debug_kv8_copy_form(pool(), -1, out), "pages=-1")
    refused(lib.ane_debug_kv8_copy_form(pool(), 4, None), "null")
    refused(lib.ane_debug_beam_form(1, 33, 100, 0, 5, out), "beams=33")
    refused(lib.ane_debug_beam_form(1, 3, 100, 0, (1 << 30) + 1, out), "history_max")
    refused(lib.ane_debug_beam_form(1, 3, 100, 0, 5, None), "null")


@pytest.mark.parametrize("case", forms.ATTEND, ids=forms.name_of)
def test_shapes_take_the_forms_of_attention_that_they_are_for(case):
    shape, want = case
    assert forms.attend_kind(forms.attend_form(**shape)) == want


@pytest.mark.parametrize("case", forms.COPY, ids=str)
def test_sizes_take_the_forms_of_copies_that_they_are_for(case):
    size, want = case
    assert forms.copy_form(**size) == want


@pytest.mark.parametrize("case", forms.BEAMS, ids=str)
def test_sizes_take_the_forms_of_the_beam_step_that_they_are_for(case):
    size, want = case
    assert forms.beam_form(**size) == want
