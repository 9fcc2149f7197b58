"""Attention over lists of pages (``KVCache8.Attend(blocks=)``) in every form that
the rules on sizes choose."""
import numpy as np
import pytest

import search_forms as forms

torch = pytest.importorskip("torch")
pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore:overflow encountered", "ignore:invalid value",
                                                          "ignore:All-NaN")]

from test_gpu_select import Run, lists  # noqa: E402


@pytest.mark.parametrize("case", forms.ATTEND, ids=forms.name_of)
def test_attention(case):
    shape, form = case
    assert forms.attend_kind(forms.attend_form(**shape)) == form
    shape = dict(shape)
    count = shape.pop("count")
    r = np.random.default_rng(count + shape["heads"])
    x = Run(r, nan=1e-5, **shape).go()
    b = lists(r, x, count)
    b[x.rows // 2] = -1     # a row that names nothing
    b[:3, 0] = -1
    x.attend(b)
