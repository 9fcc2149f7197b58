"""The choice of pages (``ane.KVBounds.Select``) in the forms that large batches
take: every row's choice equal to that of whole numbers in 64 bits."""
import numpy as np
import pytest

import search_forms as forms

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import ane  # noqa: E402

DEV = "cuda"
PAGES = 500


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).to(DEV)


def unit_of(amax):
    """The smallest e >= -30 with amax <= 127 * 2^e, in 64 bits."""
    m, e = torch.frexp(amax)
    return (e - 7 + (m > 127 / 128).int()).clamp(min=-30)


class Choice:
    """Bounds of a small pool and sequences whose tables name its pages, some of
    them several times and some places none."""

    def __init__(self, r, lens, heads, kvh, dh, P, spare=1, rows_behind=2, **hints):
        width = forms.width_of(lens, P, spare)
        self.lens, self.P, self.kvh = lens, P, kvh
        table = r.integers(0, PAGES, (len(lens), width)).astype(np.int32)
        table[r.random(table.shape) < 0.02] = r.choice([-1, PAGES, 2**31 - 1])
        self.table = dev(table)
        self.offsets = np.concatenate([[0], np.cumsum([n for _, n in lens])]).astype(np.int32)
        self.rows = int(self.offsets[-1]) + rows_behind
        self.cache = ane.KVCache8.Empty(PAGES, kvh, dh, P)
        box = r.integers(-127, 128, (PAGES, kvh, 2, dh)).astype(np.int8)
        box = np.stack([box.max(2), box.min(2)], 2)
        box[:40] = box[0]                                 # equal scores, whatever the query
        self.box, self.unit = dev(box), dev(r.integers(-9, -5, (PAGES, kvh)).astype(np.int8))
        self.unit[:40] = -7
        self.q = dev(r.standard_normal((self.rows, heads, dh)).astype(np.float16))
        self.bounds = ane.KVBounds(self.cache, self.box, self.unit)
        self.batch = ane.KVBatch(self.table, dev(np.array([s for s, _ in lens], np.int32)), dev(self.offsets), self.rows,
                                 **hints)

    def want(self, count, first, recent):
        """Each row's choice, without the kernel's arithmetic: products of whole
        numbers and powers of two, exact in 64 bits."""
        out = torch.full((self.rows, self.kvh, count), 99, dtype=torch.int32, device=DEV)
        q = self.q.double().view(self.rows, self.kvh, -1, self.q.shape[2])
        f = unit_of(q.abs().amax(-1))
        z = torch.round(torch.ldexp(q, -f[..., None]))
        for i, (held, new) in enumerate(self.lens):
            pages = -(-(held + new) // self.P)
            ids = self.table[i, :pages].long()
            there = (ids >= 0) & (ids < PAGES)
            ids = torch.where(there, ids, 0)
            row = slice(int(self.offsets[i]), int(self.offsets[i]) + new)
            page = torch.arange(pages, device=DEV)
            n = (held + torch.arange(new, device=DEV)[:, None]) // self.P + 1
            for h in range(self.kvh):
                x = z[row, h]
                big, small = self.box[ids, h].double().unbind(1)
                s = (x.clamp(min=0).flatten(0, 1) @ big.t().contiguous()
                     + x.clamp(max=0).flatten(0, 1) @ small.t().contiguous()).view(new, -1, pages)
                s = torch.ldexp(s, f[row, h][..., None]).amax(1)
                s = torch.ldexp(s, self.unit[ids, h].int()[None])
                s = torch.where((page < first) | (page >= n - recent), float("inf"), s)
                s = torch.where(there & (page < n), s, float("-inf"))
                top, at = torch.sort(s, dim=1, descending=True, stable=True)
                take = torch.full((new, count), pages, device=DEV)
                m = min(count, pages)
                take[:, :m] = torch.where(top[:, :m] > float("-inf"), at[:, :m], pages)
                take = torch.sort(take, 1)[0]
                out[row, h] = torch.where(take < pages, take, -1).int()
        return out

    def check(self, count, first, recent):
        got = torch.full((self.rows, self.kvh, count), 99, dtype=torch.int32, device=DEV)
        self.bounds.Select(self.batch, self.q, count, first, recent, got)
        assert torch.equal(got, self.want(count, first, recent))


@pytest.mark.parametrize("case", forms.SELECT, ids=forms.name_of)
def test_choice(case):
    shape, form, _ = case
    assert forms.select_form(**shape)[:4] == form
    x = Choice(np.random.default_rng(shape["heads"] + shape["dh"]), **shape)
    x.check(33, 1, 2)
    x.check(5, 0, 0)


def test_choice_against_the_plain_rows():
    """The 64-bit choice above and the one of pages_ref, a row at a time."""
    import pages_ref as ref
    r = np.random.default_rng(1)
    x = Choice(r, lens=[(200, 5), (16 * 90, 3)], heads=6, kvh=2, dh=64, P=16)
    x.q[0, 0], x.q[1, 2] = 0, 65504
    want = x.want(7, 1, 1).cpu().numpy()
    q, box, unit, table = (t.cpu().numpy() for t in (x.q, x.box, x.unit, x.table))
    for i, (held, new) in enumerate(x.lens):
        for t in range(new):
            ids = table[i, :(held + t) // 16 + 1]
            there = (ids >= 0) & (ids < PAGES)
            ids = np.where(there, ids, 0)
            for h in range(2):
                row = int(x.offsets[i]) + t
                np.testing.assert_array_equal(
                    want[row, h], ref.select(q[row, 3 * h:3 * h + 3], box[ids, h], unit[ids, h], there, 7, 1, 1))
    x.check(7, 1, 1)
