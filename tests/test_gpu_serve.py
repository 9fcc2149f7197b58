"""The serving operators on the GPU (``ane.KVCache8``, ``ane.KVBatch``,
``ane.LogitControls``) against plain 64-bit implementations (serve_ref.py).

Appended values are compared exactly but for keys within fp32 rounding of a tie
between two codes; attention within the tolerance that serve_ref.attend
derives; logits bit for bit."""
import numpy as np
import pytest

import serve_ref as ref

torch = pytest.importorskip("torch")
pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore:overflow encountered", "ignore:invalid value")]

import ane  # noqa: E402
from ane import _lib  # noqa: E402

DEV = "cuda"


def dev(x, dtype=None):
    return torch.from_numpy(np.ascontiguousarray(x)).to(DEV) if dtype is None else \
        torch.from_numpy(np.ascontiguousarray(x, dtype=dtype)).to(DEV)


def rope_tables(n, dh, theta=10000.0):
    f = np.arange(n)[:, None] / theta ** (np.arange(0, dh, 2) / dh)
    return np.cos(f).astype(np.float32), np.sin(f).astype(np.float32)


class Pool:
    """Random pages on the GPU; their bytes on the host."""

    def __init__(self, r, pages, kvh, P, dh, nan=0.0, exps=(-8, -3)):
        def codes(shape):
            b = r.integers(0, 256, shape).astype(np.uint8)
            b[(b & 127) == 127] = 0x21
            b[r.random(shape) < nan] = 0x7f
            return b
        self.kb = codes((pages, kvh, P, dh))
        self.vb = codes((pages, kvh, P // 16, 4, 16, dh // 16, 4))
        self.ke, self.ve = (r.integers(*exps, (pages, kvh)).astype(np.int8) for _ in range(2))
        self.load()

    def load(self):
        f8 = torch.float8_e4m3fn
        self.cache = ane.KVCache8(dev(self.kb).view(f8), dev(self.vb).view(f8), dev(self.ke), dev(self.ve))

    def held(self):
        """(k, v) code values in row order, from the GPU, and the exponents."""
        c = self.cache
        k = ref.VALUES[c.k.view(torch.uint8).cpu().numpy()]
        v = ref.VALUES[ref.v_rows(c.v.view(torch.uint8).cpu().numpy())]
        return k, v, c.k_exp.cpu().numpy(), c.v_exp.cpu().numpy()


def batch_of(table, start, offsets, rows, **kw):
    return ane.KVBatch(dev(table, np.int32), dev(start, np.int32), dev(offsets, np.int32), rows, **kw)


def layout(r, lens, P, spare=1):
    """Page tables for sequences of lens[i] = (held, new), shuffled pages."""
    need = [(s + n + P - 1) // P for s, n in lens]
    width = max(max(need), 1) + spare
    ids = r.permutation(sum(need) + 2)
    table = np.full((len(lens), width), -1, np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = ids[at:at + n]
        at += n
    offsets = np.concatenate([[0], np.cumsum([n for _, n in lens])]).astype(np.int32)
    return table, np.array([s for s, _ in lens], np.int32), offsets, len(ids)


def check_append(before, after, exp, xk, table, start, offsets, P, cos, sin):
    """after (k, v, k_exp, v_exp from the GPU) against the same append in 64 bits."""
    k, v, ke, ve = (x.copy() for x in before)
    np.testing.assert_array_equal(after[2], exp[2])
    np.testing.assert_array_equal(after[3], exp[3])
    np.testing.assert_array_equal(after[1], exp[1])
    off = ~((after[0] == exp[0]) | (np.isnan(after[0]) & np.isnan(exp[0])))
    # a key one code away: its exact value is within fp32 rounding of the tie.  Three roundings of products and a
    # difference of numbers up to |a| + |b|, so 3 * 2^-24 * (|a| + |b|)
    where = {}
    for i in range(len(start)):
        for t in range(int(offsets[i + 1] - offsets[i])):
            pos = int(start[i]) + t
            if pos < table.shape[1] * P:
                where[(int(table[i, pos // P]), pos % P)] = (int(offsets[i]) + t, pos)
    for page, h, s, d in np.argwhere(off):
        row, pos = where[(page, s)]
        x = xk[row:row + 1].astype(np.float64)
        y = ref.rope(x, cos[pos:pos + 1].astype(np.float64), sin[pos:pos + 1].astype(np.float64))[0, h, d]
        pair = np.abs(x[0, h, d // 2 * 2:d // 2 * 2 + 2]).sum()
        scale = 2.0 ** float(after[2][page, h])
        assert abs(after[0][page, h, s, d] * scale - y) <= abs(exp[0][page, h, s, d] * scale - y) + 6 * 2.0 ** -24 * pair
    assert off.mean() < 1e-3


def run_append(r, lens, heads, kvh, dh, P, scale=1.0, packed=True, poke=None, pool=None, spread=0.7, **hints):
    table, start, offsets, pages = layout(r, lens, P)
    rows = int(offsets[-1]) + 2   # two rows of no sequence
    pool = pool or Pool(r, pages, kvh, P, dh)
    cos, sin = rope_tables(table.shape[1] * P, dh)
    x = r.standard_normal((rows, heads + 2 * kvh, dh)) * np.exp(spread * r.standard_normal((1, heads + 2 * kvh, 1)))
    x = (x * scale).astype(np.float16)
    if poke:
        poke(x, table, start, offsets)
    before = pool.held()
    g = dev(x) if packed else None
    parts = [g[:, :heads], g[:, heads:heads + kvh], g[:, heads + kvh:]] if packed else [
        dev(x[:, a:b].transpose(1, 0, 2)).transpose(0, 1) for a, b in
        ((0, heads), (heads, heads + kvh), (heads + kvh, heads + 2 * kvh))]   # [heads][rows][dh] in memory
    q_out = torch.full((rows, heads, dh), 7.0, dtype=torch.float16, device=DEV)
    b = batch_of(table, start, offsets, rows, **hints)
    got = pool.cache.Append(b, *parts, dev(cos), dev(sin), q_out)
    torch.cuda.synchronize()
    assert got is q_out
    exp = tuple(z.copy() for z in before)
    x64 = x.astype(np.float64)
    ref.append(*exp, table, start, offsets, x64[:, heads:heads + kvh], x64[:, heads + kvh:], cos.astype(np.float64),
               sin.astype(np.float64))
    check_append(before, pool.held(), exp, x[:, heads:heads + kvh], table, start, offsets, P, cos, sin)
    q = q_out.cpu().numpy().astype(np.float64)
    for i in range(len(start)):
        a, n = int(offsets[i]), int(min(offsets[i + 1] - offsets[i], table.shape[1] * P - start[i]))
        if n <= 0:
            continue
        pos = np.arange(start[i], start[i] + n)
        want = ref.rope(x64[a:a + n, :heads], cos[pos].astype(np.float64), sin[pos].astype(np.float64))
        pair = np.abs(x64[a:a + n, :heads]).reshape(n, heads, dh // 2, 2).sum(-1).repeat(2, -1)
        fine = np.abs(want) < 65000
        err = np.abs(q[a:a + n] - want)
        lim = np.abs(want) * 2.0 ** -11 + 2.0 ** -25 + 3 * 2.0 ** -24 * pair
        assert (err <= lim)[fine].all()
    assert (q[offsets[-1]:] == 7.0).all()   # rows of no sequence, left as they were
    return pool, (table, start, offsets, rows)


@pytest.mark.parametrize("P", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("heads,kvh,dh", [(12, 4, 64), (4, 2, 128), (5, 1, 64)])
def test_append(P, heads, kvh, dh):
    r = np.random.default_rng(P + heads)
    lens = [(0, 1), (P - 1, 2), (P, 1), (3, 0), (0, P), (5, 2 * P + 3), (P // 2, P // 2), (2 * P + 7, 1), (17, 40)]
    run_append(r, lens, heads, kvh, dh, P)


FEW = {
    # more sequences than rows fill pages of, some rows on both sides of a page's end; then whole pages and more,
    # with a hint that promises one row each
    "tokens": ([(n, 1) for n in (0, 1, 15, 16, 31, 63, 64, 200, 255)] + [(15, 2), (63, 3), (0, 2), (9, 0), (255, 2)],
               {}),
    "wrong": ([(30, 1), (0, 300), (15, 2), (10, 0), (63, 9), (0, 16), (250, 45)], dict(max_new=1)),
}


@pytest.mark.parametrize("P", [16, 64, 256])
@pytest.mark.parametrize("heads,kvh,dh", [(12, 4, 64), (5, 5, 128), (0, 2, 64)])
@pytest.mark.parametrize("case", FEW)
@pytest.mark.parametrize("scale", [1.0, 3000.0])
def test_append_few_rows(case, heads, kvh, dh, P, scale):
    """A wave per page; old rows of all sizes, so that some exponents rise."""
    lens, hints = FEW[case]
    run_append(np.random.default_rng(P + dh), lens, heads, kvh, dh, P, scale=scale, packed=P != 64, **hints)


@pytest.mark.parametrize("dh", [64, 128])
def test_append_does_not_depend_on_hints(dh):
    """The same bits whichever kernel the hints choose."""
    lens = [(30, 1), (0, 40), (15, 2), (63, 9), (5, 16)]
    table, start, offsets, pages = layout(np.random.default_rng(1), lens, 32)
    x = dev((np.random.default_rng(2).standard_normal((68, 14, dh)) * 2).astype(np.float16))
    cos, sin = (dev(t) for t in rope_tables(table.shape[1] * 32, dh))
    got = []
    for hints in (dict(max_new=1), dict(max_new=40), {}):
        pool = Pool(np.random.default_rng(3), pages, 3, 32, dh)
        q = torch.zeros((68, 8, dh), dtype=torch.float16, device=DEV)
        pool.cache.Append(batch_of(table, start, offsets, 68, **hints), x[:, :8], x[:, 8:11], x[:, 11:], cos, sin, q)
        got.append([q.cpu().numpy().view(np.uint16)] + [z.copy() for z in pool.held()])
    for other in got[1:]:
        for a, b in zip(got[0], other):
            np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("scale", [1e-7, 3e-4, 30.0, 2000.0, 60000.0])
def test_append_magnitudes(scale):
    """Exponents from the bottom (codes that are subnormal, all zeros) to the
    top (numbers past 61440, infinities), against pages whose old exponents
    are larger and smaller."""
    r = np.random.default_rng(int(scale * 7) + 3)

    def poke(x, *_):
        x[1, :, 3] = 0
        if scale > 10000:
            x[2, 4:, ::7] = np.inf
            x[3, 4:, 1::9] = -np.inf
            x[4, 4:, 5] = 65504
    run_append(r, [(9, 3), (0, 30), (40, 1), (64, 5), (130, 1)], 4, 2, 64, 64, scale=scale, poke=poke, spread=0.1)


def test_append_nan_stays_where_it_is():
    r = np.random.default_rng(5)

    def poke(x, *_):
        x[2, 4:, 10] = np.nan
        x[7, 4:, :] = np.nan      # a whole row: no magnitude at all
    run_append(r, [(9, 3), (0, 1), (16, 1), (5, 1), (1, 1), (0, 1)], 4, 2, 64, 16, poke=poke)


def test_append_head_major_tensors():
    run_append(np.random.default_rng(6), [(3, 20), (0, 5)], 4, 2, 64, 32, packed=False)


def test_append_token_by_token_rounds_again():
    """A page filled one token at a time, each louder than the last: its
    exponent rises and the rows before are rounded again, step by step as the
    reference does it."""
    r = np.random.default_rng(8)
    P, kvh, dh = 16, 2, 64
    table = np.array([[2, 0, 1]], np.int32)
    pool = Pool(r, 3, kvh, P, dh)
    cos, sin = rope_tables(48, dh)
    exp = [z.copy() for z in pool.held()]
    for t in range(20):
        x = (r.standard_normal((1, 2 * kvh, dh)) * 1.7 ** t * 1e-2).astype(np.float16)
        start, offsets = np.array([t], np.int32), np.array([0, 1], np.int32)
        before = pool.held()
        g = dev(x)
        assert pool.cache.Append(batch_of(table, start, offsets, 1), None, g[:, :kvh], g[:, kvh:], dev(cos),
                                 dev(sin)) is None
        exp = [z.copy() for z in before]
        x64 = x.astype(np.float64)
        ref.append(*exp, table, start, offsets, x64[:, :kvh], x64[:, kvh:], cos.astype(np.float64),
                   sin.astype(np.float64))
        check_append(before, pool.held(), exp, x[:, :kvh], table, start, offsets, P, cos, sin)


def test_append_in_place_and_missing_pages():
    """q_out = q; pages outside the pool and positions past the table get
    nothing, and everything else is as it was."""
    r = np.random.default_rng(9)
    P, kvh, heads, dh = 16, 2, 4, 64
    table = np.array([[1, -1, 3], [4, 5, 99], [-2**31, 2**31 - 1, 0]], np.int32)
    start, offsets = np.array([10, 40, 47], np.int32), np.array([0, 20, 30, 33], np.int32)
    pool = Pool(r, 6, kvh, P, dh)
    cos, sin = rope_tables(48, dh)
    x = r.standard_normal((33, heads + 2 * kvh, dh)).astype(np.float16)
    before = pool.held()
    g = dev(x)
    q = g[:, :heads]
    out = pool.cache.Append(batch_of(table, start, offsets, 33), q, g[:, heads:heads + kvh], g[:, heads + kvh:],
                            dev(cos), dev(sin), q)
    assert out is q
    exp = [z.copy() for z in before]
    x64 = x.astype(np.float64)
    ref.append(*exp, table, start, offsets, x64[:, heads:heads + kvh], x64[:, heads + kvh:], cos.astype(np.float64),
               sin.astype(np.float64))
    check_append(before, pool.held(), exp, x[:, heads:heads + kvh], table, start, offsets, P, cos, sin)
    got = g.cpu().numpy()
    np.testing.assert_array_equal(got[:, heads:], x[:, heads:])
    np.testing.assert_array_equal(got[28:30, :heads], x[28:30, :heads])   # positions 48 and 49: no rows of the batch
    np.testing.assert_array_equal(got[31:, :heads], x[31:, :heads])
    assert (got[:28, :heads] != x[:28, :heads]).any()


def run_attend(r, lens, heads, kvh, dh, P, pool=None, q=None, rows_more=2, holes=(), scale=None, **hints):
    table, start, offsets, pages = layout(r, lens, P)
    for i, j in holes:
        table[i, j] = [-1, pages + 5, 2**31 - 1, -2**31][(i + j) % 4]
    pool = pool or Pool(r, pages, kvh, P, dh)
    rows = int(offsets[-1]) + rows_more
    if q is None:
        q = r.standard_normal((rows, heads, dh)).astype(np.float16)
    out = torch.full((rows, heads, dh), 7.0, dtype=torch.float16, device=DEV)
    got = pool.cache.Attend(batch_of(table, start, offsets, rows, **hints), dev(q), out, scale)
    torch.cuda.synchronize()
    assert got is out
    want, tol = ref.attend(*pool.held(), table, start, offsets, q, dh ** -0.5 if scale is None else scale)
    y = out.cpu().numpy().astype(np.float64)
    none = np.ones(rows, bool)
    for i in range(len(start)):
        none[offsets[i]:offsets[i] + max(0, min(offsets[i + 1] - offsets[i], table.shape[1] * P - start[i]))] = False
    assert (y[none] == 7.0).all()   # rows of no sequence, left as they were
    y, want, tol = y[~none], want[~none], tol[~none]
    bad = np.isnan(want)
    assert np.array_equal(np.isnan(y), bad)
    err = np.abs(y - want)[~bad]
    print("worst error over tolerance", (err / np.maximum(tol[~bad], 1e-300)).max() if err.size else 0)
    assert (err <= tol[~bad]).all()
    return pool, out


@pytest.mark.parametrize("P", [16, 64, 256])
@pytest.mark.parametrize("heads,kvh,dh", [(12, 4, 64), (16, 2, 128), (1, 1, 64), (32, 1, 64), (20, 1, 128)])
def test_attend_single_tokens(P, heads, kvh, dh):
    r = np.random.default_rng(P + heads)
    run_attend(r, [(n - 1, 1) for n in (1, 2, 15, 16, 17, 63, 64, 65, 255, 256, 257, 700)], heads, kvh, dh, P,
               max_new=1, max_len=700)


@pytest.mark.parametrize("heads,kvh,dh", [(12, 4, 64), (6, 2, 128), (3, 3, 64), (24, 1, 128), (31, 1, 64)])
@pytest.mark.parametrize("hints", [{}, dict(max_new=140, max_len=400), dict(max_new=1, max_len=1)])
def test_attend_prompts_and_chunks(heads, kvh, dh, hints):
    """Prompts behind nothing, chunks behind a context, sequences without new
    rows, single tokens between them; right, missing and wrong hints."""
    r = np.random.default_rng(heads)
    run_attend(r, [(0, 140), (65, 1), (10, 0), (3, 33), (250, 64), (399, 1), (0, 1), (300, 7)], heads, kvh, dh, 32,
               **hints)


@pytest.mark.parametrize("nseq", [1, 3])
@pytest.mark.parametrize("new", [1, 4, 9])
def test_attend_long_context_in_parts(nseq, new):
    r = np.random.default_rng(nseq + new)
    run_attend(r, [(5000 - 37 * i, new) for i in range(nseq)], 6, 2, 64, 64, max_new=new, max_len=5009)


LARGE = {
    # one long sequence: its keys in parts, then whole
    "chunk": ([(4100, 40)], 12, 4, dict(max_new=40, max_len=4140)),
    "long-chunk": ([(4090, 530)], 12, 4, dict(max_new=530, max_len=4620)),
    # many blocks: each wave a tile of its own
    "many": ([(i % 7 * 9, 1 + i * 37 % 90) for i in range(60)], 16, 16, dict(max_new=90, max_len=144)),
}


@pytest.mark.parametrize("P", [16, 64])
@pytest.mark.parametrize("case", LARGE)
def test_attend_large_tiles(case, P):
    """Tiles of 48 rows, with pages that are not there and NaN values."""
    lens, heads, kvh, hints = LARGE[case]
    r = np.random.default_rng(P)
    table, start, offsets, pages = layout(r, lens, P)
    pool = Pool(r, pages, kvh, P, 64)
    last = lens[-1][0] + lens[-1][1] - 5
    for p in (3, last):
        pool.vb[table[-1, p // P], 0, p % P // 16, p % 16 // 4, 37 % 16, 37 // 16, p % 4] = 0x7f
    pool.load()
    run_attend(np.random.default_rng(P), lens, heads, kvh, 64, P, pool=pool, holes=[(0, 0), (len(lens) - 1, 2)],
               **hints)


@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("lens", [[(300, 40), (2, 90), (0, 0), (1500, 33), (700, 1), (300, 40)],
                                  [(8200, 30), (100, 230)]])
def test_attend_ragged_chunks(lens, dh):
    """Enough blocks that the longest contexts are taken first: whole, and (at
    head dimension 64 and 8230 keys) in parts."""
    r = np.random.default_rng(dh + len(lens))
    run_attend(r, lens, 32, 32, dh, 32, holes=[(1, 0)], max_new=max(n for _, n in lens),
               max_len=max(s + n for s, n in lens))


@pytest.mark.parametrize("dh,heads", [(64, 4), (128, 8)])
def test_attend_missing_pages(dh, heads):
    """Keys of pages that are not there take no part; a row with none gives
    zeros (sequence 2's only page; the first rows of sequence 3)."""
    r = np.random.default_rng(3)
    run_attend(r, [(100, 1), (64, 30), (5, 3), (0, 70)], heads, 2, dh, 16,
               holes=[(0, 1), (0, 6), (1, 0), (1, 2), (1, 5), (2, 0), (3, 0), (3, 2)])


@pytest.mark.parametrize("dh,P", [(64, 64), (128, 16)])
@pytest.mark.parametrize("lens", [[(30, 1), (63, 2)], [(0, 90), (45, 70)], [(1000, 3)]])
def test_attend_ignores_what_is_behind(dh, P, lens):
    """Rows behind a sequence's last token, and pages of others, hold NaN."""
    r = np.random.default_rng(dh + lens[0][0])
    table, start, offsets, pages = layout(r, lens, P)
    pool = Pool(r, pages, 2, P, dh)
    used = np.zeros((pages, P), bool)
    for i, (s, n) in enumerate(lens):
        for p in range(s + n):
            used[table[i, p // P], p % P] = True
    kb = pool.kb.transpose(0, 2, 1, 3)
    kb[~used] = 0xff
    v = pool.vb.transpose(0, 2, 3, 6, 1, 4, 5).copy()    # [pages, P/16, 4, 4, kvh, 16, dh/16]
    v.reshape(pages, P, 2, 16, dh // 16)[~used] = 0x7f
    pool.vb = np.ascontiguousarray(v.transpose(0, 4, 1, 2, 5, 6, 3))
    pool.load()
    run_attend(np.random.default_rng(dh + lens[0][0]), lens, 4, 2, dh, P, pool=pool)


@pytest.mark.parametrize("dh,heads", [(64, 6), (128, 2)])
@pytest.mark.parametrize("where", ["k", "v"])
def test_attend_nan_reaches_its_own_rows(dh, heads, where):
    """A NaN key or value in the middle of a prompt: rows before it are as if
    it were not there, rows from it on are NaN (a key: whole rows; a value:
    its dimension)."""
    r = np.random.default_rng(dh)
    lens, P = [(0, 150), (20, 40)], 32
    table, start, offsets, pages = layout(r, lens, P)
    pool = Pool(r, pages, 2, P, dh)
    for i, p in ((0, 97), (0, 131), (1, 25)):
        page, s = table[i, p // P], p % P
        if where == "k":
            pool.kb[page, 0, s, 5] = 0x7f
        else:
            pool.vb[page, 0, s // 16, s % 16 // 4, 37 % 16, 37 // 16, s % 4] = 0xff
    pool.load()
    pool, out = run_attend(np.random.default_rng(dh), lens, heads, 2, dh, P, pool=pool)
    assert np.isfinite(out.float().cpu().numpy()[:97]).all() and not np.isfinite(out.float().cpu().numpy()[:150]).all()


def test_attend_infinities_and_large_scores():
    """Scores far apart (weights that are exactly 0 or 1), a large scale, and
    queries with infinities (NaN rows, as softmax of an infinite score is)."""
    r = np.random.default_rng(12)
    lens = [(100, 20), (300, 1)]
    q = (r.standard_normal((23, 4, 64)) * 200).astype(np.float16)
    run_attend(np.random.default_rng(1), lens, 4, 2, 64, 64, q=q, scale=3.0)
    q[3, 1, 7] = np.inf
    table, start, offsets, pages = layout(np.random.default_rng(1), lens, 64)
    pool = Pool(np.random.default_rng(2), pages, 2, 64, 64)
    out = pool.cache.Attend(batch_of(table, start, offsets, 23), dev(q)).float().cpu().numpy()
    assert np.isnan(out[3, 1]).all()
    assert np.isfinite(out[:3]).all() and np.isfinite(out[3, [0, 2, 3]]).all() and np.isfinite(out[4:21]).all()


def test_attend_strided_tensors():
    """Queries as part of packed rows, outputs head-major: the same bits."""
    r = np.random.default_rng(13)
    lens = [(40, 9), (0, 30)]
    table, start, offsets, pages = layout(r, lens, 16)
    pool = Pool(r, pages, 2, 16, 64)
    b = batch_of(table, start, offsets, 39)
    qkv = dev(r.standard_normal((39, 10, 64)).astype(np.float16))
    want = pool.cache.Attend(b, qkv[:, :6].contiguous())
    out = torch.zeros((6, 39, 64), dtype=torch.float16, device=DEV).transpose(0, 1)
    pool.cache.Attend(b, qkv[:, :6], out)
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_offsets_past_32_bits():
    """Pools of more than 4 GiB each, the pages used at both ends."""
    P, kvh, dh, pages = 256, 8, 128, 17000     # 256 KiB a page and side
    free = torch.cuda.mem_get_info()[0]
    if free < 16 << 30:
        pytest.skip("needs 16 GiB")
    cache = ane.KVCache8.Empty(pages, kvh, dh, P)
    small = ane.KVCache8.Empty(4, kvh, dh, P)
    r = np.random.default_rng(14)
    cos, sin = (dev(x) for x in rope_tables(4 * P, dh))
    x = dev(r.standard_normal((500, 8 + 2 * kvh, dh)).astype(np.float16))
    outs = []
    for c, table in ((cache, [[pages - 1, 3, pages - 2, 16999 // 2]]), (small, [[0, 1, 2, 3]])):
        b = batch_of(np.array(table), np.array([0]), np.array([0, 500]), 500)
        q = c.Append(b, x[:, :8], x[:, 8:8 + kvh], x[:, 8 + kvh:], cos, sin)
        outs.append((q, c.Attend(b, q), [c.k.view(torch.uint8)[t] for t in table[0]],
                     [c.v.view(torch.uint8)[t] for t in table[0]]))
    torch.cuda.synchronize()
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
    for s in (2, 3):
        for a, c in zip(outs[0][s], outs[1][s]):
            assert torch.equal(a, c)
    assert int(cache.k.view(torch.uint8)[4:8400].count_nonzero()) == 0


CONTROL = [dict(), dict(rep=True), dict(freq=True, prompts=False), dict(rep=True, freq=True, pres=True),
           dict(bias="one"), dict(bias="rows", mask="one"), dict(mask="rows"),
           dict(rep=True, freq=True, pres=True, bias="one", mask="rows")]


@pytest.mark.parametrize("kw", CONTROL, ids=lambda k: "-".join(k) or "plain")
@pytest.mark.parametrize("rows,vocab,hist", [(1, 1, 1), (3, 33, 5), (2, 4096, 700), (5, 4097, 0), (4, 32000, 1100),
                                             (3, 65535, 9000), (131, 9001, 250), (128, 8192, 40)])
def test_control(rows, vocab, hist, kw):
    r = np.random.default_rng(rows * vocab + hist)
    lg = (r.standard_normal((rows, vocab)) * 3).astype(np.float32)
    lg[r.random((rows, vocab)) < 0.01] = 0.0
    h = np.minimum((r.random((rows, hist)) ** 3 * vocab).astype(np.int64), 65535).astype(np.uint16)
    h[r.random(h.shape) < 0.02] = 65535          # no token
    lengths = r.integers(0, hist + 1, rows).astype(np.int32)
    lengths[0] = hist + 50                        # taken as hist
    prompts = r.integers(-1, hist + 2, rows).astype(np.int32) if kw.get("prompts", True) else None
    u = lambda lo, hi: r.uniform(lo, hi, rows).astype(np.float32)  # noqa: E731
    p = dict(repetition=u(0.8, 1.6) if kw.get("rep") else None, frequency=u(-0.2, 0.5) if kw.get("freq") else None,
             presence=u(0, 1) if kw.get("pres") else None)
    bias = mask = None
    if kw.get("bias"):
        bias = (r.standard_normal((rows, vocab)) * (r.random((rows, vocab)) < 0.1)).astype(np.float32)
        bias = bias[0] if kw["bias"] == "one" else bias
    if kw.get("mask"):
        mask = r.integers(0, 2**32, (rows, (vocab + 31) // 32), dtype=np.uint64).astype(np.uint32)
        mask[-1] = 0                              # a row that allows nothing
        mask = mask[0] if kw["mask"] == "one" else mask
    use = any(x is not None for x in p.values())
    c = ane.LogitControls(vocab, **{k: None if x is None else dev(x) for k, x in p.items()},
                          bias=None if bias is None else dev(bias),
                          mask=None if mask is None else dev(mask.view(np.int32)))
    args = (dev(h.view(np.int16)), dev(lengths), None if prompts is None else dev(prompts)) if use else ()
    x = dev(lg)
    out, tok = c.Apply(x, *args)
    torch.cuda.synchronize()
    want, wt = ref.control(lg, h if use else None, lengths, prompts, p["repetition"], p["frequency"], p["presence"],
                           bias, mask)
    np.testing.assert_array_equal(out.cpu().numpy().view(np.uint32), want.view(np.uint32))
    np.testing.assert_array_equal(tok.cpu().numpy(), wt)
    assert torch.equal(x, dev(lg))
    c.Apply(x, *args, out=x, tokens=tok)          # in place
    torch.cuda.synchronize()
    assert torch.equal(x.view(torch.int32), out.view(torch.int32))


def test_control_ties_nan_and_infinities():
    lg = np.zeros((6, 9000), np.float32)
    lg[0, [17, 4200, 8999]] = 5.0
    lg[1, :] = np.nan
    lg[2, :] = np.nan
    lg[2, 8500] = -3.0
    lg[3, [8192, 700]] = np.inf
    lg[4, :] = -np.inf
    lg[5, :] = -np.inf
    lg[5, 8999] = -1e38
    out, tok = ane.LogitControls(9000).Apply(dev(lg))
    assert tok.tolist() == [17, ane.NO_TOKEN, 8500, 700, ane.NO_TOKEN, 8999]
    np.testing.assert_array_equal(out.cpu().numpy(), lg)


def test_control_strided_rows():
    r = np.random.default_rng(20)
    lg = r.standard_normal((4, 700)).astype(np.float32)
    wide = torch.zeros((4, 1001), device=DEV)
    wide[:, 100:800] = dev(lg)
    hist = torch.zeros((4, 77), dtype=torch.int16, device=DEV)
    h = r.integers(0, 700, (4, 31)).astype(np.uint16)
    hist[:, 5:36] = dev(h.view(np.int16))
    rep = r.uniform(1, 2, 4).astype(np.float32)
    n = np.array([31, 30, 1, 0], np.int32)
    into = torch.zeros((4, 1501), device=DEV)
    out, tok = ane.LogitControls(700, repetition=dev(rep)).Apply(wide[:, 100:800], hist[:, 5:36], dev(n),
                                                                out=into[:, 3:703])
    want, wt = ref.control(lg, h, n, None, rep, None, None, None, None)
    np.testing.assert_array_equal(out.cpu().numpy(), want)
    np.testing.assert_array_equal(tok.cpu().numpy(), wt)
    assert float(into[:, :3].abs().sum()) == 0 and float(into[:, 703:].abs().sum()) == 0


def serving_steps(r, lens, steps, heads=6, kvh=2, dh=64, P=32, vocab=5000):
    """Inputs of a run of steps: prompts first, then a token each."""
    all_lens = [(s, n) for s, n in lens]
    table, _, _, pages = layout(r, [(s, n + steps) for s, n in all_lens], P)
    cos, sin = rope_tables(table.shape[1] * P, dh)
    out = []
    start = np.array([s for s, _ in all_lens])
    new = np.array([n for _, n in all_lens])
    for t in range(steps + 1):
        rows = int(new.sum())
        out.append((start.copy(), np.concatenate([[0], np.cumsum(new)]), rows,
                    r.standard_normal((rows, heads + 2 * kvh, dh)).astype(np.float16),
                    r.standard_normal((len(new), vocab)).astype(np.float32)))
        start = start + new
        new = np.ones_like(new)
    return table, pages, cos, sin, out


def test_run_of_all_operators():
    """A batch's life: prompts, then steps of a token each; append, attend and
    control in turn on the state that the calls before left."""
    r = np.random.default_rng(30)
    heads, kvh, dh, P, vocab, steps = 6, 2, 64, 32, 5000, 5
    table, pages, cos, sin, run = serving_steps(r, [(0, 70), (0, 3), (0, 33)], steps)
    pool = Pool(r, pages, kvh, P, dh)
    g = [dev(x) for x in (cos, sin)]
    hist = np.zeros((3, 100), np.uint16)
    lens = np.array([70, 3, 33], np.int32)
    for i, n in enumerate(lens):
        hist[i, :n] = r.integers(0, vocab, n)
    prompts = lens.copy()
    hist_d, lens_d, prompts_d = dev(hist.view(np.int16)), dev(lens), dev(prompts)
    pen = [r.uniform(1.1, 1.5, 3).astype(np.float32), r.uniform(0.1, 0.5, 3).astype(np.float32)]
    ctl = ane.LogitControls(vocab, repetition=dev(pen[0]), presence=dev(pen[1]))
    for start, offsets, rows, x, lg in run:
        b = batch_of(table, start, offsets, rows)
        before = pool.held()
        d = dev(x)
        q = pool.cache.Append(b, d[:, :heads], d[:, heads:heads + kvh], d[:, heads + kvh:], *g)
        out = pool.cache.Attend(b, q)
        exp = [z.copy() for z in before]
        x64 = x.astype(np.float64)
        ref.append(*exp, table, start, offsets, x64[:, heads:heads + kvh], x64[:, heads + kvh:],
                   cos.astype(np.float64), sin.astype(np.float64))
        check_append(before, pool.held(), exp, x[:, heads:heads + kvh], table, start, offsets, P, cos, sin)
        want, tol = ref.attend(*pool.held(), table, start, offsets, q.cpu().numpy(), dh ** -0.5)
        assert (np.abs(out.cpu().numpy() - want) <= tol).all()
        _, tok = ctl.Apply(dev(lg), hist_d, lens_d, prompts_d)
        w, wt = ref.control(lg, hist, lens, prompts, pen[0], None, pen[1], None, None)
        np.testing.assert_array_equal(tok.cpu().numpy(), wt)
        hist[np.arange(3), lens] = wt
        hist_d[torch.arange(3, device=DEV), lens_d.long()] = tok.to(torch.int16)
        lens += 1
        lens_d += 1


def test_captured_step_replays_with_new_contents():
    """One captured step (append, attend over parts, control), replayed as the
    sequences grow, with eager work and waits in between, against the same
    calls made eagerly on a second cache."""
    r = np.random.default_rng(31)
    heads, kvh, dh, P, vocab, steps = 6, 2, 64, 32, 9000, 6
    table, pages, cos, sin, run = serving_steps(r, [(0, 600), (0, 1), (0, 90)], steps, vocab=vocab)
    pools = [Pool(np.random.default_rng(1), pages, kvh, P, dh) for _ in range(2)]
    g = [dev(x) for x in (cos, sin)]
    start, offsets, rows, x, lg = run[0]
    d = dev(x)
    for p in pools:
        p.cache.Append(batch_of(table, start, offsets, rows), None, d[:, heads:heads + kvh], d[:, heads + kvh:], *g)
    t_d = dev(table, np.int32)
    s_d = dev(run[1][0], np.int32)
    o_d = dev(run[1][1], np.int32)
    b = ane.KVBatch(t_d, s_d, o_d, 3, max_len=1000, max_new=1)
    x_d, lg_d = dev(run[1][3]), dev(run[1][4])
    mask = torch.full(((vocab + 31) // 32,), 0x5f5f5f5f, dtype=torch.int32, device=DEV)
    ctl = ane.LogitControls(vocab, mask=mask)

    def step(cache, x, lg, b):
        q = cache.Append(b, x[:, :heads], x[:, heads:heads + kvh], x[:, heads + kvh:], *g)
        return cache.Attend(b, q), ctl.Apply(lg)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):      # a warm-up on a pool of its own
        step(Pool(np.random.default_rng(2), pages, kvh, P, dh).cache, x_d, lg_d, b)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(pools[0].cache, x_d, lg_d, b)
    for start, offsets, rows, x, lg in run[1:]:
        s_d.copy_(dev(start, np.int32))
        x_d.copy_(dev(x))
        lg_d.copy_(dev(lg))
        graph.replay()
        eager = step(pools[1].cache, dev(x), dev(lg), batch_of(table, start, offsets, rows, max_len=1000, max_new=1))
        torch.cuda.synchronize()
        assert torch.equal(captured[0], eager[0])
        assert torch.equal(captured[1][0], eager[1][0]) and torch.equal(captured[1][1], eager[1][1])
        for a, c in zip(pools[0].held(), pools[1].held()):
            np.testing.assert_array_equal(a, c)


def test_empty_calls():
    """Batches without rows or sequences, logits without rows."""
    pool = Pool(np.random.default_rng(33), 2, 2, 16, 64)
    before = pool.held()
    x = torch.zeros((0, 8, 64), dtype=torch.float16, device=DEV)
    cs = torch.zeros((32, 32), device=DEV)
    for b in (batch_of(np.array([[0, 1]]), np.array([0]), np.array([0, 0]), 0),
              batch_of(np.zeros((0, 2)), np.zeros(0), np.array([0]), 0)):
        assert pool.cache.Append(b, x[:, :4], x[:, 4:6], x[:, 6:], cs, cs).shape == (0, 4, 64)
        assert pool.cache.Attend(b, x).shape == (0, 8, 64)
    out, tok = ane.LogitControls(70).Apply(torch.zeros((0, 70), device=DEV))
    assert out.shape == (0, 70) and tok.shape == (0,)
    torch.cuda.synchronize()
    for a, c in zip(before, pool.held()):
        np.testing.assert_array_equal(a, c)


def test_two_streams_at_once():
    """Long attentions in parts and logits on two streams at the same time:
    each as alone."""
    r = np.random.default_rng(32)
    lens = [[(9000, 1), (8000, 1)], [(7000, 4)]]
    sides = []
    for ls in lens:
        table, start, offsets, pages = layout(r, ls, 64)
        pool = Pool(r, pages, 2, 64, 64)
        n = int(offsets[-1])
        sides.append((pool, batch_of(table, start, offsets, n), dev(r.standard_normal((n, 8, 64)).astype(np.float16)),
                      dev(r.standard_normal((5, 50000)).astype(np.float32))))
    ctl = ane.LogitControls(50000)
    alone = [(p.cache.Attend(b, q), *ctl.Apply(lg)) for p, b, q, lg in sides]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sides]
    got = [[], []]
    for _ in range(10):
        for k, (p, b, q, lg) in enumerate(sides):
            with torch.cuda.stream(streams[k]):
                got[k].append((p.cache.Attend(b, q), *ctl.Apply(lg)))
    torch.cuda.synchronize()
    for k in range(2):
        for trio in got[k]:
            assert all(torch.equal(a, c) for a, c in zip(trio, alone[k]))


@pytest.mark.parametrize("nseq", [65, 700, 4200])
def test_many_sequences(nseq):
    """More sequences than one round of the search takes (64 and 4096), a few
    without new rows."""
    r = np.random.default_rng(nseq)
    lens = [(int(r.integers(0, 20)), int(r.choice([0, 1, 1, 1, 3]))) for _ in range(nseq)]
    run_append(np.random.default_rng(1), lens, 2, 1, 64, 16)
    run_attend(np.random.default_rng(2), lens, 2, 1, 64, 16, max_new=3, max_len=23)


def test_nonsense_offsets_and_starts_stay_inside():
    """What lies outside is not followed: no fault, and memory before and
    behind the tensors is as it was."""
    r = np.random.default_rng(50)
    P, kvh, heads, dh, pages, rows = 16, 2, 4, 64, 6, 40
    wild = np.array([-2**31, -7, 0, 3, 2**30, 2**31 - 1])
    cos, sin = (dev(x) for x in rope_tables(3 * P, dh))
    for seed in range(6):
        r = np.random.default_rng(seed)
        nseq = int(r.integers(1, 90))
        pool = Pool(r, pages + 2, kvh, P, dh)
        c = pool.cache
        # a cache and rows inside larger ones, whose ends must not change
        inner = ane.KVCache8(c.k[1:-1], c.v[1:-1], c.k_exp[1:-1], c.v_exp[1:-1])
        table = np.where(r.random((nseq, 3)) < 0.3, r.choice(wild, (nseq, 3)), r.integers(0, pages, (nseq, 3)))
        start = np.where(r.random(nseq) < 0.3, r.choice(wild, nseq), r.integers(0, 60, nseq))
        offsets = np.where(r.random(nseq + 1) < 0.3, r.choice(wild, nseq + 1), r.integers(0, rows, nseq + 1))
        x = torch.zeros((rows + 2, heads + 2 * kvh, dh), dtype=torch.float16, device=DEV)
        q_out = torch.full((rows + 2, heads, dh), 7.0, dtype=torch.float16, device=DEV)
        out = torch.full((rows + 2, heads, dh), 7.0, dtype=torch.float16, device=DEV)
        before = pool.held()
        b = batch_of(table, start, offsets, rows)
        y = x[1:-1]
        inner.Append(b, y[:, :heads], y[:, heads:heads + kvh], y[:, heads + kvh:], cos, sin, q_out[1:-1])
        inner.Attend(b, q_out[1:-1], out[1:-1])
        torch.cuda.synchronize()
        for t in (q_out, out):
            assert (t[[0, -1]] == 7.0).all()
        for p, a in zip(before, pool.held()):
            np.testing.assert_array_equal(p[[0, -1]], a[[0, -1]])


def test_refusals():
    r = np.random.default_rng(40)
    pool = Pool(r, 4, 2, 16, 64)
    c = pool.cache
    b = batch_of(np.array([[0, 1]]), np.array([0]), np.array([0, 5]), 5)
    x = torch.zeros((5, 8, 64), dtype=torch.float16, device=DEV)
    cs = torch.zeros((32, 32), device=DEV)

    def bad(word, f, *a, **k):
        with pytest.raises(ane.EngineError, match=word) as e:
            f(*a, **k)
        assert e.value.code == _lib.ANE_ERR_ARG
    bad("float32, want", c.Attend, b, x.float())
    bad("want \\(5, heads, 64\\)", c.Attend, b, x[:4])
    bad("on cpu", c.Attend, b, x.cpu())
    bad("heads=3", c.Attend, b, x[:, :3])
    bad("last dimension", c.Attend, b, x.transpose(1, 2).contiguous().transpose(1, 2))
    bad("overlap", c.Attend, b, x, torch.zeros((1, 8, 64), dtype=torch.float16, device=DEV).expand(5, 8, 64))
    bad("scale", c.Attend, b, x, scale=0.0)
    bad("aligned", c.Attend, b, torch.zeros(5 * 512 + 1, dtype=torch.float16, device=DEV)[1:].view(5, 8, 64))
    bad("multiple of 8", c.Attend, b, torch.zeros((5, 8, 68), dtype=torch.float16, device=DEV)[:, :, :64])
    bad("positions=31", c.Append, b, x[:, :4], x[:, 4:6], x[:, 6:], cs[:31], cs[:31])
    bad("cos", c.Append, b, x[:, :4], x[:, 4:6], x[:, 6:], cs[:, :16].contiguous(), cs[:, :16].contiguous())
    bad("k has shape", c.Append, b, x[:, :4], x[:, 4:7], x[:, 6:], cs, cs)
    bad("q_out without q", c.Append, b, None, x[:, 4:6], x[:, 6:], cs, cs, x[:, :4])
    bad("other strides", c.Append, b, x[:, :4], x[:, 4:6], x[:, 6:], cs, cs,
        torch.as_strided(x, (5, 4, 64), (256, 64, 1)))
    bad("offsets has shape", batch_of, np.array([[0, 1]]), np.array([0]), np.array([0, 5, 6]), 5)
    bad("int64", ane.KVBatch, torch.zeros((1, 2), dtype=torch.int64, device=DEV), None, None, 5)
    bad("GPU", ane.KVBatch, torch.zeros((1, 2), dtype=torch.int32), None, None, 5)
    bad("v has shape", ane.KVCache8, c.k, c.k, c.k_exp, c.v_exp)
    bad("page_tokens=48", ane.KVCache8.Empty(2, 2, 64, 48).Attend, b, x)
    bad("head_dim=96", ane.KVCache8.Empty(2, 2, 96, 16).Attend, b, torch.zeros((5, 8, 96), dtype=torch.float16,
                                                                               device=DEV))
    lg = torch.zeros((2, 100), device=DEV)
    one = torch.ones(2, device=DEV)
    bad("penalties without", ane.LogitControls(100, repetition=one).Apply, lg)
    bad("without lengths", ane.LogitControls(100, repetition=one).Apply, lg,
        torch.zeros((2, 3), dtype=torch.int16, device=DEV))
    bad("logits have shape", ane.LogitControls(99).Apply, lg)
    bad("others have 2", ane.LogitControls, 100, repetition=one, presence=torch.ones(3, device=DEV))
    bad("bias has shape", ane.LogitControls, 100, bias=torch.zeros(99, device=DEV))
    bad("mask has shape", ane.LogitControls, 100, mask=torch.zeros(3, dtype=torch.int32, device=DEV))
