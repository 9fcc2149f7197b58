"""Bounds on the keys of pages, the choice of pages and the attention over them
on the GPU (``ane.KVBounds``, ``KVCache8.Attend(blocks=)``) against plain
implementations: bounds and choices equal, attention within the tolerance that
serve_ref.attend derives."""
import numpy as np
import pytest

import pages_ref as ref
import serve_ref
from test_gpu_serve import Pool, batch_of, dev, layout

torch = pytest.importorskip("torch")
pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore:overflow encountered", "ignore:invalid value",
                                                          "ignore:All-NaN")]

import ane  # noqa: E402

DEV = "cuda"


class Run:
    """Sequences of lens[i] = (held, new) over random pages with their bounds."""

    def __init__(self, r, lens, heads=4, kvh=2, dh=64, P=16, nan=0.0, spare=1, rows_behind=2, **hints):
        self.table, self.start, self.offsets, self.pages = layout(r, lens, P, spare)
        self.rows = int(self.offsets[-1]) + rows_behind
        self.pool = Pool(r, self.pages, kvh, P, dh, nan=nan)
        self.lens, self.heads, self.kvh, self.dh, self.P = lens, heads, kvh, dh, P
        self.q = r.standard_normal((self.rows, heads, dh)).astype(np.float16)
        self.box = r.integers(-128, 128, (self.pages, kvh, 2, dh)).astype(np.int8)
        self.unit = r.integers(-12, -6, (self.pages, kvh)).astype(np.int8)
        self.hints = hints

    def go(self):
        self.batch = batch_of(self.table, self.start, self.offsets, self.rows, **self.hints)
        self.bounds = ane.KVBounds(self.pool.cache, dev(self.box), dev(self.unit))
        return self

    def update(self):
        """Update, and the same on the host."""
        self.bounds.Update(self.batch)
        torch.cuda.synchronize()
        k, _, ke, _ = self.pool.held()
        for i, (st, n) in enumerate(self.lens):
            end = min(st + n, self.table.shape[1] * self.P)
            for j in range(st // self.P, -(-end // self.P)) if end > st else ():
                page = int(self.table[i, j])
                if 0 <= page < self.pages:
                    for h in range(self.kvh):
                        x = k[page, h, :min(self.P, end - j * self.P)] * 2.0 ** float(ke[page, h])
                        self.box[page, h], self.unit[page, h] = ref.bound(x)
        np.testing.assert_array_equal(self.bounds.box.cpu().numpy(), self.box)
        np.testing.assert_array_equal(self.bounds.unit.cpu().numpy(), self.unit)
        return self

    def select(self, count, first=1, recent=1, q=None):
        blocks = torch.full((self.rows, self.kvh, count), 99, dtype=torch.int32, device=DEV)
        got = self.bounds.Select(self.batch, dev(self.q) if q is None else q, count, first, recent, blocks)
        torch.cuda.synchronize()
        assert got is blocks
        want = np.full((self.rows, self.kvh, count), 99, np.int32)
        g = self.heads // self.kvh
        for i, (st, n) in enumerate(self.lens):
            for t in range(min(n, self.table.shape[1] * self.P - st)):
                row, np_ = int(self.offsets[i]) + t, (st + t) // self.P + 1
                ids = self.table[i, :np_]
                there = (ids >= 0) & (ids < self.pages)
                ids = np.where(there, ids, 0)
                for h in range(self.kvh):
                    want[row, h] = ref.select(self.q[row, h * g:h * g + g], self.box[ids, h], self.unit[ids, h], there,
                                              count, first, recent)
        np.testing.assert_array_equal(blocks.cpu().numpy(), want)
        return want

    def attend(self, blocks, scale=None, q=None, out=None):
        scale = self.dh ** -0.5 if scale is None else scale
        if out is None:
            out = torch.full((self.rows, self.heads, self.dh), 7.0, dtype=torch.float16, device=DEV)
        self.pool.cache.Attend(self.batch, dev(self.q) if q is None else q, out, scale, blocks=dev(blocks))
        torch.cuda.synchronize()
        got = out.cpu().numpy().astype(np.float64)
        k, v, ke, ve = self.pool.held()
        width, g = self.table.shape[1], self.heads // self.kvh
        for i, (st, n) in enumerate(self.lens):
            for t in range(min(n, width * self.P - st)):
                row, p = int(self.offsets[i]) + t, st + t
                for h in range(self.kvh):
                    # a sequence of the named pages: whole ones first, then what is seen of the last
                    K, V = [], []
                    for b in blocks[row, h]:
                        if not 0 <= b < width or not 0 <= self.table[i, b] < self.pages:
                            continue
                        m = min(max(p + 1 - int(b) * self.P, 0), self.P)
                        page = int(self.table[i, b])
                        K.append(k[page, h, :m] * 2.0 ** float(ke[page, h]))
                        V.append(v[page, h, :m] * 2.0 ** float(ve[page, h]))
                    n_keys = sum(len(x) for x in K)
                    for c in range(h * g, h * g + g):
                        if n_keys == 0:
                            assert (got[row, c] == 0).all()
                            continue
                        # serve_ref.attend on one page that holds just these keys
                        z = np.zeros((1, 1))
                        o, tol = serve_ref.attend(np.concatenate(K)[None, None], np.concatenate(V)[None, None], z, z,
                                                  np.zeros((1, 1), int), np.array([n_keys - 1]), np.array([0, 1]),
                                                  self.q[row:row + 1, c:c + 1], scale)
                        bad = np.isnan(o[0, 0])
                        assert (np.isnan(got[row, c]) == bad).all()
                        assert (np.abs(got[row, c] - o[0, 0]) <= tol[0, 0])[~bad].all(), (row, h, c)
        assert (got[self.offsets[-1]:] == 7.0).all()
        return out


@pytest.mark.parametrize("P", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("kvh, heads, dh", [(1, 1, 64), (2, 6, 64), (3, 3, 128), (1, 16, 64), (1, 17, 128), (2, 64, 64)])
def test_single_tokens(P, kvh, heads, dh):
    r = np.random.default_rng(P + heads)
    lens = [(5 * P + 3, 1), (P - 1, 1), (0, 1), (P, 1), (9 * P - 1, 1)]
    x = Run(r, lens, heads, kvh, dh, P).go().update()
    x.attend(x.select(4))


@pytest.mark.parametrize("count, first, recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (2, 1, 1), (5, 0, 5), (7, 3, 1),
                                                  (64, 1, 1), (65, 0, 0), (300, 10, 20)])
def test_counts(count, first, recent):
    r = np.random.default_rng(count)
    x = Run(r, [(16 * 70 + 5, 1), (40, 2), (16 * 9, 1)], 4, 2, 64, 16).go().update()
    x.attend(x.select(count, first, recent))


@pytest.mark.parametrize("heads, kvh, dh, P", [(4, 2, 64, 16), (12, 4, 64, 64), (6, 1, 128, 32), (40, 2, 128, 16)])
def test_chunks(heads, kvh, dh, P):
    """Ragged chunks of new tokens, some sequences without any, each row its
    own choice."""
    r = np.random.default_rng(heads)
    lens = [(3 * P + 1, 7), (0, 2 * P + 5), (50, 0), (2 * P - 3, 5), (0, 1), (11 * P, 3)]
    x = Run(r, lens, heads, kvh, dh, P).go().update()
    x.attend(x.select(3, 1, 1))
    x.attend(x.select(4, 0, 0))


def test_bounds_of_prompts_and_single_tokens():
    r = np.random.default_rng(1)
    for P, dh in ((16, 64), (64, 128), (256, 64)):
        Run(r, [(0, 3 * P + 7), (P - 1, 1), (P, P), (5, 0), (2 * P + 3, 2), (0, 1)], 2, 2, dh, P).go().update()


def test_bounds_of_special_keys():
    """NaN does not count; a dimension of NaN, a page of zeros, of one value and
    of the largest codes."""
    r = np.random.default_rng(2)
    x = Run(r, [(0, 16 * 6)], 2, 2, 64, 16, nan=0.3)
    t = x.table[0]
    x.pool.kb[t[0]] = 0
    x.pool.kb[t[1]] = 0x80
    x.pool.kb[t[2], :, :, 5] = 0x7f
    x.pool.kb[t[3]] = 0x7e
    x.pool.kb[t[4]] = 0x7f
    x.pool.kb[t[5]] = r.choice([1, 0x81, 0], x.pool.kb[t[5]].shape)
    x.pool.ke[t[3]], x.pool.ke[t[5]] = 8, -15
    x.pool.load()
    x.go().update()


def test_special_queries():
    r = np.random.default_rng(3)
    x = Run(r, [(16 * 40 + 5, 1), (16 * 30, 9)], 4, 2, 64, 16).go().update()
    x.q[0, 0] = 0
    x.q[0, 1, 3] = np.inf
    x.q[1, 0, :] = np.nan
    x.q[2, 1, 5] = -np.inf
    x.q[3] = 6e-8
    x.q[4] = 65504
    x.q[5, 2, 7] = np.nan
    x.select(5)


def test_equal_scores_go_to_the_lower_page():
    r = np.random.default_rng(4)
    x = Run(r, [(16 * 100 + 5, 1), (16 * 20, 3)], 4, 2, 64, 16)
    x.box[:] = x.box[:1]
    x.unit[:] = -8
    x.go()
    w = x.select(6, 0, 0)
    np.testing.assert_array_equal(w[0, 0], np.arange(6))
    x.select(6, 2, 2)


@pytest.mark.parametrize("P, n", [(16, 4095), (16, 4096), (16, 4097), (16, 9000)])
def test_long_contexts(P, n):
    r = np.random.default_rng(n)
    x = Run(r, [(P * (n - 1) + 3, 1), (100, 2)], 2, 1, 64, P, max_len=0 if n == 4097 else P * n).go()
    x.attend(x.select(70, 1, 2))


def test_wrong_hints():
    r = np.random.default_rng(5)
    x = Run(r, [(16 * 300 + 3, 1), (100, 2)], 4, 2, 64, 16, max_len=20, max_new=1).go().update()
    x.attend(x.select(9))


def test_pages_that_are_not_there():
    r = np.random.default_rng(6)
    x = Run(r, [(16 * 12 + 5, 1), (16 * 5, 3)], 4, 2, 64, 16)
    x.table[0, [0, 3, 12]] = [-1, x.pages, 2**31 - 1]
    x.table[1, :] = -5
    x.go().update()
    w = x.select(5)
    assert (w[1] == -1).all()
    x.attend(w)


def test_any_list():
    """Places in no order, twice, behind the row's position, outside the table."""
    r = np.random.default_rng(7)
    x = Run(r, [(16 * 12 + 5, 4), (16 * 3, 2)], 6, 2, 64, 16, nan=0.02).go()
    b = r.integers(-3, 20, (x.rows, 2, 11)).astype(np.int32)
    b[1, 0] = -1
    b[2, 1] = 12
    b[3, 1, :] = [2**31 - 1, -2**31, 0, 0, 5, -1, -1, 12, 13, 3, 1]
    x.attend(b)
    b = r.integers(0, 12, (x.rows, 2, 200)).astype(np.int32)
    b[0, 0, 100:] = -1
    x.attend(b)


def test_all_pages_are_the_whole_attention():
    r = np.random.default_rng(8)
    x = Run(r, [(200, 3), (33, 1)], 6, 2, 128, 32).go()
    b = np.broadcast_to(np.arange(8, dtype=np.int32), (x.rows, 2, 8))
    x.attend(np.ascontiguousarray(b))


def test_positions_behind_the_table():
    r = np.random.default_rng(9)
    x = Run(r, [(28, 10), (3, 2)], 4, 2, 64, 16)
    x.table = np.ascontiguousarray(x.table[:, :2])
    x.lens = [(28, 10), (3, 2)]
    x.go()
    blocks = torch.full((x.rows, 2, 2), 99, dtype=torch.int32, device=DEV)
    x.bounds.Update(x.batch)
    x.bounds.Select(x.batch, dev(x.q), 2, blocks=blocks)
    b = blocks.cpu().numpy()
    assert (b[4:10] == 99).all() and (b[:4] != 99).all() and (b[10:12] != 99).all() and (b[12:] == 99).all()


def test_strided_queries_and_in_place():
    r = np.random.default_rng(10)
    x = Run(r, [(16 * 9 + 5, 2), (40, 1)], 4, 2, 64, 16).go().update()
    wide = torch.zeros((x.rows, 8, 64), dtype=torch.float16, device=DEV)
    q = wide[:, 2:6]
    q.copy_(dev(x.q))
    w = x.select(4, q=q)
    plain = x.attend(w)
    turned = dev(x.q.transpose(1, 0, 2)).transpose(0, 1)
    x.pool.cache.Attend(x.batch, turned, turned, blocks=dev(w))
    n = int(x.offsets[-1])
    assert torch.equal(turned[:n], plain[:n])


def test_of_nothing():
    r = np.random.default_rng(11)
    x = Run(r, [(5, 0)], 4, 2, 64, 16, rows_behind=0).go()
    x.bounds.Update(x.batch)
    b = x.bounds.Select(x.batch, dev(x.q), 3)
    assert b.shape == (0, 2, 3)
    assert x.pool.cache.Attend(x.batch, dev(x.q), blocks=b).shape == (0, 4, 64)


def test_refusals():
    r = np.random.default_rng(12)
    x = Run(r, [(40, 2)], 4, 2, 64, 16).go()
    q = dev(x.q)
    b = torch.zeros((x.rows, 2, 3), dtype=torch.int32, device=DEV)
    c = x.pool.cache
    for call in (lambda: x.bounds.Select(x.batch, q, 0), lambda: x.bounds.Select(x.batch, q, 70000),
                 lambda: x.bounds.Select(x.batch, q, 3, first=2, recent=2), lambda: x.bounds.Select(x.batch, q, 3, first=-1),
                 lambda: x.bounds.Select(x.batch, q.float(), 3), lambda: x.bounds.Select(x.batch, q[:, :3], 3),
                 lambda: x.bounds.Select(x.batch, q, 4, blocks=b), lambda: x.bounds.Select(x.batch, q, 3, blocks=b.long()),
                 lambda: c.Attend(x.batch, q, blocks=b[:2]), lambda: c.Attend(x.batch, q, blocks=b.long()),
                 lambda: c.Attend(x.batch, q, blocks=b[:, :, :0]), lambda: c.Attend(x.batch, q, blocks=b[:, :, ::2]),
                 lambda: ane.KVBounds(c, x.bounds.box[:1], x.bounds.unit)):
        with pytest.raises(ane.EngineError):
            call()


def test_captured():
    """Update, choice and attention captured together, replayed with other
    tables and queries."""
    r = np.random.default_rng(13)
    x = Run(r, [(16 * 60 + 5, 1), (300, 1)], 4, 2, 64, 16).go()
    q = dev(x.q)
    out = torch.zeros((x.rows, 4, 64), dtype=torch.float16, device=DEV)
    b = torch.zeros((x.rows, 2, 40), dtype=torch.int32, device=DEV)

    def step():
        x.bounds.Update(x.batch)
        x.bounds.Select(x.batch, q, 40, blocks=b)
        x.pool.cache.Attend(x.batch, q, out, blocks=b)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
    start = x.batch._keep[1]
    for i in range(4):
        q.copy_(dev(r.standard_normal(x.q.shape).astype(np.float16)))
        start.copy_(dev(np.array([16 * (60 - 7 * i) + 5, 300 - 31 * i], np.int32)))
        torch.cuda.synchronize()
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got, gb = out.clone(), b.clone()
        out.zero_()
        b.fill_(3)
        step()
        torch.cuda.synchronize()
        assert torch.equal(gb[:2], b[:2]) and torch.equal(got[:2], out[:2])


@pytest.mark.parametrize("heads, kvh, dh", [(2, 2, 64), (6, 1, 128), (12, 1, 64), (20, 1, 64), (3, 1, 128)])
def test_long_chunks_and_wrong_hints(heads, kvh, dh):
    """Contexts of more pages than a token's waves hold, with scores in LDS, and
    (hints of a shorter one) without."""
    r = np.random.default_rng(heads)
    for hints in (dict(max_new=3), dict(max_new=3, max_len=100), dict(max_new=1, max_len=100), {}):
        x = Run(r, [(16 * 1100 + 3, 3), (70, 2)], heads, kvh, dh, 16, **hints).go()
        lo = np.minimum(x.box[:, :, 0], x.box[:, :, 1])
        x.box[:, :, 0], x.box[:, :, 1] = np.maximum(x.box[:, :, 0], x.box[:, :, 1]), lo
        x.bounds.box.copy_(dev(x.box))
        x.select(33, 1, 2)


def test_most_scores_in_lds_under_capture():
    r = np.random.default_rng(14)
    x = Run(r, [(16 * 12000 + 3, 1)], 2, 1, 64, 16, max_len=16 * 12001, max_new=1).go()
    q, b = dev(x.q), torch.zeros((x.rows, 1, 50), dtype=torch.int32, device=DEV)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            x.bounds.Select(x.batch, q, 50, blocks=b)
    for _ in range(3):
        b.fill_(77)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = x.select(50)
        np.testing.assert_array_equal(b.cpu().numpy()[:1], want[:1])


def test_scores_far_apart():
    """Outliers, so that the first histograms leave nearly all pages in a bin."""
    r = np.random.default_rng(15)
    x = Run(r, [(16 * 700 + 5, 1), (16 * 300, 2)], 4, 2, 64, 16)
    x.box[:] = r.integers(-3, 4, x.box.shape)
    x.unit[:] = r.choice([-30, -20, -8, 0, 9], x.unit.shape, p=[0.5, 0.3, 0.1, 0.09, 0.01])
    x.go()
    for count in (5, 64, 100, 300):
        x.select(count, 0, 0)
    x.box[:] = 0
    x.bounds.box.zero_()
    x.select(9, 0, 0)


def test_units_that_no_update_wrote_stay_in_range():
    r = np.random.default_rng(16)
    x = Run(r, [(16 * 200 + 5, 1)], 4, 2, 64, 16)
    x.unit[:] = r.choice([-128, -31, 41, 127], x.unit.shape)
    x.go()
    b = x.bounds.Select(x.batch, dev(x.q), 7).cpu().numpy()[0]
    assert ((b >= 0) & (b <= 200)).all() and (np.diff(b, axis=1) > 0).all() and (b[:, 0] == 0).all() and (b[:, -1] == 200).all()


@pytest.mark.parametrize("P, heads, kvh, dh", [(16, 4, 2, 64), (64, 12, 1, 128), (32, 20, 1, 64)])
def test_nan_in_keys_and_values(P, heads, kvh, dh):
    r = np.random.default_rng(17)
    x = Run(r, [(P * 9 + 5, 3), (P * 3, 1), (2, 2)], heads, kvh, dh, P, nan=0.001).go()
    b = np.sort(r.integers(-2, 10, (x.rows, kvh, 4)).astype(np.int32))
    x.attend(b)


@pytest.mark.parametrize("heads, kvh, dh", [(4, 4, 64), (12, 4, 64), (16, 2, 128), (40, 2, 64)])
def test_many_parts(heads, kvh, dh):
    """Lists long enough to be cut, some of them short."""
    r = np.random.default_rng(18)
    x = Run(r, [(64 * 90 + 3, 1), (64 * 3, 1), (7, 1)], heads, kvh, dh, 64).go()
    b = np.full((x.rows, kvh, 80), -1, np.int32)
    b[0] = np.sort(np.stack([r.permutation(91)[:80] for _ in range(kvh)]))
    b[0, 0, 60:] = -1
    b[1, :, :4], b[2, :, 0] = np.arange(4), 0
    x.attend(b)


def test_two_streams_at_once():
    r = np.random.default_rng(19)
    runs = [Run(r, [(64 * 40 + i, 1), (64 * 30, 2)], 4, 2, 64, 64).go() for i in range(2)]
    qs = [dev(x.q) for x in runs]
    torch.cuda.synchronize()
    got = []
    for x, q in zip(runs, qs):
        with torch.cuda.stream(torch.cuda.Stream()):
            x.bounds.Update(x.batch)
            b = x.bounds.Select(x.batch, q, 40)
            got.append((b, x.pool.cache.Attend(x.batch, q, blocks=b)))
    torch.cuda.synchronize()
    for x, q, (b, o) in zip(runs, qs, got):
        n = int(x.offsets[-1])
        w = x.bounds.Select(x.batch, q, 40)
        y = x.pool.cache.Attend(x.batch, q, blocks=w)
        assert torch.equal(b[:n], w[:n]) and torch.equal(o[:n], y[:n])


def lists(r, x, count, twice=False, none=0.1):
    """`count` places a row and head, rising, some behind the position, some no
    place at all."""
    b = np.empty((x.rows, x.kvh, count), np.int32)
    width = x.table.shape[1]
    for i in range(x.rows):
        for h in range(x.kvh):
            b[i, h] = np.sort(r.choice(width, count, replace=twice or count > width))
    b[r.random(b.shape) < none] = -1
    return b


@pytest.mark.parametrize("heads, kvh, dh, P, count, lens", [
    (8, 8, 64, 128, 8, [(128 * 20, 70), (5, 31)]),               # 16 tokens a tile, the last ones of few
    (16, 8, 64, 16, 64, [(16 * 70 + 3, 50), (0, 1), (900, 52)]),
    (24, 8, 128, 32, 16, [(32 * 40, 97)]),
    (32, 8, 64, 256, 4, [(256 * 9 + 200, 61), (1, 40)]),
    (16, 4, 64, 64, 20, [(2000, 161), (2100, 3), (77, 170)]),    # four waves a tile
    (9, 3, 128, 16, 50, [(3000, 220)]),
])
def test_chunks_whose_tokens_share_pages(heads, kvh, dh, P, count, lens):
    r = np.random.default_rng(heads + P)
    x = Run(r, lens, heads, kvh, dh, P).go()
    b = lists(r, x, count)
    b[x.rows // 2] = -1                   # a row that names nothing
    b[:20, 1] = -1                        # tiles that name nothing
    x.attend(b)


def test_chunks_that_name_pages_twice_or_further_than_the_hint():
    r = np.random.default_rng(23)
    lens = [(128 * 18 + 5, 60), (9, 45)]
    x = Run(r, lens, 16, 8, 64, 128).go()
    b = lists(r, x, 8)
    b[0, 0, :2], b[70, 5, 3:] = 4, 0      # twice in some tiles
    x.attend(b)
    x.attend(r.permuted(lists(r, x, 8, twice=True), axis=2))
    y = Run(r, lens, 16, 8, 64, 128, max_len=300, max_new=7).go()
    y.attend(lists(r, y, 8))


@pytest.mark.parametrize("dh, heads", [(64, 24), (128, 8)])
def test_chunks_with_nan_in_pages_of_others(dh, heads):
    r = np.random.default_rng(24)
    x = Run(r, [(128 * 20 + 7, 90)], heads, 8, dh, 128, nan=2e-6).go()
    x.attend(lists(r, x, 8))
    x = Run(r, [(128 * 20 + 7, 90)], heads, 8, dh, 128, nan=1e-3).go()
    x.attend(lists(r, x, 8))


def test_chunks_captured_and_in_place():
    """Lists, starts and queries change between replays."""
    r = np.random.default_rng(25)
    x = Run(r, [(128 * 20, 70), (128 * 12, 40)], 16, 8, 64, 128).go()
    q, b = dev(x.q), dev(lists(r, x, 8))
    work = torch.empty_like(q)

    def step():
        work.copy_(q)
        x.pool.cache.Attend(x.batch, work, work, blocks=b)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
    start = x.batch._keep[1]
    for i in range(4):
        q.copy_(dev(r.standard_normal(x.q.shape).astype(np.float16)))
        b.copy_(dev(lists(r, x, 8, twice=i == 2)))
        start.copy_(dev(np.array([128 * (20 - 3 * i) + i, 128 * 12 - 50 * i], np.int32)))
        torch.cuda.synchronize()
        work.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = work.clone()
        out = torch.zeros_like(q)
        x.pool.cache.Attend(x.batch, q, out, blocks=b)
        torch.cuda.synchronize()
        assert torch.equal(got[:110], out[:110])
        assert torch.equal(got[110:], q[110:])


def test_chunks_with_as_many_places_and_lists_as_lds_holds():
    r = np.random.default_rng(26)
    x = Run(r, [(16 * 8130 + 3, 640)], 1, 1, 64, 16, spare=0).go()
    assert 8160 < x.table.shape[1] <= 8192
    x.attend(lists(r, x, 128, none=0.01))


@pytest.mark.parametrize("heads, kvh, dh, P, count, lens", [
    (12, 4, 64, 16, 7, [(700, 1)] * 201),
    (16, 8, 128, 64, 2, [(130, 1), (0, 1), (63, 3)] * 34),
    (40, 2, 64, 32, 13, [(900, 60), (3, 170), (0, 191)]),
    (24, 1, 128, 16, 30, [(500, 801)]),
])
def test_many_short_lists(heads, kvh, dh, P, count, lens):
    r = np.random.default_rng(heads + count)
    x = Run(r, lens, heads, kvh, dh, P, nan=1e-5, max_new=max(n for _, n in lens)).go()
    b = lists(r, x, count, twice=True, none=0.3)
    b[5:9] = -1
    x.attend(b)


@pytest.mark.parametrize("n, count", [(1024, 7), (1500, 100), (16383, 40), (16384, 40), (16385, 40), (17500, 3000)])
@pytest.mark.parametrize("heads, kvh, dh", [(3, 1, 64), (34, 2, 128)])
def test_long_contexts_in_parts(n, count, heads, kvh, dh):
    """Scores and choice in launches of their own, next to short contexts, and
    with hints of shorter ones."""
    r = np.random.default_rng(n + heads)
    for hints in ({}, dict(max_len=16 * 1100)):
        x = Run(r, [(16 * (n - 1) + 3, 1), (40, 2), (0, 1)], heads, kvh, dh, 16, **hints).go()
        x.box[:, :, 0], x.box[:, :, 1] = np.maximum(x.box[:, :, 0], x.box[:, :, 1]), np.minimum(x.box[:, :, 0],
                                                                                              x.box[:, :, 1])
        x.table[0, r.integers(0, n, 9)] = -1
        x.batch = batch_of(x.table, x.start, x.offsets, x.rows, **hints)
        x.bounds.box.copy_(dev(x.box))
        x.select(count, 1, 2)


@pytest.mark.parametrize("n", [1100, 9000])
def test_long_contexts_of_wide_tables(n):
    """In one launch, as the scores of all places would be too many."""
    r = np.random.default_rng(n)
    x = Run(r, [(16 * (n - 1) + 3, 1), (40, 1)], 3, 1, 64, 16, spare=1 << 21, rows_behind=0, max_len=16 * n).go()
    x.select(50, 1, 2)


def test_long_contexts_in_parts_captured():
    r = np.random.default_rng(29)
    x = Run(r, [(16 * 1500, 1), (16 * 1200, 1)], 4, 2, 64, 16).go()
    q = dev(x.q)
    b = torch.zeros((x.rows, 2, 33), dtype=torch.int32, device=DEV)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        x.bounds.Select(x.batch, q, 33, blocks=b)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            x.bounds.Select(x.batch, q, 33, blocks=b)
    start = x.batch._keep[1]
    for i in range(4):
        q.copy_(dev(r.standard_normal(x.q.shape).astype(np.float16)))
        start.copy_(dev(np.array([16 * (1500 - 300 * i) + i, 16 * 1200 - 999 * i], np.int32)))
        torch.cuda.synchronize()
        b.fill_(-7)
        graph.replay()
        torch.cuda.synchronize()
        got = b.clone()
        b.fill_(-7)
        x.bounds.Select(x.batch, q, 33, blocks=b)
        torch.cuda.synchronize()
        assert torch.equal(got, b) and (b[:2] >= -1).all() and (b[2:] == -7).all()


@pytest.mark.parametrize("heads, kvh, dh, P, count, lens", [
    (40, 8, 64, 128, 8, [(128 * 20, 70), (5, 31)]),             # three tokens a tile
    (48, 8, 128, 64, 16, [(64 * 40 + 3, 50), (0, 1), (900, 52)]),
    (32, 4, 64, 256, 6, [(256 * 9 + 200, 161), (1, 40)]),
])
def test_chunks_of_wide_groups_share_pages(heads, kvh, dh, P, count, lens):
    r = np.random.default_rng(heads + P)
    x = Run(r, lens, heads, kvh, dh, P, nan=3e-6).go()
    b = lists(r, x, count)
    b[x.rows // 2] = -1
    b[:20, 1] = -1
    b[5, 0, :2] = 1                       # twice
    x.attend(b)
