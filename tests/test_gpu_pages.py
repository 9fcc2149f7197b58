"""The tables of the cache's pages on the GPU (``ane.KVPages``) against plain
implementations (pages_ref.py): tables, counts and every byte of the pages
equal."""
import numpy as np
import pytest

import pages_ref as ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import ane  # noqa: E402

DEV = "cuda"


def dev(x, dtype=None):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=dtype)).to(DEV)


class Pool:
    """Layers of random pages, on the host and on the GPU."""

    def __init__(self, r, pages, layers=2, kvh=2, P=16, dh=64, bounds=False):
        self.P = P
        self.host, self.boxes = [], []
        self.caches, self.bounds = [], []
        for l in range(layers):
            k = r.integers(0, 256, (pages, kvh, P, dh)).astype(np.uint8)
            v = r.integers(0, 256, (pages, kvh, P // 16, 4, 16, dh // 16, 4)).astype(np.uint8)
            ke, ve = (r.integers(-15, 9, (pages, kvh)).astype(np.int8) for _ in range(2))
            self.host.append([k, v, ke, ve])
            f8 = torch.float8_e4m3fn
            c = ane.KVCache8(dev(k).view(f8), dev(v).view(f8), dev(ke), dev(ve))
            self.caches.append(c)
            if bounds and l % 3 != 1:   # some layer without
                box = r.integers(-128, 128, (pages, kvh, 2, dh)).astype(np.int8)
                u = r.integers(-30, 10, (pages, kvh)).astype(np.int8)
                self.boxes.append([box, u])
                self.bounds.append(ane.KVBounds(c, dev(box), dev(u)))
            else:
                self.boxes.append(None)
                self.bounds.append(None)

    def copy(self, copies, into=None):
        into = into or self
        # all are read before any is written
        old = [[x.copy() for x in layer] for layer in self.host]
        old_box = [b and [x.copy() for x in b] for b in self.boxes]
        for l in range(len(self.host)):
            for src, dst, tokens in copies:
                ref.copy_units(*old[l], src, into.host[l], dst, tokens, old_box[l], into.boxes[l])

    def check(self):
        for l, (c, host) in enumerate(zip(self.caches, self.host)):
            for t, x in zip((c.k.view(torch.uint8), c.v.view(torch.uint8), c.k_exp, c.v_exp), host):
                np.testing.assert_array_equal(t.cpu().numpy(), x, err_msg=f"layer {l}")
            if self.boxes[l]:
                np.testing.assert_array_equal(self.bounds[l].box.cpu().numpy(), self.boxes[l][0])
                np.testing.assert_array_equal(self.bounds[l].unit.cpu().numpy(), self.boxes[l][1])


def beams(r, P, requests, width, lens, beams_each, pages):
    """Tables of requests whose beams share all pages but their last one or two."""
    ids = list(r.permutation(pages))
    table = np.full((requests * beams_each, width), -1, np.int32)
    for q in range(requests):
        held = -(-lens[q] // P)
        alone = min(held, int(r.integers(1, 3)))
        shared = [ids.pop() for _ in range(held - alone)]
        for w in range(beams_each):
            table[q * beams_each + w, :held] = shared + [ids.pop() for _ in range(alone)]
    refs = np.bincount(table[table >= 0], minlength=pages).astype(np.int32)
    return table, np.repeat(lens, beams_each).astype(np.int32), refs


def run_fork(pool, table, start, refs, parents, new, stride=0, with_bounds=False):
    """One fork on the GPU and plainly; both states must agree."""
    n, width = table.shape
    room = torch.full((n, width + stride), 777, dtype=torch.int32, device=DEV)
    t = room[:, :width]
    t.copy_(dev(table))
    s, c = dev(start, np.int32), dev(refs, np.int32)
    pages = ane.KVPages(pool.caches, c, pool.bounds if with_bounds else None)
    news = [new] * n if np.isscalar(new) else new
    got = pages.Fork(t, s, parents=None if parents is None else dev(parents, np.int32),
                     new=new if np.isscalar(new) else dev(new, np.int32))
    torch.cuda.synchronize()
    wt, ws, wr, missing, copies = ref.fork(table, start, refs, pool.P, parents, news)
    np.testing.assert_array_equal(t.cpu().numpy(), wt)
    np.testing.assert_array_equal(s.cpu().numpy(), ws)
    np.testing.assert_array_equal(c.cpu().numpy(), wr)
    assert int(got) == missing
    if stride:
        assert (room[:, width:] == 777).all()
    pool.copy(copies)
    pool.check()
    return wt, ws, wr, missing, copies


@pytest.mark.parametrize("P, kvh, dh", [(16, 1, 64), (32, 3, 128), (64, 4, 64), (128, 2, 64), (256, 1, 128), (16, 8, 64)])
def test_beams_go_on(P, kvh, dh):
    r = np.random.default_rng(P + kvh)
    lens = np.array([3 * P + 5, P, 2 * P + 15, 1, 2 * P - 1])
    pages = 90
    table, start, refs = beams(r, P, 5, 5, lens, 4, pages)
    pool = Pool(r, pages, 3, kvh, P, dh, bounds=True)
    for step in range(4):
        parents = np.repeat(np.arange(5) * 4, 4) + r.integers(0, 4, 20)
        table, start, refs, missing, copies = run_fork(pool, table, start, refs, parents, 1, stride=step,
                                                       with_bounds=True)
        assert missing == 0
        start = start + 1
    assert copies


def test_all_beams_from_one():
    r = np.random.default_rng(0)
    pool = Pool(r, 40)
    table, start, refs = beams(r, 16, 1, 4, np.array([37]), 8, 40)
    wt, _, refs, _, copies = run_fork(pool, table, start, refs, np.full(8, 3), 1)
    assert len(copies) == 7 and (wt[1:, 2] != wt[0, 2]).all() and wt[0, 2] == table[3, 2]


@pytest.mark.parametrize("seed", range(6))
def test_anything_goes(seed):
    """Parents of other requests, ended sequences, cut-off starts, several new
    tokens, holders outside the table, pools that run out, nonsense ids."""
    r = np.random.default_rng(seed)
    P = 16
    requests, each, width, pages = 4, 3, 6, [80, 30, 26, 200, 33, 64][seed]
    lens = r.integers(1, 3 * P, requests)
    table, start, refs = beams(r, P, requests, width, lens, each, max(pages, 40))
    pages = max(pages, 40) if seed not in (1, 2) else 40
    pool = Pool(r, pages, 1)
    refs[r.integers(0, pages, 5)] += 1          # others hold some
    if seed in (1, 2):
        refs[r.random(pages) < 0.9] += 1        # hardly any is free
    n = len(start)
    for _ in range(5):
        parents = r.integers(-2, n + 2, n)
        new = r.integers(0, 40, n)
        start = np.maximum(start - r.integers(0, 9, n), 0)
        if seed == 5:
            table[r.random(table.shape) < 0.1] = r.choice([-7, pages, 2**31 - 1, -2**31])
            start[r.random(n) < 0.2] = r.choice([-5, 10**6])
        table, start, refs, missing, _ = run_fork(pool, table, start, refs, parents, new)
        start = np.minimum(start + new, width * P).astype(np.int32)


@pytest.mark.parametrize("nseq, width", [(1, 1), (1, 300), (1500, 2), (2100, 3)])
def test_reserve_truncate_and_free(nseq, width):
    r = np.random.default_rng(nseq + width)
    P, pages = 16, nseq * width + 4200
    pool = Pool(r, pages, 1, 1)
    table = np.full((nseq, width), -1, np.int32)
    start, refs = np.zeros(nseq, np.int32), np.zeros(pages, np.int32)
    refs[r.random(pages) < 0.4] = 1   # held elsewhere; more than enough left? maybe not: missing counts
    new = r.integers(0, width * P + 5, nseq)
    table, start, refs, missing, copies = run_fork(pool, table, start, refs, None, new)
    assert not copies
    start = np.minimum(new, width * P)
    run = run_fork(pool, table, (start // 2).astype(np.int32), refs, None, 0)
    table, start, refs, _, _ = run
    held = int((refs > 0).sum())
    table, start, refs, _, _ = run_fork(pool, table, np.zeros(nseq, np.int32), refs, None, 0)
    assert (table == -1).all() and int((refs > 0).sum()) <= held


def test_many_layers_take_more_launches():
    r = np.random.default_rng(1)
    pool = Pool(r, 30, 70, 1)
    table, start, refs = beams(r, 16, 2, 4, np.array([37, 20]), 4, 30)
    run_fork(pool, table, start, refs, np.array([1, 1, 0, 3, 4, 4, 4, 4]), 1)
    moved(pool, refs, None)
    held = Pool(r, 20, 70, 1)
    copy_pages(pool, held, [3, 5], [7, 1], [9, 16])


def test_page_with_another_holder_is_left_to_it():
    """A page that somebody outside the call holds is copied by all its writers;
    one that a sequence without new tokens holds, too."""
    r = np.random.default_rng(2)
    pool = Pool(r, 12)
    table = np.array([[1, 2], [1, 2], [1, 2]], np.int32)
    refs = np.zeros(12, np.int32)
    refs[[1, 2]] = 3
    more = refs.copy()
    more[2] += 1
    *_, copies = run_fork(pool, table, np.full(3, 20, np.int32), more, None, 1)
    assert len(copies) == 3
    *_, copies = run_fork(pool, table, np.full(3, 20, np.int32), refs, None, np.array([1, 0, 1]))
    assert len(copies) == 2


def test_page_that_is_not_there_stays_so():
    r = np.random.default_rng(3)
    pool = Pool(r, 12)
    refs = np.zeros(12, np.int32)
    refs[4] = 1
    wt, *_, missing, _ = run_fork(pool, np.array([[4, -1, -1]], np.int32), np.array([20], np.int32), refs, None, 30)
    assert missing == 1 and wt[0, 1] == -1 and wt[0, 2] == -1 or wt[0, 2] == 0


def test_pool_is_exhausted():
    r = np.random.default_rng(4)
    pool = Pool(r, 6)
    table, start = np.full((3, 4), -1, np.int32), np.zeros(3, np.int32)
    table, start, refs, missing, _ = run_fork(pool, table, start, np.zeros(6, np.int32), None, 40)
    assert missing == 3 and (table[2, :] == -1).all()


def test_no_sequences():
    pool = Pool(np.random.default_rng(5), 5)
    run_fork(pool, np.full((0, 3), -1, np.int32), np.zeros(0, np.int32), np.ones(5, np.int32), None, 1)


# ---- compact


def moved(pool, refs, table, with_bounds=False):
    c = dev(refs, np.int32)
    pages = ane.KVPages(pool.caches, c, pool.bounds if with_bounds else None)
    t = None if table is None else dev(table, np.int32)
    got = pages.Compact(t)
    torch.cuda.synchronize()
    wm, wr, wt, copies = ref.compact(refs, table)
    np.testing.assert_array_equal(got.cpu().numpy(), wm)
    np.testing.assert_array_equal(c.cpu().numpy(), wr)
    if table is not None:
        np.testing.assert_array_equal(t.cpu().numpy(), wt)
    pool.copy([(a, b, pool.P) for a, b in copies])
    pool.check()
    return copies


@pytest.mark.parametrize("pages", [1, 2, 63, 1000, 4095, 4096, 4097, 9000])
@pytest.mark.parametrize("fill", [0.0, 0.3, 0.8, 1.0])
def test_compact(pages, fill):
    r = np.random.default_rng(pages)
    pool = Pool(r, pages, 1 if pages > 100 else 4, 1, bounds=True)
    refs = (r.random(pages) < fill).astype(np.int32) * r.integers(1, 5, pages).astype(np.int32)
    refs[r.random(pages) < 0.05] = -3
    table = r.integers(-3, pages + 3, (7, 40)).astype(np.int32)
    moved(pool, refs, table, with_bounds=True)


@pytest.mark.parametrize("P, kvh, dh", [(256, 2, 128), (32, 5, 64)])
def test_compact_from_one_end_to_the_other(P, kvh, dh):
    r = np.random.default_rng(P)
    pool = Pool(r, 40, 2, kvh, P, dh)
    refs = np.zeros(40, np.int32)
    refs[20:] = 1
    assert len(moved(pool, refs, None)) == 20


# ---- copy


def copy_pages(pool, into, src, dst, tokens, **kw):
    a = ane.KVPages(pool.caches, torch.zeros(pool.host[0][0].shape[0], dtype=torch.int32, device=DEV), pool.bounds)
    b = a if into is pool else ane.KVPages(into.caches, torch.zeros(into.host[0][0].shape[0], dtype=torch.int32,
                                                                    device=DEV), into.bounds)
    a.Copy(dev(src, np.int32), dev(dst, np.int32), None if tokens is None else dev(tokens, np.int32),
           into=None if into is pool else b)
    torch.cuda.synchronize()
    n, m = pool.host[0][0].shape[0], into.host[0][0].shape[0]
    pool.copy([(s, d, pool.P if tokens is None else min(max(int(tokens[i]), 0), pool.P))
               for i, (s, d) in enumerate(zip(src, dst)) if 0 <= s < n and 0 <= d < m], into)
    into.check()
    pool.check()


@pytest.mark.parametrize("P, kvh, dh", [(16, 2, 64), (64, 3, 128), (256, 2, 64)])
def test_copy_to_another_pool(P, kvh, dh):
    r = np.random.default_rng(P)
    a, b = Pool(r, 30, 3, kvh, P, dh, bounds=True), Pool(r, 19, 3, kvh, P, dh, bounds=True)
    src, dst = r.permutation(30)[:15], r.permutation(19)[:15]
    tokens = r.integers(-3, P + 9, 15)
    tokens[:4] = [0, 1, 16, P]
    copy_pages(a, b, src, dst, tokens)
    copy_pages(a, b, src, dst, None)
    copy_pages(a, b, [3, -1, 30, 5, 2], [-1, 4, 4, 19, 2**31 - 1], None)   # none of these is there
    copy_pages(a, a, [1, 2], [9, 8], [5, 16])
    copy_pages(a, a, [], [], None)


def test_bounds_of_one_side_alone_do_not_move():
    r = np.random.default_rng(7)
    a, b = Pool(r, 8, 1, bounds=True), Pool(r, 8, 1)
    copy_pages(a, b, [1], [2], None)
    copy_pages(b, a, [1], [2], None)


# ---- the manner of the calls


def test_refusals():
    r = np.random.default_rng(8)
    pool, other = Pool(r, 9), Pool(r, 9, P=32)
    i32 = dict(dtype=torch.int32, device=DEV)
    refs = torch.zeros(9, **i32)
    p = ane.KVPages(pool.caches, refs)
    t, s = torch.full((2, 3), -1, **i32), torch.zeros(2, **i32)
    for call in (lambda: ane.KVPages([], refs), lambda: ane.KVPages(pool.caches, refs[:8]),
                 lambda: ane.KVPages(pool.caches, refs.float()), lambda: ane.KVPages(pool.caches + other.caches, refs),
                 lambda: ane.KVPages(pool.caches, refs, [None]), lambda: p.Fork(t, s[:1]), lambda: p.Fork(t.long(), s),
                 lambda: p.Fork(t.t(), s), lambda: p.Fork(t, s, new=-1), lambda: p.Fork(t, s, parents=s[:1]),
                 lambda: p.Fork(t, s, parents=s), lambda: p.Fork(t, s, new=s.long()), lambda: p.Fork(t[:, :0], s),
                 lambda: p.Fork(t.cpu(), s), lambda: p.Fork(t, s, missing=s), lambda: p.Fork(t, s, missing=refs[:1]),
                 lambda: p.Compact(moved=refs), lambda: p.Compact(moved=s), lambda: p.Compact(t.float()),
                 lambda: p.Copy(s, s[:1]), lambda: p.Copy(s, s, tokens=s[:1]), lambda: p.Copy(s.long(), s),
                 lambda: p.Copy(s, s, into=ane.KVPages.Empty(other.caches)),
                 lambda: ane.KVBounds(pool.caches[0], torch.zeros(3, dtype=torch.int8, device=DEV), refs)):
        with pytest.raises(ane.EngineError):
            call()


def test_captured_forks():
    """A captured fork and compact, replayed with other tables and with eager
    work between, each time the eager result."""
    r = np.random.default_rng(9)
    pool = Pool(r, 60, 2)
    i32 = dict(dtype=torch.int32, device=DEV)
    refs, t, s, par = torch.zeros(60, **i32), torch.full((8, 5), -1, **i32), torch.zeros(8, **i32), torch.zeros(8, **i32)
    missing, to = torch.zeros(1, **i32), torch.zeros(60, **i32)
    p = ane.KVPages(pool.caches, refs)

    def step():
        p.Fork(t, s, parents=par, new=1, missing=missing)
        p.Compact(t, moved=to)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
    for _ in range(4):
        table, start, c = beams(r, 16, 2, 5, r.integers(1, 60, 2), 4, 60)
        parents = np.repeat([0, 4], 4) + r.integers(0, 4, 8)
        for x, y in ((t, table), (s, start), (refs, c), (par, parents)):
            x.copy_(dev(y, np.int32))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        table, start, c, m, copies = ref.fork(table, start, c, 16, parents, [1] * 8)
        pool.copy(copies)
        wm, c, table, moves = ref.compact(c, table)
        pool.copy([(a, b, 16) for a, b in moves])
        np.testing.assert_array_equal(t.cpu().numpy(), table)
        np.testing.assert_array_equal(refs.cpu().numpy(), c)
        np.testing.assert_array_equal(to.cpu().numpy(), wm)
        assert int(missing) == m
        pool.check()


@pytest.mark.parametrize("nseq, width", [(1024, 8), (1025, 8), (1024, 9), (3000, 4)])
def test_every_size_of_table(nseq, width):
    """By one block, and by many; writers of shared pages by hashing and by
    marks."""
    r = np.random.default_rng(nseq + width)
    P, pages = 16, nseq * 3 + 100
    pool = Pool(r, pages, 1, 1)
    table = np.full((nseq, width), -1, np.int32)
    ids = r.permutation(pages)
    table[:, 0], table[:, 1] = ids[:nseq], ids[nseq + r.integers(0, nseq // 2, nseq)]   # second pages shared
    start = r.integers(17, 31, nseq).astype(np.int32)
    refs = np.bincount(table[table >= 0], minlength=pages).astype(np.int32)
    refs[table[::7, 1]] += 1
    run_fork(pool, table, start, refs, r.integers(0, nseq, nseq), r.integers(0, 20, nseq))


def test_copies_of_many_small_pages():
    """Four sides a block, more layers than make whole fours, and past the
    caches."""
    r = np.random.default_rng(10)
    for layers, kvh, P, n in ((5, 1, 16, 600), (3, 2, 16, 900), (7, 4, 16, 2100)):
        a, b = Pool(r, n + 5, layers, kvh, P), Pool(r, n + 9, layers, kvh, P, bounds=True)
        copy_pages(a, b, r.permutation(n + 5)[:n], r.permutation(n + 9)[:n], r.integers(0, P + 1, n))
        copy_pages(a, b, r.permutation(n + 5)[:n], r.permutation(n + 9)[:n], None)


def test_copies_of_more_pages_than_a_launch_takes():
    r = np.random.default_rng(11)
    a, b = Pool(r, 6, 32, 1), Pool(r, 5, 32, 1)
    n = 1 << 22
    src = np.full(n, -1)
    at = [0, n // 2 - 1, n // 2, n - 1]
    src[at] = [5, 2, 0, 3]
    dst = np.full(n, 4)
    dst[at] = [1, 3, 2, 0]
    copy_pages(a, b, src, dst, None)
    copy_pages(b, a, src, dst, r.integers(0, 17, n))


@pytest.mark.parametrize("pages", [20480, 20481, 24576, 41000])
def test_large_pools(pages):
    """Hardly any page is free, and those lie far apart, or at the end; then none
    is; fewer and more sequences than a block has threads."""
    r = np.random.default_rng(pages)
    pool = Pool(r, pages, 1, 1)
    for requests, each, width, free in ((4, 3, 6, 40), (4, 3, 6, 5), (300, 4, 4, 4000), (300, 4, 4, 300)):
        lens = r.integers(1, 3 * 16, requests)
        table, start, refs = beams(r, 16, requests, width, lens, each, pages)
        others = np.ones(pages, int)
        others[r.permutation(pages)[:free] if free != 300 else slice(-free, None)] = 0
        refs = refs + others
        n = len(start)
        for parents in (None, np.repeat(np.arange(requests) * each, each)):
            new = r.integers(0, 40, n)
            table, start, refs, missing, _ = run_fork(pool, table, start, refs, parents, new)
            start = np.minimum(start + new, width * 16).astype(np.int32)
        assert (missing > 0) == (free in (5, 300))


def test_captured_forks_in_a_large_pool():
    r = np.random.default_rng(31)
    pages, P, width = 20500, 16, 5
    c = Pool(r, pages, 1, 1)
    refs, table, start = (torch.zeros(n, dtype=torch.int32, device=DEV) for n in (pages, (24, width), 24))
    parents, missing = torch.zeros(24, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    p = ane.KVPages(c.caches, refs)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        p.Fork(table, start, parents=parents, new=20, missing=missing)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            p.Fork(table, start, parents=parents, new=20, missing=missing)
    for i in range(4):
        t, s, f = beams(r, P, 6, width, r.integers(1, 3 * P, 6), 4, pages)
        others = (r.random(pages) < (0.99, 1.0, 0.9, 0.999)[i]).astype(int)
        f = f + others
        q = np.repeat(np.arange(6) * 4, 4) + r.integers(0, 4, 24)
        for x, y in ((table, t), (start, s), (refs, f), (parents, q)):
            x.copy_(dev(y, np.int32))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        wt, ws, wr, wm, _ = ref.fork(t, s, f, P, q, [20] * 24)
        np.testing.assert_array_equal(table.cpu().numpy(), wt)
        np.testing.assert_array_equal(start.cpu().numpy(), ws)
        np.testing.assert_array_equal(refs.cpu().numpy(), wr)
        assert int(missing) == wm and (wm > 0) == (i in (1, 3))
        p.Fork(table, start, parents=parents, new=1)      # eager between the replays
        torch.cuda.synchronize()
