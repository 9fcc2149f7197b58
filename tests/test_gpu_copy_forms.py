"""Copies and compactions of many pages (``ane.KVPages``), below and above the
size from which they go past the caches: every byte of every page."""
import numpy as np
import pytest

import pages_ref as ref
import search_forms as forms

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import ane  # noqa: E402

DEV = "cuda"


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).to(DEV)


def layers_of(g, pages, layers, kvh, dh, P, bare=()):
    """Caches of random bytes and their bounds (None for the layers in `bare`)."""
    def some(shape, lo=0, hi=256, dtype=torch.uint8):
        return torch.randint(lo, hi, shape, dtype=dtype, device=DEV, generator=g)
    caches, bounds = [], []
    for l in range(layers):
        f8 = torch.float8_e4m3fn
        c = ane.KVCache8(some((pages, kvh, P, dh)).view(f8), some((pages, kvh, P // 16, 4, 16, dh // 16, 4)).view(f8),
                         some((pages, kvh), -15, 9, torch.int8), some((pages, kvh), -15, 9, torch.int8))
        caches.append(c)
        bounds.append(None if l in bare else ane.KVBounds(c, some((pages, kvh, 2, dh), -128, 128, torch.int8),
                                                          some((pages, kvh), -30, 10, torch.int8)))
    return caches, bounds


def tensors(caches, bounds):
    """[(tensor, its pages in 16-token units, or None), ...] of each layer."""
    out = []
    for c, b in zip(caches, bounds):
        n, h, P, dh = c.k.shape
        out.append([(c.k.view(torch.uint8).view(n, h, P // 16, 16 * dh), True),
                    (c.v.view(torch.uint8).view(n, h, P // 16, 16 * dh), True), (c.k_exp, False), (c.v_exp, False)]
                   + ([(b.box, False), (b.unit, False)] if b else []))
    return out


def copied(src, dst, tokens, P):
    """lay(new, whole, into): `into` when the first tokens of the pages src of `new`,
    in whole units, are laid over its pages dst."""
    def lay(new, whole, into):
        want = into.clone()
        page = new[src]
        if tokens is None:
            want[dst] = page
            return want
        units = (tokens.clamp(0, P) + 15) // 16
        if whole:
            mask = torch.arange(P // 16, device=DEV)[None, None, :, None] < units[:, None, None, None]
        else:
            mask = (units > 0).view(-1, *[1] * (new.dim() - 1))
        want[dst] = torch.where(mask, page, want[dst])
        return want
    return lay


@pytest.mark.parametrize("case", forms.COPY, ids=str)
@pytest.mark.parametrize("part", [False, True], ids=["whole", "tokens"])
def test_copy(case, part):
    size, form = case
    assert forms.copy_form(**size) == form
    size = dict(size)
    n, P = size.pop("pages"), size["P"]
    g = torch.Generator(device=DEV).manual_seed(n + part)
    a, b = layers_of(g, n + 7, bare=(1,), **size), layers_of(g, n + 12, bare=(2,), **size)
    src, dst = (torch.randperm(m, device=DEV, generator=g)[:n] for m in (n + 7, n + 12))
    tokens = torch.randint(-3, P + 9, (n,), device=DEV, generator=g) if part else None
    lay = copied(src, dst, tokens, P)
    want = []
    for l, (x, y) in enumerate(zip(tensors(*a), tensors(*b))):
        both = a[1][l] is not None and b[1][l] is not None
        want.append([lay(s, whole, t) if i < 4 or both else t.clone() for i, ((s, whole), (t, _)) in enumerate(zip(x, y))]
                    + [t.clone() for t, _ in y[len(x):]])
    before = [[s.clone() for s, _ in x] for x in tensors(*a)]
    pools = [ane.KVPages.Empty(*x) for x in (a, b)]
    pools[0].Copy(src.int(), dst.int(), tokens=None if tokens is None else tokens.int(), into=pools[1])
    for x, w in zip(tensors(*b), want):
        assert len(x) == len(w)
        for (t, _), u in zip(x, w):
            assert torch.equal(t, u)
    for x, w in zip(tensors(*a), before):
        assert all(torch.equal(t, u) for (t, _), u in zip(x, w))


# pages of a pool, half of them held in no order: a quarter moves
@pytest.mark.parametrize("pages, far, size", [
    (13000, 1, dict(layers=2, kvh=4, dh=64, P=64)),
    (1600, 1, dict(layers=3, kvh=4, dh=128, P=256)),
    (20000, 1, dict(layers=5, kvh=2, dh=64, P=32)),
    (136000, 1, dict(layers=3, kvh=1, dh=64, P=16)),
    (8000, 0, dict(layers=2, kvh=4, dh=64, P=64)),
])
@pytest.mark.parametrize("order", ["mixed", "end"])
def test_compact(pages, far, size, order):
    r = np.random.default_rng(pages)
    refs = r.integers(1, 4, pages).astype(np.int32)
    held = r.permutation(pages) < pages // 2 if order == "mixed" else np.arange(pages) >= pages * 3 // 4
    refs[~held] = 0
    table = r.integers(-2, pages + 2, (9, 50)).astype(np.int32)
    moved, want_refs, want_table, copies = ref.compact(refs, table)
    assert forms.copy_form(pages=len(copies), **size)[0] == far
    g = torch.Generator(device=DEV).manual_seed(pages)
    caches, bounds = layers_of(g, pages, bare=(1,), **size)
    src, dst = (dev(np.array(x)).long() for x in zip(*copies))
    lay = copied(src, dst, None, size["P"])
    want = [[lay(t, whole, t) for t, whole in x] for x in tensors(caches, bounds)]
    pool = ane.KVPages(caches, dev(refs), bounds)
    t = dev(table)
    got = pool.Compact(t)
    np.testing.assert_array_equal(got.cpu().numpy(), moved)
    np.testing.assert_array_equal(pool.refs.cpu().numpy(), want_refs)
    np.testing.assert_array_equal(t.cpu().numpy(), want_table)
    for x, w in zip(tensors(caches, bounds), want):
        assert all(torch.equal(a, b) for (a, _), b in zip(x, w))


def test_captured_past_the_caches():
    """A copy and a compaction above the line, replayed over other pools, with
    eager ones between."""
    r = np.random.default_rng(5)
    size, pages, n = dict(layers=2, kvh=4, dh=64, P=64), 14000, 3500
    assert forms.copy_form(pages=n, **size)[0] == 1
    g = torch.Generator(device=DEV).manual_seed(7)
    caches, bounds = layers_of(g, pages, **size)
    pool = ane.KVPages.Empty(caches, bounds)
    src, dst, moved = (torch.zeros(m, dtype=torch.int32, device=DEV) for m in (n, n, pages))

    def step():
        pool.Copy(src, dst)
        pool.Compact(moved=moved)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
    for _ in range(3):
        start = [[t.clone() for t, _ in x] for x in tensors(caches, bounds)]
        order = r.permutation(pages)
        refs = np.zeros(pages, np.int32)
        refs[order[:pages // 2]] = 1
        src.copy_(dev(order[:n].astype(np.int32)))
        dst.copy_(dev(order[n:2 * n].astype(np.int32)))
        want_moved, want_refs, _, copies = ref.compact(refs)
        a, b = (dev(np.array(x)).long() for x in zip(*copies))
        for run in (graph.replay, step):
            for x, y in zip(tensors(caches, bounds), start):
                for (t, _), u in zip(x, y):
                    t.copy_(u)
            pool.refs.copy_(dev(refs))
            moved.fill_(-9)
            torch.cuda.synchronize()
            run()
            torch.cuda.synchronize()
            np.testing.assert_array_equal(moved.cpu().numpy(), want_moved)
            np.testing.assert_array_equal(pool.refs.cpu().numpy(), want_refs)
            for x, y in zip(tensors(caches, bounds), start):
                for (t, _), u in zip(x, y):
                    w = u.clone()
                    w[dst.long()] = w[src.long()]
                    w[b] = w[a]
                    assert torch.equal(t, w)
