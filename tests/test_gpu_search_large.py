"""Beam search, the tables of pages and the choice of pages where offsets pass 32
bits, and captured together."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import ane  # noqa: E402

DEV = "cuda"


def ids(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def test_logits_and_histories_of_more_than_2_to_the_32_bytes():
    rows, vocab, hist = 40000, 60001, 54000     # 2.4e9 logits, 2.2e9 ids
    logits = torch.zeros((rows, vocab), dtype=torch.float16, device=DEV)
    history = torch.full((rows, hist), 7, dtype=torch.int16, device=DEV)
    lengths = torch.full((rows,), hist - 1, dtype=torch.int32, device=DEV)
    last = rows - 4
    logits[last, 59999], logits[last + 1, 3], logits[last + 1, 60000], logits[last + 2, 1] = 9, 11, 10, 1
    history[last + 1, ::1000] = 1234
    tokens, parents, _ = ane.BeamSearch(vocab, 4).Select(logits, torch.zeros(rows, device=DEV), history=history,
                                                         lengths=lengths)
    assert tokens[last:].tolist() == [3, 60000, 59999, 1]
    assert parents[last:].tolist() == [last + 1, last + 1, last, last + 2]
    assert tokens[:8].tolist() == [0, 1, 2, 3] * 2 and parents[:8].tolist() == [0] * 4 + [4] * 4
    assert (lengths == hist).all()
    assert history[last:, -1].view(torch.uint16).to(torch.int32).tolist() == [3, 60000, 59999, 1]
    for row, from_one in ((last, True), (last + 1, True), (last + 2, False), (last + 3, False)):
        want = torch.full((hist - 1,), 7, dtype=torch.int16, device=DEV)
        if from_one:
            want[::1000] = 1234
        assert torch.equal(history[row, :-1], want)


def test_pages_behind_2_to_the_32_bytes():
    P, kvh, dh, pages = 64, 4, 64, 280_000       # 4.6e9 bytes of keys, as many of values
    cache = ane.KVCache8.Empty(pages, kvh, dh, P)
    bounds = ane.KVBounds.Empty(cache)
    g = torch.Generator(device=DEV).manual_seed(1)
    k, v = cache.k.view(torch.uint8), cache.v.view(torch.uint8)
    high = torch.tensor([pages - 1, pages - 2, pages - 7, pages - 9], device=DEV)
    for t in (k, v):
        t[high] = torch.randint(0, 0x70, (4, *t.shape[1:]), dtype=torch.uint8, device=DEV, generator=g)
    cache.k_exp[high], cache.v_exp[high] = -7, -6
    low = torch.tensor([3, 5, 8, 2], device=DEV)
    pool = ane.KVPages.Empty([cache], [bounds])
    pool.Copy(high.int(), low.int())
    for t in (k, v, cache.k_exp, cache.v_exp):
        assert torch.equal(t[high], t[low])

    # the same sequence in the high pages and in the low ones
    q = torch.randn((2, 8, dh), device=DEV, generator=g).half()
    table = torch.stack([high.int(), low.int()])
    whole = ane.KVBatch(table, ids([0, 0]), ids([0, 200, 400]), 400, max_new=200)
    bounds.Update(whole)
    batch = ane.KVBatch(table, ids([199, 199]), ids([0, 1, 2]), 2, max_new=1)
    q[1] = q[0]
    blocks = bounds.Select(batch, q, 3)
    assert torch.equal(blocks[0], blocks[1])
    assert torch.equal(bounds.box[high], bounds.box[low]) and torch.equal(bounds.unit[high], bounds.unit[low])
    out = cache.Attend(batch, q, blocks=blocks)
    assert torch.equal(out[0], out[1]) and out[0].abs().max() > 0
    chunk = ane.KVBatch(table, ids([0, 0]), ids([0, 200, 400]), 400, max_new=200)
    rows = torch.randn((200, 8, dh), device=DEV, generator=g).half().repeat(2, 1, 1)
    named = torch.randint(-1, 4, (200, kvh, 5), dtype=torch.int32, device=DEV, generator=g).repeat(2, 1, 1)
    out = cache.Attend(chunk, rows, blocks=named)
    assert torch.equal(out[:200], out[200:])

    # held by the high pages' sequence alone: a fork copies the last page to the lowest free one,
    # and compacting moves all but that
    pool.refs[high] = 1
    row, start = torch.full((2, 4), -1, dtype=torch.int32, device=DEV), ids([200, 0])
    row[0] = high.int()
    before = [t[high].clone() for t in (k, v, cache.k_exp, cache.v_exp, bounds.box)]
    assert int(pool.Fork(row, start, parents=ids([0, 0]))) == 0
    assert row.tolist() == [[pages - 1, pages - 2, pages - 7, pages - 9], [pages - 1, pages - 2, pages - 7, 0]]
    # 200 tokens: 8 in the last page, one unit of 16
    assert torch.equal(k[0, :, :16], before[0][3, :, :16]) and torch.equal(v[0, :, 0], before[1][3, :, 0])
    moved = pool.Compact(row)
    assert moved[high].tolist() == [4, 3, 2, 1] and int(moved[0]) == 0
    assert sorted(set(row.flatten().tolist())) == [0, 1, 2, 3, 4]
    for t, b in zip((k, v, cache.k_exp, cache.v_exp, bounds.box), before):
        assert torch.equal(t[[4, 3, 2, 1]], b)
    assert pool.refs[:5].tolist() == [1, 1, 2, 2, 2] and int(pool.refs.sum()) == 8


def test_compact_and_copy_captured():
    """Replayed over other tables, between eager calls and synchronizations."""
    r = np.random.default_rng(3)
    pages, layers = 200, 3
    caches = [ane.KVCache8.Empty(pages, 2, 64, 16) for _ in range(layers)]
    pool = ane.KVPages.Empty(caches)
    table = torch.full((6, 9), -1, dtype=torch.int32, device=DEV)
    src, dst = ids([0] * 5), ids([0] * 5)
    moved = ids([0] * pages)

    def step():
        pool.Copy(src, dst)
        pool.Compact(table, moved=moved)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
    for i in range(4):
        held = r.permutation(pages)[:54]
        state = []
        for t in [x for c in caches for x in (c.k, c.v)]:
            t.view(torch.uint8).copy_(torch.randint(0, 256, t.shape, dtype=torch.uint8, device=DEV))
        table.copy_(ids(held.reshape(6, 9)))
        pool.refs.zero_()
        pool.refs[table.flatten().long()] = 1
        src.copy_(ids(held[:5]))
        dst.copy_(ids(held[20:25]))
        start = [x.clone() for c in caches for x in (c.k.view(torch.uint8), c.v.view(torch.uint8))] + [
            table.clone(), pool.refs.clone()]
        torch.cuda.synchronize()
        for run in (graph.replay, step):
            now = [x for c in caches for x in (c.k.view(torch.uint8), c.v.view(torch.uint8))] + [table, pool.refs]
            for a, b in zip(now, start):
                a.copy_(b)
            moved.fill_(-9)
            torch.cuda.synchronize()
            run()
            torch.cuda.synchronize()
            t = table.long()
            assert sorted(t.flatten().tolist()) == list(range(54))
            # what the table's pages hold is as before, behind the copies
            ref = [x.clone() for x in start[:2 * layers]]
            for x in ref:
                x[dst.long()] = x[src.long()]
            for x, y in zip(now, ref):
                assert torch.equal(x[t], y[start[-2].long()])
            state.append([moved.clone(), table.clone(), pool.refs.clone()])
        assert all(torch.equal(a, b) for a, b in zip(*state))
