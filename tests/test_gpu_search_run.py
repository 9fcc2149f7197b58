"""Beam search over the paged 8-bit cache as a program runs it: append, bounds,
choice of pages, attention, controls, selection and fork, step by step, against
the same search in plain 64-bit steps on caches that are whole.

The two models' logits differ by the fp16 roundings of their layers, so a choice
between close candidates may differ; the plain search then goes on from the
GPU's, and most steps have to agree as they are."""
import numpy as np
import pytest

import pages_ref as ref
import serve_ref
from test_gpu_serve import dev, rope_tables

torch = pytest.importorskip("torch")
pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore:overflow encountered", "ignore:invalid value")]

import ane  # noqa: E402

DEV = "cuda"
P, KVH, HEADS, DH, VOCAB, LAYERS = 16, 2, 4, 64, 257, 2
DIM = HEADS * DH


def model(seed):
    r = np.random.default_rng(seed)
    m = dict(embed=r.standard_normal((VOCAB, DIM)))
    for l in range(LAYERS):
        m[l] = r.standard_normal((DIM, (HEADS + 2 * KVH) * DH)) / DIM ** 0.5, r.standard_normal((DIM, DIM)) / DIM ** 0.5
    return m


def plain_logits(m, ids, cos, sin):
    """The model over one whole sequence in 64 bits: logits of its last token.
    Keys and values are held as the cache holds them, a page's exponent over the
    page, row by row as they arrive."""
    x = m["embed"][ids]
    for l in range(LAYERS):
        w, o = m[l]
        y = (x @ w).astype(np.float16).astype(np.float64).reshape(len(ids), HEADS + 2 * KVH, DH)
        pages = -(-len(ids) // P)
        k, v = np.zeros((2, pages, KVH, P, DH))
        ke, ve = np.zeros((2, pages, KVH), int)
        table = np.arange(pages)[None]
        cuts = m["cuts"] + list(range(m["cuts"][-1] + 1, len(ids) + 1))
        q = serve_ref.rope(y[:, :HEADS], cos[:len(ids)], sin[:len(ids)]).astype(np.float16)
        for a, b in zip(cuts, cuts[1:]):
            serve_ref.append(k, v, ke, ve, table, np.array([a]), np.array([0, b - a]), y[a:b, HEADS:HEADS + KVH],
                             y[a:b, HEADS + KVH:], cos, sin)
        out, _ = serve_ref.attend(k, v, ke, ve, table, np.array([0]), np.array([0, len(ids)]), q, DH ** -0.5)
        x = x + out.reshape(len(ids), DIM) @ o
    return x[-1] @ m["embed"].T / DIM ** 0.5 * 3


@pytest.mark.parametrize("seed, beams, compact", [(0, 4, False), (1, 3, True), (2, 6, True)])
def test_search(seed, beams, compact):
    r = np.random.default_rng(seed)
    m = model(seed)
    prompts = [r.integers(0, VOCAB, n) for n in (37, 16, 21)]
    requests, rows = len(prompts), len(prompts) * beams
    width, steps, eos, pages = 6, 12, 5, 60
    cos, sin = rope_tables(width * P, DH)
    cos64, sin64 = cos.astype(np.float64), sin.astype(np.float64)

    caches = [ane.KVCache8.Empty(pages, KVH, DH, P) for _ in range(LAYERS)]
    bounds = [ane.KVBounds.Empty(c) for c in caches]
    pool = ane.KVPages.Empty(caches, bounds)
    table = torch.full((rows, width), -1, dtype=torch.int32, device=DEV)
    start = torch.zeros(rows, dtype=torch.int32, device=DEV)
    search = ane.BeamSearch(VOCAB, beams, eos=eos)
    controls = ane.LogitControls(VOCAB, repetition=torch.full((rows,), 1.2, device=DEV))
    hist = torch.zeros((rows, 64), dtype=torch.int16, device=DEV)
    lens = torch.zeros(rows, dtype=torch.int32, device=DEV)
    scores = torch.full((rows,), float("-inf"), device=DEV)
    scores[::beams] = 0
    done = torch.zeros(rows, dtype=torch.bool, device=DEV)
    w = {l: (dev(m[l][0]).double(), dev(m[l][1]).double()) for l in range(LAYERS)}
    embed = dev(m["embed"])

    def forward(tokens, offsets, most):
        """The new tokens' rows through the layers; logits of each."""
        n = len(tokens)
        batch = ane.KVBatch(table, start, dev(offsets, np.int32), n, max_new=most)
        x = embed[torch.as_tensor(tokens, device=DEV).long()]
        for l in range(LAYERS):
            y = (x @ w[l][0]).half().view(n, HEADS + 2 * KVH, DH)
            q, k, v = y.split([HEADS, KVH, KVH], 1)
            q = caches[l].Append(batch, q, k, v, dev(cos), dev(sin))
            bounds[l].Update(batch)
            # enough places for every page: the choice is then all of them
            blocks = bounds[l].Select(batch, q, width)
            x = x + caches[l].Attend(batch, q, blocks=blocks).double().view(n, DIM) @ w[l][1]
        return (x @ embed.t().contiguous() / DIM ** 0.5 * 3).float()

    # the prompts, in the first beam of each request; the others fork from it
    news = np.zeros(rows, np.int32)
    news[::beams] = [len(p) for p in prompts]
    assert int(pool.Fork(table, start, new=dev(news))) == 0
    offsets = np.concatenate([[0], np.cumsum(news)])
    x = forward(np.concatenate(prompts), offsets, int(news.max()))
    last = np.repeat(np.cumsum([len(p) for p in prompts]) - 1, beams)
    logits = x[torch.as_tensor(last, device=DEV)]
    start += dev(news)
    for i, p in enumerate(prompts):
        hist[i * beams:(i + 1) * beams, :len(p)] = dev(p.astype(np.int16))
        lens[i * beams:(i + 1) * beams] = len(p)

    # the plain search
    seqs = [list(p) for p in prompts for _ in range(beams)]
    s_plain = np.full(rows, -np.inf)
    s_plain[::beams] = 0
    d_plain = np.zeros(rows, bool)
    clear = 0
    for step in range(steps):
        logits, _ = controls.Apply(logits, hist, lens)
        tokens, parents, scores = search.Select(logits, scores, finished=done, history=hist, lengths=lens)
        missing = pool.Fork(table, start, parents=parents, new=1)
        if compact and step % 3 == 2:
            pool.Compact(table)
        torch.cuda.synchronize()
        assert int(missing) == 0

        z = np.empty((rows, VOCAB))
        for i, ids in enumerate(seqs):
            if step == 0 and i % beams:
                z[i] = 0
                continue
            n = len(prompts[i // beams])
            m["cuts"] = [0, n]
            z[i] = plain_logits(m, np.array(ids), cos64, sin64)
            ids = np.unique(ids)
            z[i, ids] = np.where(z[i, ids] > 0, z[i, ids] / np.float32(1.2), z[i, ids] * np.float32(1.2))
        h = np.zeros((rows, 64), np.uint16)
        n = np.array([len(s) for s in seqs], np.int32)
        for i, s in enumerate(seqs):
            h[i, :len(s)] = s
        want = ref.beam_select(z, s_plain, beams, None, d_plain, eos, h, n)
        # scores differ by the fp16 and fp32 roundings of two layers; choices have to be the same where the plain
        # ones are clear, and are taken over from the GPU where they are not
        np.testing.assert_allclose(scores.cpu().numpy(), want["scores"], atol=2e-2 * (step + 1))
        same = (tokens.cpu().numpy() == want["tokens"]) & (parents.cpu().numpy() == want["parents"])
        clear += same.all()
        hn, ln = hist.cpu().numpy().view(np.uint16), lens.cpu().numpy()
        if same.all():
            np.testing.assert_array_equal(ln, want["lengths"])
            for i in range(rows):
                np.testing.assert_array_equal(hn[i, :ln[i]], want["history"][i, :ln[i]])
        seqs = [[int(t) for t in hn[i, :ln[i]]] for i in range(rows)]
        s_plain, d_plain = scores.cpu().numpy().astype(np.float64), done.cpu().numpy()
        refs = pool.refs.cpu().numpy()
        t = table.cpu().numpy()
        np.testing.assert_array_equal(refs, np.bincount(t[t >= 0], minlength=pages))
        # a finished beam's row goes on with its last token: its logits are not looked at
        logits = forward(tokens.cpu().numpy(), np.arange(rows + 1), 1)
        start += 1
    assert clear >= steps * 2 // 3
