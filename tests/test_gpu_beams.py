"""Beam search's step on the GPU (``ane.BeamSearch``) against a plain 64-bit
implementation (pages_ref.beam_select): choices and states equal, scores within
what the kernel's fp32 exponentials leave."""
import numpy as np
import pytest

import pages_ref as ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import ane  # noqa: E402

DEV = "cuda"


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).to(DEV)


class Case:
    """Inputs of a step; rows of logits and histories `wide` elements apart."""

    def __init__(self, r, requests, beams, vocab, half=False, hist=20, eos=None, weights=True, wide=0, masked=0.0):
        n = requests * beams
        self.beams, self.vocab, self.eos, self.half = beams, vocab, eos, half
        x = r.standard_normal((n, vocab)) * 3
        x[r.random((n, vocab)) < masked] = -np.inf
        self.logits = x.astype(np.float16 if half else np.float32)
        self.scores = (-20 - 2 * r.standard_normal(n)).astype(np.float32)
        self.weights = (1 / r.uniform(3, 9, n)).astype(np.float32) if weights else None
        self.finished = r.random(n) < 0.3 if eos is not None else None
        self.history = r.integers(0, 65536, (n, hist)).astype(np.uint16) if hist is not None else None
        self.lengths = r.integers(0, hist + 1, n).astype(np.int32) if hist is not None else None
        self.wide = wide

    def run(self, in_place=False, offset=0):
        n, v = self.logits.shape
        pad = torch.full((n * (v + self.wide) + offset,), float("nan"), device=DEV,
                         dtype=torch.float16 if self.half else torch.float32)
        logits = torch.as_strided(pad, (n, v), (v + self.wide, 1), offset)
        logits.copy_(dev(self.logits))
        search = ane.BeamSearch(v, self.beams, eos=self.eos)
        scores = dev(self.scores)
        kw = dict(scores_out=scores) if in_place else {}
        if self.weights is not None:
            kw["weights"] = dev(self.weights)
        if self.finished is not None:
            kw["finished"] = dev(self.finished)
            if not in_place:
                kw["finished_out"] = torch.full((n,), 9, dtype=torch.uint8, device=DEV)
        hist = lengths = None
        if self.history is not None:
            m = self.history.shape[1]
            room = torch.full((n * (m + self.wide) + offset,), 4321, dtype=torch.int16, device=DEV)
            hist = torch.as_strided(room, (n, m), (m + self.wide, 1), offset)
            hist.copy_(dev(self.history.view(np.int16)))
            lengths = dev(self.lengths)
        tokens, parents, out = search.Select(logits, scores, history=hist, lengths=lengths, **kw)
        torch.cuda.synchronize()
        got = dict(tokens=tokens.cpu().numpy(), parents=parents.cpu().numpy(), scores=out.cpu().numpy())
        if self.finished is not None:
            got["finished"] = (kw["finished"] if in_place else kw["finished_out"]).cpu().numpy().astype(int)
        if hist is not None:
            got["history"], got["lengths"] = hist.cpu().numpy().view(np.uint16), lengths.cpu().numpy()
            if self.wide:
                between = torch.as_strided(room, (n - 1, self.wide), (m + self.wide, 1), offset + m)
                assert (between == 4321).all()
        return got

    def want(self):
        return ref.beam_select(self.logits, self.scores, self.beams, self.weights, self.finished,
                               -1 if self.eos is None else self.eos, self.history, self.lengths)

    def check(self, **kw):
        got, want = self.run(**kw), self.want()
        for name in ("tokens", "parents", "history", "lengths", "finished"):
            if name in got:
                np.testing.assert_array_equal(got[name], want[name], err_msg=name)
        there = want["parents"] >= 0
        assert (got["scores"][~there] == -np.inf).all()
        same = got["scores"] == want["scores"]   # infinities
        err = np.abs(np.where(same, 0, got["scores"].astype(np.float64) - np.where(same, 0, want["scores"])))
        assert (err[there] <= want["tol"][there]).all(), (err[there] / want["tol"][there]).max()
        return got


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("vocab", [1, 2, 31, 255, 256, 257, 511, 513, 2048, 2049, 5001, 32000])
def test_vocabularies(vocab, half):
    r = np.random.default_rng(vocab)
    for beams in (1, 3, 8):
        Case(r, 2, beams, vocab, half).check()


@pytest.mark.parametrize("half", [False, True])
def test_largest_vocabulary_and_most_beams(half):
    r = np.random.default_rng(5)
    Case(r, 1, 32, 65535, half, hist=3).check()
    Case(r, 2, 5, 60011, half, eos=60010).check()


@pytest.mark.parametrize("beams", [1, 2, 3, 4, 5, 7, 8, 11, 16, 17, 27, 31, 32])
def test_beams(beams):
    r = np.random.default_rng(beams)
    Case(r, 3, beams, 777, eos=3).check()
    Case(r, 3, beams, 777, eos=3, half=True, weights=False).check(in_place=True)


def test_many_requests():
    r = np.random.default_rng(1)
    Case(r, 300, 2, 101, eos=0).check()
    Case(r, 65535, 1, 2, hist=2).check()


@pytest.mark.parametrize("wide", [1, 3, 8, 130])
@pytest.mark.parametrize("half", [False, True])
def test_rows_apart_and_unaligned(wide, half):
    r = np.random.default_rng(wide)
    Case(r, 2, 5, 1003, half, eos=9, wide=wide).check(offset=1)
    Case(r, 2, 4, 3001, half, hist=700, wide=wide).check(offset=7)


@pytest.mark.parametrize("masked", [0.5, 0.97, 0.999])
def test_masks(masked):
    r = np.random.default_rng(int(masked * 1000))
    c = Case(r, 4, 6, 900, eos=5, masked=masked)
    c.logits[3] = -np.inf            # a beam with nothing to offer
    c.logits[12:18] = -np.inf        # a request with nothing but its finished beams
    c.check()
    c.finished[:] = False
    c.check()


def test_nothing_at_all():
    r = np.random.default_rng(2)
    c = Case(r, 2, 4, 50, eos=1)
    c.finished[:4] = False
    c.logits[:4] = -np.inf
    got = c.check()
    assert (got["tokens"][:4] == ane.NO_TOKEN).all() and (got["parents"][:4] == -1).all()
    assert (got["lengths"][:4] == 0).all() and (got["finished"][:4] == 0).all()


def test_first_step_has_one_beam():
    r = np.random.default_rng(3)
    c = Case(r, 5, 8, 400)
    c.scores[:] = -np.inf
    c.scores[::8] = 0
    got = c.check()
    assert (got["parents"] == np.repeat(np.arange(5) * 8, 8)).all()


def test_fewer_candidates_than_beams():
    r = np.random.default_rng(4)
    c = Case(r, 2, 16, 3, eos=2)
    c.scores[2:16] = -np.inf
    c.finished[:2] = False
    got = c.check()
    assert (got["parents"][6:16] == -1).all() and (got["parents"][:6] >= 0).all()


def test_scores_and_weights_that_are_none():
    r = np.random.default_rng(6)
    c = Case(r, 3, 6, 300, eos=4)
    c.scores[0], c.scores[7] = np.nan, -np.inf
    c.weights[2], c.weights[8], c.weights[13] = 0.0, -1.0, np.nan
    c.check()


def test_nan_and_infinite_logits():
    r = np.random.default_rng(7)
    c = Case(r, 3, 4, 600)
    c.logits[r.random(c.logits.shape) < 0.05] = np.nan
    c.logits[2] = np.nan
    c.logits[5, 77] = np.inf         # its log sum is no number: the beam offers nothing
    c.check()
    h = Case(r, 2, 4, 600, half=True)
    h.logits[1, :] = np.float16(-65504)
    h.logits[1, 9] = np.float16(65504)
    h.logits[6, 5] = -np.float16(np.inf)
    h.check()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("beams", [3, 16, 32])
def test_ties_go_to_the_lower_beam_and_token(beams, half):
    """Equal rows of few values: most candidates are equal."""
    r = np.random.default_rng(beams)
    c = Case(r, 2, beams, 4000, half, weights=False)
    c.logits[:] = r.integers(0, 3, 4000)[None]
    c.scores[:] = np.repeat([-4.0, -9.0], beams)
    c.check()
    c.logits[:] = 0
    c.check()
    c.logits[:] = -np.sort(r.standard_normal(4000))[None]   # the best ones next to each other
    c.scores += r.standard_normal(2 * beams).astype(np.float32)
    c.check()


def test_signed_zeros_are_equal():
    c = Case(np.random.default_rng(8), 1, 4, 10, weights=False)
    c.logits[:] = -5
    c.logits[0, [3, 4, 7]] = [0.0, -0.0, 0.0]
    c.scores[1:] = -1000
    got = c.check()
    assert got["tokens"].tolist()[:3] == [3, 4, 7]


@pytest.mark.parametrize("hist", [0, 1, 2, 7, 8, 9, 15, 64, 1000, 9001])
def test_histories(hist):
    r = np.random.default_rng(hist)
    for beams in (1, 5, 32):
        c = Case(r, 2, beams, 90, hist=hist, eos=0)
        c.lengths[0] = hist
        c.lengths[-1] = 0
        c.check(in_place=True)
        c.lengths[:] = hist           # full: the token has no room
        c.check()
        c.lengths[:] = np.where(r.random(len(c.lengths)) < 0.5, -7, 1 << 30)
        c.check()


def test_no_history_and_no_end():
    Case(np.random.default_rng(9), 3, 4, 256, hist=None).check()


def test_of_nothing():
    s = ane.BeamSearch(100, 4)
    t, p, o = s.Select(torch.empty((0, 100), device=DEV), torch.empty(0, device=DEV))
    assert t.shape == p.shape == o.shape == (0,)


def test_refusals():
    s = ane.BeamSearch(100, 4, eos=3)
    x, z = torch.zeros((8, 100), device=DEV), torch.zeros(8, device=DEV)
    f = torch.zeros(8, dtype=torch.bool, device=DEV)
    for call in (lambda: s.Select(x.double(), z, f), lambda: s.Select(x[:7], z[:7], f[:7]), lambda: s.Select(x, z),
                 lambda: s.Select(x[:, :99], z, f), lambda: s.Select(x, z[:7], f), lambda: s.Select(x, z.half(), f),
                 lambda: s.Select(x, z, f.int()), lambda: s.Select(x.t().contiguous().t(), z, f),
                 lambda: s.Select(x, z, f, history=torch.zeros((8, 4), dtype=torch.int16, device=DEV)),
                 lambda: s.Select(x, z, f, lengths=torch.zeros(8, dtype=torch.int32, device=DEV)),
                 lambda: s.Select(x.cpu(), z, f), lambda: s.Select(x, z.cpu(), f),
                 lambda: s.Select(x, x.view(-1)[:8], f, scores_out=x.view(-1)[4:12]),
                 lambda: ane.BeamSearch(100, 4).Select(x, z, finished_out=f),
                 lambda: ane.BeamSearch(100, 33), lambda: ane.BeamSearch(0, 3), lambda: ane.BeamSearch(100, 3, eos=100)):
        with pytest.raises(ane.EngineError):
            call()


def test_captured_steps_on_a_stream():
    """A captured step, replayed with other logits and with eager work between,
    each time the eager result."""
    r = np.random.default_rng(10)
    c = Case(r, 3, 5, 3000, eos=11, hist=40)
    n = 15
    logits, scores, fin = dev(c.logits), dev(c.scores), dev(c.finished)
    hist, lens = dev(c.history.view(np.int16)), dev(c.lengths)
    outs = [torch.zeros(n, dtype=t, device=DEV) for t in (torch.int32, torch.int32, torch.float32, torch.bool)]
    search = ane.BeamSearch(3000, 5, eos=11)

    def step():
        search.Select(logits, scores, finished=fin, history=hist, lengths=lens, tokens=outs[0], parents=outs[1],
                      scores_out=outs[2], finished_out=outs[3])
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
    for _ in range(4):
        c = Case(r, 3, 5, 3000, eos=11, hist=40, weights=False)
        for t, x in ((logits, c.logits), (scores, c.scores), (fin, c.finished), (hist, c.history.view(np.int16)),
                     (lens, c.lengths)):
            t.copy_(dev(x))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = c.want()
        np.testing.assert_array_equal(outs[0].cpu().numpy(), want["tokens"])
        np.testing.assert_array_equal(outs[1].cpu().numpy(), want["parents"])
        np.testing.assert_array_equal(outs[3].cpu().numpy(), want["finished"])
        np.testing.assert_array_equal(hist.cpu().numpy().view(np.uint16), want["history"])
        np.testing.assert_array_equal(lens.cpu().numpy(), want["lengths"])


def test_two_calls_at_once():
    r = np.random.default_rng(11)
    cases = [Case(r, 30, 4, 9000, hist=500) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in cases]
    state = [[dev(c.logits), dev(c.scores), dev(c.history.view(np.int16)), dev(c.lengths), dev(c.weights)] for c in cases]
    torch.cuda.synchronize()
    search = ane.BeamSearch(9000, 4)
    got = []
    for s, (x, z, h, n, w) in zip(streams, state):
        with torch.cuda.stream(s):
            got.append(search.Select(x, z, weights=w, history=h, lengths=n))
    torch.cuda.synchronize()
    for c, g, (_, _, h, n, _) in zip(cases, got, state):
        want = c.want()
        np.testing.assert_array_equal(g[0].cpu().numpy(), want["tokens"])
        np.testing.assert_array_equal(g[1].cpu().numpy(), want["parents"])
        np.testing.assert_array_equal(h.cpu().numpy().view(np.uint16), want["history"])


@pytest.mark.parametrize("beams, hist", [(4, 2040), (4, 2056), (4, 4096), (4, 4104), (8, 1023), (8, 2050), (16, 500),
                                         (16, 513), (16, 4095), (16, 4097), (32, 256), (32, 2049), (9, 7000)])
def test_histories_in_every_form(beams, hist):
    """Read ahead, moved by the second launch, and by one of their own."""
    r = np.random.default_rng(beams * 10000 + hist)
    c = Case(r, 2, beams, 64, hist=hist, eos=1, wide=beams % 3)
    c.lengths[:] = np.maximum(hist - r.integers(0, 20, 2 * beams), 0)
    c.lengths[0], c.lengths[-1] = hist, 0
    c.check(offset=beams % 2)


@pytest.mark.parametrize("beams", [8, 9, 16, 32])
@pytest.mark.parametrize("vocab", [64, 300, 5000, 20000])
def test_uneven_groups(beams, vocab):
    """Sorted logits and few segments: far more than a wave's lanes reach the
    first bar."""
    r = np.random.default_rng(vocab)
    for order in (1, -1):
        c = Case(r, 2, beams, vocab, hist=None, weights=False)
        c.logits[:] = np.sort(r.standard_normal((2 * beams, vocab)).astype(np.float32))[:, ::order]
        c.scores[:] = -5 - 1e-3 * np.arange(2 * beams)
        c.check()


def test_scores_far_from_each_other():
    c = Case(np.random.default_rng(12), 2, 6, 500, weights=False)
    c.scores[:] = [0, -1e4, -1e30, 1e30, 3e38, -3e38] * 2
    c.logits[3, 7] = 60000
    c.check()


@pytest.mark.parametrize("half", [False, True])
def test_logits_of_large_magnitude(half):
    r = np.random.default_rng(13)
    c = Case(r, 2, 4, 700, half, weights=False)
    top = 60000.0 if half else 3e38
    c.logits[:4] = (r.uniform(-1, 1, (4, 700)) * top).astype(c.logits.dtype)
    c.logits[4:] = (top - r.integers(0, 3, (4, 700)) * (32 if half else 1e33)).astype(c.logits.dtype)
    c.check()


@pytest.mark.parametrize("x", [49984.0, 58592.0, 63872.0, -63872.0])
def test_large_fp16_maximum(x):
    """Where the maximum times log2(e) is furthest from what 32 bits hold of
    it."""
    c = Case(np.random.default_rng(10), 1, 2, 1000, half=True, weights=False)
    c.scores[:] = [0.0, -0.5]
    c.logits[:] = x
    c.check()


@pytest.mark.parametrize("half", [False, True])
def test_more_candidates_at_the_bar_than_there_is_room_for(half):
    """All of the best segments' candidates equal; and fewer segments than
    beams."""
    r = np.random.default_rng(12)
    c = Case(r, 2, 32, 20000, half, weights=False)
    c.logits[:] = 1.5
    c.scores[:] = -3
    got = c.check()
    assert got["tokens"].tolist() == list(range(32)) * 2
    for beams, vocab in ((32, 7000), (32, 4097), (32, 900), (5, 900), (16, 3000)):
        c = Case(r, 2, beams, vocab, half)
        c.scores[:] = -np.inf
        c.scores[[1, beams + 2]] = -1
        c.check()
        c.logits[:] = np.round(c.logits)      # many equal ones
        c.check()
