"""The decoder over the paged 8-bit cache (``Decoder.SetCache``) and with
controls on its logits (``Decoder.SetControls``).

The 8-bit decoder is compared with a 64-bit forward of the same model whose keys
and values go through the same cache (serve_ref.append / attend).  What may lie
between the two, with logits of standard deviation s (0.8 to 1 here):

* fp16 weights and activations shift a key or value by about 2^-11 * sqrt(2) *
  0.58 = 4e-4 of itself (two roundings, 0.58 the rms of a uniform error).  Codes
  lie 2^-3 to 2^-4 of a value apart, 9 % on average, so 0.4 % of layer 1's codes
  come out one code away: a noise of sqrt(0.004) * 9 % = 0.6 % on each value,
  from keys (through the scores, whose rms is 1) and from values, 0.8 % of an
  attention output, and, the embedding being small (0.05), of the stream.
* Layer 2's keys and values are thus off by 0.8 %, and 0.8 / 9 of its codes come
  out one away: sqrt(0.09) * 9 % = 2.7 % on each value, 3.8 % of its output, half
  of the stream: 2 % of a logit, rms.  The largest of some 15,000 is 4.2 times
  that, 0.085 s, and 2e-2 is the fp16 path's own (test_gpu_decode.py).

So 0.03 s rms and 0.1 at most.  (A plain emulation of the fp16 roundings in numpy
gives 0.0134 rms and 0.071 at most for the model with the largest.)

The controls are compared bit for bit: the same decoder without them gives the
raw logits, serve_ref.control changes them."""
import numpy as np
import pytest

import ane
import serve_ref as ref
from ane import _lib

pytestmark = pytest.mark.gpu

TOL = 0.1


def check(got, want):
    d = np.abs(got - want)
    rms = np.sqrt((d ** 2).mean())
    print("logits: largest error", d.max(), "rms", rms, "of", want.std())
    assert d.max() <= TOL and rms <= 0.03 * want.std()


def model_in_64_bits(cfg, params, prefix, forced, page):
    """Logits [nseq, 1 + steps, V] of prefix and forced tokens over the 8-bit cache."""
    w = {k: v.astype(np.float64) for k, v in ane.views(cfg, params).items()}
    nseq, plen = prefix.shape
    steps = forced.shape[1]
    H, KV, L = cfg.heads, cfg.kv_heads, cfg.layers
    per = (plen + steps + page - 1) // page
    table = np.arange(nseq * per).reshape(nseq, per)
    pools = [(np.zeros((nseq * per, KV, page, 64)), np.zeros((nseq * per, KV, page, 64)),
              np.zeros((nseq * per, KV), int), np.zeros((nseq * per, KV), int)) for _ in range(L)]
    pos = np.arange(per * page)[:, None] / cfg.rope_theta ** (np.arange(0, 64, 2) / 64)
    cos, sin = np.cos(pos), np.sin(pos)
    norm = lambda x, g: x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-5) * g  # noqa: E731
    out, held = [], 0
    for tok in [prefix] + [forced[:, i:i + 1] for i in range(steps)]:
        n = tok.shape[1]
        start, offsets = np.full(nseq, held), np.arange(nseq + 1) * n
        at = np.tile(np.arange(held, held + n), nseq)
        x = w["embed"][tok.reshape(-1)]
        for l in range(L):
            p = {k.split(".")[-1]: v for k, v in w.items() if k.startswith(f"layers.{l}.")}
            y = norm(x, p["g_att"])
            q, k, v = ((y @ p[m].T).reshape(-1, h, 64) for m, h in (("wq", H), ("wk", KV), ("wv", KV)))
            ref.append(*pools[l], table, start, offsets, k, v, cos, sin)
            o, _ = ref.attend(*pools[l], table, start, offsets, ref.rope(q, cos[at], sin[at]), 0.125)
            x = x + o.reshape(len(x), -1) @ p["wo"].T
            y = norm(x, p["g_ffn"])
            a = y @ p["w1"].T
            x = x + (a / (1 + np.exp(-a)) * (y @ p["w3"].T)) @ p["w2"].T
        held += n
        last = norm(x.reshape(nseq, n, -1)[:, -1], w["g_final"])
        out.append(last @ w["embed"].T)
    return np.stack(out, 1)


def setup(cfg, nseq, plen, steps, seed):
    p = ane.init_params(cfg, seed=seed, std=0.05)
    r = np.random.default_rng(seed + 1)
    return (p, r.integers(0, cfg.vocab, (nseq, plen)).astype(np.uint16),
            r.integers(0, cfg.vocab, (nseq, steps)).astype(np.uint16))


def run(dec, prefix, forced):
    lg = [dec.Prefill(prefix, want_logits=True)[1]]
    for i in range(forced.shape[1]):
        lg.append(dec.Step(forced[:, i], want_logits=True)[1])
    return np.stack(lg, 1)


@pytest.mark.parametrize("tail", ["2", "1", "0"])
@pytest.mark.parametrize("page,heads,kv_heads", [(64, 4, 2), (16, 6, 2), (256, 4, 4)])
def test_8_bit_cache_matches_64_bits(page, heads, kv_heads, tail, monkeypatch):
    monkeypatch.setenv("ANE_DEC_TAIL", tail)
    cfg = ane.tiny_decode(heads=heads, kv_heads=kv_heads, dim=64 * heads)
    p, prefix, forced = setup(cfg, 3, 64, 4, 11)
    want = model_in_64_bits(cfg, p, prefix, forced, page)
    dec = ane.Decoder(cfg, p, max_batch=4, max_ctx=100, page_tokens=page)
    try:
        dec.DebugFillCache(0xFF)      # NaN everywhere: nothing unwritten is read
        check(run(dec, prefix, forced), want)
        # greedy: generated steps are the single steps
        t0, _ = dec.Prefill(prefix)
        one = [dec.Step()[0] for _ in range(6)]
        dec.Prefill(prefix)
        np.testing.assert_array_equal(dec.Generate(6), np.stack(one, 1))
    finally:
        dec.Close()


def test_many_sequences_and_a_long_context():
    """A batch that takes several prefill chunks, and a context past one part
    of the attention: as near to the fp16 cache's logits as the codes allow.  A
    value is off by 9 % / sqrt(12) = 2.6 % rms; a layer-1 output, through keys
    and values, by 3.6 %; layer 2's inputs by 3.6 % and its cache by 4.4 %, its
    output by 6.3 %: 6 % of a logit at most, rms, 8 % allowed; the largest of
    160,000 is 4.7 times 6 %, 0.3 with logits of standard deviation up to 1."""
    cfg = ane.tiny_decode()
    for nseq, plen, ctx in ((40, 256, 320), (2, 4096, 4200)):
        p, prefix, forced = setup(cfg, nseq, plen, 3, 21)
        got = []
        for page in (0, 64):
            dec = ane.Decoder(cfg, p, max_batch=nseq, max_ctx=ctx, page_tokens=page)
            try:
                got.append(run(dec, prefix, forced))
            finally:
                dec.Close()
        d = np.abs(got[0] - got[1])
        print("logits: largest difference", d.max(), "rms", np.sqrt((d ** 2).mean()), "of", got[0].std())
        assert np.isfinite(got[1]).all()
        assert d.max() <= 0.3 and np.sqrt((d ** 2).mean()) <= 0.08 * got[0].std()


@pytest.mark.parametrize("nseq,page,heads,kv_heads", [(1, 16, 4, 2), (3, 64, 6, 2), (20, 32, 4, 4), (5, 256, 8, 2)])
def test_steps_in_one_launch_a_layer_and_in_two_are_the_same_bits(nseq, page, heads, kv_heads):
    """Contexts of up to 1280 tokens have the append in the attention's launch;
    room for more does not, and up to 128 tokens its keys are one part all the
    same."""
    cfg = ane.tiny_decode(heads=heads, kv_heads=kv_heads, dim=64 * heads)
    p, prefix, forced = setup(cfg, nseq, 64, 60, 61)
    got = []
    for ctx in (192, 1344):
        dec = ane.Decoder(cfg, p, max_batch=nseq, max_ctx=ctx, page_tokens=page)
        try:
            dec.DebugFillCache(0xFF)
            got.append(run(dec, prefix, forced))
        finally:
            dec.Close()
    np.testing.assert_array_equal(got[0].view(np.uint32), got[1].view(np.uint32))


def test_switching_the_cache():
    """8 bit and back: as if never switched; the batch is dropped."""
    cfg = ane.tiny_decode()
    p, prefix, forced = setup(cfg, 2, 64, 2, 31)
    a = ane.Decoder(cfg, p, max_batch=2, max_ctx=128)
    b = ane.Decoder(cfg, p, max_batch=2, max_ctx=128, page_tokens=32)
    try:
        want = run(a, prefix, forced)
        first = run(b, prefix, forced)
        b.SetCache(0)
        with pytest.raises(ane.EngineError, match="no prefill"):
            b._check(b._lib.ane_decode_step(b._h, None, None, None))
        np.testing.assert_array_equal(run(b, prefix, forced), want)
        b.SetCache(32)
        np.testing.assert_array_equal(run(b, prefix, forced), first)
        for bad in (8, 48, 512, -16):
            with pytest.raises(ane.EngineError, match="page_tokens"):
                b.SetCache(bad)
    finally:
        a.Close()
        b.Close()


def test_failed_chain_wait_leaves_the_8_bit_cache_whole(monkeypatch):
    """Every wait of the chain times out: the call is redone with one launch
    per GEMM, and nothing of the failed attempt's rows stays in the cache."""
    cfg = ane.tiny_decode()
    p, prefix, forced = setup(cfg, 3, 64, 4, 41)
    want = model_in_64_bits(cfg, p, prefix, forced, 64)
    monkeypatch.setenv("ANE_DEC_TAIL_SPIN", "0")
    dec = ane.Decoder(cfg, p, max_batch=3, max_ctx=128, page_tokens=64)
    try:
        got = run(dec, prefix, forced)
        assert dec.FusedChain() == 2
        check(got, want)
    finally:
        dec.Close()


def controls(r, cfg, B, mask_rows):
    words = (cfg.vocab + 31) // 32
    m = r.integers(0, 2**32, (mask_rows, words), dtype=np.uint64).astype(np.uint32)
    m |= r.integers(0, 2**32, (mask_rows, words), dtype=np.uint64).astype(np.uint32)
    return dict(repetition=r.uniform(1.0, 1.8, B).astype(np.float32), frequency=r.uniform(0, 0.4, B).astype(np.float32),
                presence=r.uniform(0, 0.4, B).astype(np.float32),
                bias=(r.standard_normal(cfg.vocab) * (r.random(cfg.vocab) < 0.05)).astype(np.float32),
                mask=m if mask_rows > 1 else m[0])


@pytest.mark.parametrize("tail,page", [("2", 0), ("0", 0), ("2", 32)])
@pytest.mark.parametrize("use", [("repetition",), ("frequency", "presence"), ("bias", "mask"),
                                 ("repetition", "frequency", "presence", "bias", "mask")])
def test_controls_on_prefill_step_and_generate(use, tail, page, monkeypatch):
    monkeypatch.setenv("ANE_DEC_TAIL", tail)
    cfg = ane.tiny_decode()
    B, nseq, plen, steps = 4, 3, 64, 6
    p, prefix, _ = setup(cfg, nseq, plen, steps, 51)
    prefix = (prefix % 50).astype(np.uint16)       # words that come again
    r = np.random.default_rng(52)
    c = {k: v for k, v in controls(r, cfg, B, nseq).items() if k in use}
    full = {k: c.get(k) for k in ("repetition", "frequency", "presence", "bias", "mask")}
    raw = ane.Decoder(cfg, p, max_batch=B, max_ctx=128, page_tokens=page)
    dec = ane.Decoder(cfg, p, max_batch=B, max_ctx=128, page_tokens=page)
    try:
        dec.SetControls(**c)
        hist = np.zeros((nseq, 128), np.uint16)
        hist[:, :plen] = prefix
        n = np.full(nseq, plen, np.int32)
        count = any(k in use for k in ("repetition", "frequency", "presence"))
        toks = []
        feed = None
        for i in range(steps + 1):
            if i == 0:
                tok, lg = dec.Prefill(prefix, want_logits=True)
                _, rl = raw.Prefill(prefix, want_logits=True)
            else:
                hist[np.arange(nseq), n] = feed
                n += 1
                tok, lg = dec.Step(None if i % 2 else feed, want_logits=True)
                _, rl = raw.Step(feed, want_logits=True)
            cut = {k: (v if v is None or k in ("bias", "mask") else v[:nseq]) for k, v in full.items()}
            want, wt = ref.control(rl, hist if count else None, n, np.full(nseq, plen), cut["repetition"],
                                   cut["frequency"], cut["presence"], cut["bias"], cut["mask"])
            np.testing.assert_array_equal(lg.view(np.uint32), want.view(np.uint32))
            np.testing.assert_array_equal(tok, wt.astype(np.uint16))
            toks.append(tok)
            feed = tok
        dec.Prefill(prefix)
        np.testing.assert_array_equal(dec.Generate(steps), np.stack(toks[1:], 1))
        # without them again: the plain argmax
        dec.ClearControls()
        a, b = dec.Prefill(prefix)[0], raw.Prefill(prefix)[0]
        np.testing.assert_array_equal(a, b)
        np.testing.assert_array_equal(dec.Generate(4), raw.Generate(4))
    finally:
        raw.Close()
        dec.Close()


def test_mask_of_each_step_and_a_row_that_allows_nothing():
    cfg = ane.tiny_decode()
    p, prefix, _ = setup(cfg, 2, 64, 3, 61)
    words = (cfg.vocab + 31) // 32
    dec = ane.Decoder(cfg, p, max_batch=3, max_ctx=128)
    try:
        dec.SetControls(mask=np.full(words, 0xffffffff, np.uint32))
        dec.Prefill(prefix)
        for want in ([5, 700], [33, 64], [ane.NO_TOKEN, 1023]):
            m = np.zeros((2, words), np.uint32)
            for b, t in enumerate(want):
                if t < cfg.vocab:
                    m[b, t // 32] = np.uint32(1) << np.uint32(t % 32)
            dec.SetControls(mask=m)
            tok, lg = dec.Step(want_logits=True)
            assert tok.tolist() == want
        tok, lg = dec.Step(want_logits=True)    # the sequence without a token is fed the zero embedding
        assert not np.isnan(lg).any()
    finally:
        dec.Close()


def test_control_refusals():
    cfg = ane.tiny_decode()
    p, prefix, _ = setup(cfg, 2, 64, 1, 71)
    words = (cfg.vocab + 31) // 32
    dec = ane.Decoder(cfg, p, max_batch=3, max_ctx=128)
    try:
        def bad(word, **kw):
            with pytest.raises(ane.EngineError, match=word):
                dec.SetControls(**kw)
        bad("repetition has shape", repetition=np.ones(2, np.float32))
        bad("bias has shape", bias=np.ones(cfg.vocab + 1, np.float32))
        bad("want 32-bit words", mask=np.ones(words + 1, np.uint32))
        bad("want 32-bit words", mask=np.ones(words, np.float32))
        bad("mask_rows=4", mask=np.ones((4, words), np.uint32))
        dec.Prefill(prefix)
        bad("before Prefill", repetition=np.ones(3, np.float32))
        dec.SetCache(16)                       # drops the batch
        dec.SetControls(mask=np.full((2, words), 0xffffffff, np.uint32))
        dec.Prefill(prefix)
        with pytest.raises(ane.EngineError, match="mask has 2 rows"):
            dec.Prefill(np.zeros((3, 64), np.uint16))
        rc = dec._lib.ane_decode_set_controls(dec._h, _lib.DecodeControls(mask_rows=1))
        assert rc == _lib.ANE_ERR_ARG
    finally:
        dec.Close()
