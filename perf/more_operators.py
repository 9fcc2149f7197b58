"""Operators of beam search and of long contexts over the paged 8-bit cache, as cases that can be timed and compared:
the choice of the next beams over beams and vocabulary; the tables of the cache's pages (forking with copy on write,
reserving and freeing, compacting, copying); and attention over the pages that a bound on their keys selects.

Where `own` is false, `run` computes an operator with elementary torch operations in fp32 (64 bits where choices lie
close to each other); where it is true, it makes the calls that a serving program makes of this framework.  `exact` is
the definition in 64 bits.

The cache is that of `operators.py`: pages of P tokens, e4m3 codes with one exponent for each page and key/value head;
K is [pages, kv_heads, P, head_dim], V [pages, kv_heads, P/16, 4, 16, head_dim/16, 4].
"""
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
NO_TOKEN = 65535
B_MIN = -30  # smallest exponent of a bound's unit


def listed():
    return [
        # One user's beams over the classifier's vocabulary: latency.
        _beam("beam_one", requests=1, beams=4, vocab=32000, history=300),
        # The decoder's full batch of 64 rows as 16 users' beams, behind a grammar's mask.
        _beam("beam_step_b64", requests=16, beams=4, vocab=32000, history=1100, masked=0.75),
        # Many users, wide beams, a large odd vocabulary held in fp16: the logits' bytes count.
        _beam("beam_many_fp16", requests=40, beams=16, vocab=60011, history=2500, half=True),
        # One user's beams move on by a token: latency of the table and of what is copied on write.
        _fork("fork_one", requests=1, beams=4, ctx=(200, 200), layers=12),
        # Many users' wide beams, long ragged contexts.
        _fork("fork_many", requests=48, beams=8, ctx=(900, 8000), layers=6),
        # A small pool, half of it free in between.
        _pool("compact_small", "compact", nseq=8, ctx=(100, 700), layers=2, fill=0.5),
        # The pool of a busy server, brought together so that its end can be given back.
        _pool("compact_pool", "compact", nseq=64, ctx=(500, 4000), layers=12, fill=0.7),
        # One sequence's pages into another pool of the same model (a user moves to another batch).
        _pool("copy_one", "copy", nseq=1, ctx=(777, 777), layers=12, fill=0.9),
        # A whole batch's, with wide heads and small pages.
        _pool("copy_batch_d128", "copy", nseq=24, ctx=(300, 5000), layers=8, fill=0.8, kv_heads=2, head_dim=128,
              page=16),
        # One user's next token behind a long context: a few pages of it are attended to.
        _sparse("sparse_one", nseq=1, ctx=(20000, 20000), new=(1, 1), count=32),
        # A decoding step of a full batch, ragged long contexts, wide heads.
        _sparse("sparse_step_b64", nseq=64, ctx=(3500, 24000), new=(1, 1), count=48, heads=16, kv_heads=2,
                head_dim=128, page=32),
        # Chunks of prompts, each token with its own choice of pages.
        _sparse("sparse_chunks", nseq=5, ctx=(2000, 12000), new=(50, 333), count=24),
    ]


def _beam(name, requests, beams, vocab, history, masked=0.0, half=False, mix=4):
    return dict(name=name, kind="beam", requests=requests, beams=beams, vocab=vocab, history=history, masked=masked,
                half=half, mix=mix)


def _fork(name, requests, beams, ctx, layers, kv_heads=4, head_dim=64, page=64, mix=5):
    return dict(name=name, kind="fork", requests=requests, beams=beams, ctx_lo=ctx[0], ctx_hi=ctx[1], layers=layers,
                kv_heads=kv_heads, head_dim=head_dim, page=page, mix=mix)


def _pool(name, kind, nseq, ctx, layers, fill, kv_heads=4, head_dim=64, page=64, mix=6):
    return dict(name=name, kind=kind, nseq=nseq, ctx_lo=ctx[0], ctx_hi=ctx[1], layers=layers, fill=fill,
                kv_heads=kv_heads, head_dim=head_dim, page=page, mix=mix)


def _sparse(name, nseq, ctx, new, count, heads=12, kv_heads=4, head_dim=64, page=64, first=1, recent=2, mix=7):
    return dict(name=name, kind="sparse", nseq=nseq, ctx_lo=ctx[0], ctx_hi=ctx[1], new_lo=new[0], new_hi=new[1],
                count=count, first=first, recent=recent, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page,
                mix=mix)


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    mix = rng.randrange(1 << 30)
    kind = rng.choice(["beam", "beam", "fork", "compact", "copy", "sparse", "sparse"])
    if kind == "beam":
        beams, vocab, half = rng.choice([1, 2, 3, 4, 5, 8, 16, 32]), _log(rng, 500, 60011), rng.random() < 0.5
        # the bytes of the logits stay within the largest listed case's
        requests = _log(rng, 1, max(1, min(64, (38_000_000 if half else 19_000_000) // (beams * vocab))))
        c = _beam("", requests, beams, vocab, _log(rng, 1, 2500), rng.choice([0.0, 0.0, 0.75, 0.99]), half, mix)
    else:
        page = rng.choice([16, 32, 64, 128])
        kv_heads, head_dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 128])
        token = 2 * kv_heads * head_dim  # bytes of a token in a layer
        if kind == "sparse":
            group = rng.choice([1, 2, 3, 4, 6, 8, 16])
            count = _log(rng, 4, 64)
            # the keys that are attended to, the products and the pool stay within the largest listed cases
            rows = max(1, 4_100_000_000 // (count * page * group * kv_heads * head_dim * 4))
            nseq = _log(rng, 1, max(1, min(64, rows, 60_000_000 // (count * page * token))))
            hi = 1 if rng.random() < 0.5 else _log(rng, 1, max(1, min(400, rows // nseq)))
            top = _log(rng, 1, max(2, min(40000, 250_000_000 // (nseq * token))))
            c = _sparse("", nseq, (rng.randrange(top // 2 + 1), top), (max(1, hi // 5), hi), count,
                        group * kv_heads, kv_heads, head_dim, page, rng.randrange(3), rng.randint(1, 2), mix)
        else:
            layers = _log(rng, 1, 12)
            if kind == "fork":
                beams = rng.choice([1, 2, 4, 5, 8])
                requests = _log(rng, 1, max(1, min(48, 60_000_000 // (beams * page * token * layers))))
                held = max(64, 600_000_000 // (layers * token * requests) - 2 * page * beams)
                top = _log(rng, 1, min(8000, held))
                c = _fork("", requests, beams, (max(1, top // 8), top), layers, kv_heads, head_dim, page, mix)
            else:
                nseq = _log(rng, 1, 64)
                top = _log(rng, 1, max(2, min(5000, 400_000_000 // (layers * token * nseq))))
                c = _pool("", kind, nseq, (max(1, top // 8), top), layers, rng.uniform(0.3, 0.95), kv_heads, head_dim,
                          page, mix)
    del c["name"]
    return c


def _lengths(case):
    """Tokens held before and new ones, of each sequence (of each request's beams)."""
    rng = random.Random(case["mix"])
    n = case["requests"] if case["kind"] == "fork" else case["nseq"]
    new = (case["new_lo"], case["new_hi"]) if case["kind"] == "sparse" else (1, 1)
    return [(rng.randint(case["ctx_lo"], case["ctx_hi"]), rng.randint(*new)) for _ in range(n)]


def _up(n, m):
    return (n + m - 1) // m


def work(case):
    if case["kind"] == "beam":
        n, v = case["requests"] * case["beams"], case["vocab"]
        # the logits once; the histories of the beams that change places (at most all), read and written
        return {"bytes": n * v * (2 if case["half"] else 4) + n * (2 * 2 * case["history"] + 40), "flops": 4 * n * v}
    kvh, dh, page = case["kv_heads"], case["head_dim"], case["page"]
    lens = _lengths(case)
    if case["kind"] == "sparse":
        h, rows = case["heads"], sum(n for _, n in lens)
        pairs = pages = scored = touched = union = 0
        for s, n in lens:
            touched += (s + n - 1) // page - s // page + 1
            scored += _up(s + n, page)  # bounds of the sequence's pages
            for p in range(s, s + n):
                seen = min(case["count"], p // page + 1)
                pages += p // page + 1
                pairs += seen * page if seen <= p // page else p + 1
            # what is attended to, once: no more than the sequence, no less than one token's choice
            union += min(s + n, case["count"] * page)
        return {"bytes": rows * h * dh * 4 + rows * kvh * case["count"] * 4 + union * kvh * dh * 2
                + (scored + touched) * kvh * (2 * dh + 1) + touched * kvh * page * dh,
                "flops": 4 * h * dh * pairs + 2 * 2 * h * dh * pages}
    unit = 2 * kvh * dh  # bytes of a token in a layer
    if case["kind"] == "fork":
        # each beam's part of its last page into a page of its own (but one), the rows of the table
        tokens = sum((case["beams"] - 1) * (s % page) for s, _ in lens)
        entries = sum(case["beams"] * _up(s, page) for s, _ in lens)
        return {"bytes": tokens * unit * case["layers"] * 2 + entries * 8 + _pages_of(case) * 4, "flops": 0}
    held = sum(_up(s, page) for s, _ in lens)
    if case["kind"] == "copy":
        return {"bytes": sum(s for s, _ in lens) * unit * case["layers"] * 2, "flops": 0}
    pages = _pages_of(case)
    moved = held * (pages - held) // pages  # of pages in no order, those behind the place where they will end
    return {"bytes": moved * unit * page * case["layers"] * 2 + pages * 8 + held * 8, "flops": 0}


def _pages_of(case):
    page, lens = case["page"], _lengths(case)
    if case["kind"] == "fork":
        used = sum(s // page + 2 * case["beams"] for s, _ in lens)
        return used + used // 4 + 8
    held = sum(_up(s, page) for s, _ in lens)
    return max(held + 1, int(held / case.get("fill", 0.95)) + 1)


# ---- inputs ----------------------------------------------------------------------------------------------------------


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return {"beam": _prepare_beam, "fork": _prepare_fork, "compact": _prepare_pool, "copy": _prepare_pool,
            "sparse": _prepare_sparse}[case["kind"]](case, g)


def _prepare_beam(case, g):
    r, w, v, hist = (case[k] for k in ("requests", "beams", "vocab", "history"))
    n = r * w
    x = torch.randn((n, v), device=DEV, generator=g) * 3
    if case["masked"]:
        x.masked_fill_(torch.rand((n, v), device=DEV, generator=g) < case["masked"], float("-inf"))
    finished = torch.rand(n, device=DEV, generator=g) < 0.15
    lengths = torch.full((n,), hist, device=DEV, dtype=torch.int32)
    lengths -= (finished * (torch.rand(n, device=DEV, generator=g) * min(hist, 30)).int()).int()
    ids = (torch.rand((n, hist + 64), device=DEV, generator=g).pow_(3) * v).to(torch.int32).clamp_(max=v - 1)
    s = dict(case=case, logits=x.half() if case["half"] else x, eos=2 % v, finished=finished, lengths=lengths,
             # sums of log probabilities, the best beam first
             scores=-torch.sort(20 + 1.5 * torch.randn((r, w), device=DEV, generator=g), 1)[0].flatten().contiguous(),
             # longer hypotheses are not worse for being longer
             weights=lengths.float().clamp(min=1).pow(-0.6),
             history=torch.where(ids < 32768, ids, ids - 65536).to(torch.int16).contiguous(),
             scores_out=torch.zeros(n, device=DEV), finished_out=torch.zeros(n, device=DEV, dtype=torch.bool),
             tokens=torch.zeros(n, device=DEV, dtype=torch.int32), parents=torch.zeros(n, device=DEV, dtype=torch.int32))
    if own:
        s["search"] = _package().BeamSearch(v, w, eos=s["eos"])
    return s


def _codes(g, *shape):
    """e4m3 codes of what earlier calls left (none of them NaN)."""
    x = torch.randint(0, 254, shape, device=DEV, generator=g, dtype=torch.uint8)
    return torch.where(x < 127, x, x + 1).view(torch.float8_e4m3fn)


def _layers(case, pages, g, count):
    kvh, dh, page = case["kv_heads"], case["head_dim"], case["page"]
    return [dict(k=_codes(g, pages, kvh, page, dh), v=_codes(g, pages, kvh, page // 16, 4, 16, dh // 16, 4),
                 k_exp=torch.randint(-15, 9, (pages, kvh), device=DEV, generator=g, dtype=torch.int8),
                 v_exp=torch.randint(-15, 9, (pages, kvh), device=DEV, generator=g, dtype=torch.int8))
            for _ in range(count)]


def _caches(layers):
    ane = _package()
    return [ane.KVCache8(x["k"], x["v"], x["k_exp"], x["v_exp"]) for x in layers]


def _prepare_fork(case, g):
    r, w, page = case["requests"], case["beams"], case["page"]
    lens = [s for s, _ in _lengths(case)]
    pages = _pages_of(case)
    order = torch.randperm(pages, device=DEV, generator=g).to(torch.int32).tolist()
    width = max(_up(s + 1, page) for s in lens) + 1
    table, at = [], 0
    for s in lens:
        held = _up(s, page)
        alone = min(held, 2)  # a beam's own last pages; those before are the request's
        shared = order[at:at + held - alone]
        at += held - alone
        for _ in range(w):
            mine = order[at:at + alone]
            at += alone
            table.append(shared + mine + [-1] * (width - held))
    s = dict(case=case, table=torch.tensor(table, device=DEV, dtype=torch.int32),
             layers=_layers(case, pages, g, case["layers"]),
             start=torch.tensor([x for x in lens for _ in range(w)], device=DEV, dtype=torch.int32))
    s["refs"] = torch.bincount(s["table"][s["table"] >= 0].long(), minlength=pages).to(torch.int32)
    # most of the next beams come from a request's best ones
    best = (torch.rand((r, w), device=DEV, generator=g).square() * w).int().clamp(max=w - 1)
    s["parents"] = (best + torch.arange(r, device=DEV, dtype=torch.int32)[:, None] * w).flatten().int().contiguous()
    if own:
        s["pages"] = _package().KVPages(_caches(s["layers"]), s["refs"])
    return s


def _prepare_pool(case, g):
    page = case["page"]
    lens = [s for s, _ in _lengths(case)]
    pages = _pages_of(case)
    order = torch.randperm(pages, device=DEV, generator=g).to(torch.int32).tolist()
    width = max(_up(s, page) for s in lens) + 1
    table, at = [], 0
    for s in lens:
        held = _up(s, page)
        table.append(order[at:at + held] + [-1] * (width - held))
        at += held
    s = dict(case=case, layers=_layers(case, pages, g, case["layers"]))
    if case["kind"] == "copy":
        other = max(at, pages // 2) + 5
        s["into"] = _layers(case, other, g, case["layers"])
        s["src"] = torch.tensor(order[:at], device=DEV, dtype=torch.int32)
        s["dst"] = torch.randperm(other, device=DEV, generator=g)[:at].to(torch.int32)
        s["tokens"] = torch.tensor([min(page, n - j) for n in lens for j in range(0, n, page)], device=DEV,
                                   dtype=torch.int32)
        refs = torch.zeros(pages, device=DEV, dtype=torch.int32)
        refs[s["src"].long()] = 1
    else:
        t = torch.tensor(table, device=DEV, dtype=torch.int32)
        refs = torch.bincount(t[t >= 0].long(), minlength=pages).to(torch.int32)
        # A pass compacts the pool as it was: by the time a server does it again, its pages lie about again.
        s["before"] = torch.cat([refs, t.flatten()])
        s["book"] = s["before"].clone()
        refs, s["table"] = s["book"][:pages], s["book"][pages:].view(t.shape)
    s["refs"] = refs
    if own:
        ane = _package()
        s["pages"] = ane.KVPages(_caches(s["layers"]), refs)
        if case["kind"] == "copy":
            s["target"] = ane.KVPages(_caches(s["into"]), torch.zeros(other, device=DEV, dtype=torch.int32))
    return s


def _prepare_sparse(case, g):
    h, kvh, dh, page, nseq = (case[k] for k in ("heads", "kv_heads", "head_dim", "page", "nseq"))
    lens = _lengths(case)
    rows, total = sum(n for _, n in lens), [s + n for s, n in lens]
    held = [_up(t, page) for t in total]
    pages = sum(held) + 3
    order = torch.randperm(pages, device=DEV, generator=g).to(torch.int32)
    width = max(held) + 1
    at = [[sum(held[:i]) + min(j, held[i] - 1) for j in range(width)] for i in range(nseq)]
    offsets = [0]
    for _, n in lens:
        offsets.append(offsets[-1] + n)
    s = dict(case=case, table=order[torch.tensor(at, device=DEV)].contiguous(), rows=rows, max_len=max(total),
             start=torch.tensor([a for a, _ in lens], device=DEV, dtype=torch.int32), max_new=max(n for _, n in lens),
             offsets=torch.tensor(offsets, device=DEV, dtype=torch.int32))
    # Keys of a page lie near each other, and the query near those of some pages.
    for name, shape in (("k", (pages, kvh, page, dh)), ("v", (pages, kvh, page // 16, 4, 16, dh // 16, 4))):
        x = torch.empty(shape, device=DEV, dtype=torch.uint8)
        for a in range(0, pages, 4096):
            b = min(pages, a + 4096)
            y = torch.randn((b - a, *shape[1:]), device=DEV, generator=g).mul_(50.0)
            if name == "k":
                y += 40.0 * torch.randn((b - a, kvh, 1, dh), device=DEV, generator=g)
            x[a:b] = y.clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        s[name] = x.view(torch.float8_e4m3fn)
    s["k_exp"] = torch.randint(-7, -4, (pages, kvh), device=DEV, generator=g).to(torch.int8)
    s["v_exp"] = torch.randint(-8, -5, (pages, kvh), device=DEV, generator=g).to(torch.int8)
    s["q"] = torch.randn((rows, h, dh), device=DEV, generator=g).half()
    s["out"] = torch.zeros((rows, h, dh), device=DEV, dtype=torch.half)
    # the bounds that the steps before left, of all pages
    s["bounds"] = torch.zeros((pages, kvh, 2, dh), device=DEV, dtype=torch.int8)
    s["unit"] = torch.zeros((pages, kvh), device=DEV, dtype=torch.int8)
    ids = torch.arange(pages, device=DEV)
    for a in range(0, pages, 4096):
        _bound_plain(s, ids[a:a + 4096], torch.full_like(ids[a:a + 4096], page))
    if own:
        ane = _package()
        s["cache"] = ane.KVCache8(s["k"], s["v"], s["k_exp"], s["v_exp"])
        s["batch"] = ane.KVBatch(s["table"], s["start"], s["offsets"], rows, max_len=s["max_len"], max_new=s["max_new"])
        s["keys"] = ane.KVBounds(s["cache"], s["bounds"], s["unit"])
    return s


def _package():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "autoresearch-go-ane_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import ane
    return ane


# ---- the framework's calls -------------------------------------------------------------------------------------------


def run(s):
    kind = s["case"]["kind"]
    if kind == "beam":
        (_beam_own if own else _beam_plain)(s)
        return {k: s[k] for k in ("tokens", "parents", "history", "lengths")} | {
            "scores": s["scores_out"], "finished": s["finished_out"]}
    if kind == "sparse":
        blocks = (_sparse_own if own else _sparse_plain)(s)
        return {"out": s["out"], "blocks": blocks, "bounds": s["bounds"], "unit": s["unit"]}
    if kind == "copy":
        if own:
            s["pages"].Copy(s["src"], s["dst"], tokens=s["tokens"], into=s["target"])
        else:
            _copy_pages(s["layers"], s["into"], s["src"].long(), s["dst"].long(), s["tokens"].long())
        return {"into": s["into"]}
    if kind == "compact":
        s["book"].copy_(s["before"])
        moved = s["pages"].Compact(s["table"]) if own else _compact_plain(s)
        return {"moved": moved, "table": s["table"], "refs": s["refs"], "layers": s["layers"]}
    if own:
        missing = s["pages"].Fork(s["table"], s["start"], parents=s["parents"], new=1)
    else:
        missing = _fork_plain(s)
    return {"missing": missing, "table": s["table"], "start": s["start"], "refs": s["refs"], "layers": s["layers"]}


def _beam_own(s):
    s["search"].Select(s["logits"], s["scores"], finished=s["finished"], weights=s["weights"], history=s["history"],
                       lengths=s["lengths"], tokens=s["tokens"], parents=s["parents"], scores_out=s["scores_out"],
                       finished_out=s["finished_out"])


def _sparse_own(s):
    c = s["case"]
    s["keys"].Update(s["batch"])
    blocks = s["keys"].Select(s["batch"], s["q"], c["count"], first=c["first"], recent=c["recent"])
    s["cache"].Attend(s["batch"], s["q"], s["out"], blocks=blocks)
    return blocks


# ---- plain forms -----------------------------------------------------------------------------------------------------


def _beam_plain(s):
    c = s["case"]
    r, w, v = c["requests"], c["beams"], c["vocab"]
    x = s["logits"].float()
    x = torch.where(torch.isnan(x), float("-inf"), x) + 0.0
    top = x.amax(-1, keepdim=True)
    # candidates lie close to each other: the sums that order them in 64 bits
    lse = top.double() + torch.log(torch.exp((x - top).double()).sum(-1, keepdim=True))
    bits = x.view(torch.int32)
    bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    k = min(w, v)
    at = torch.topk((bits << 32) | (v - 1 - torch.arange(v, device=DEV)), k, dim=-1)[0]
    at = v - 1 - (at & 0xFFFFFFFF)  # a row's best tokens, ties to the lower one
    score = s["scores"].double()[:, None] + (x.gather(1, at).double() - lse)
    first = torch.arange(k, device=DEV)[None] == 0
    done = s["finished"][:, None]
    score = torch.where(done, torch.where(first, s["scores"].double()[:, None], float("-inf")), score)
    at = torch.where(done & first, s["eos"], at)
    key = torch.nan_to_num(score * s["weights"].double()[:, None], nan=float("-inf"), posinf=float("inf"),
                           neginf=float("-inf"))
    key = torch.where(s["weights"][:, None] > 0, key, float("-inf"))
    flat = (torch.arange(r * w, device=DEV)[:, None] % w * v + at).reshape(r, w * k)
    key, score = key.reshape(r, w * k), score.reshape(r, w * k)
    by = torch.sort(flat, 1)[1]
    by = by.gather(1, torch.sort(key.gather(1, by), dim=1, descending=True, stable=True)[1])[:, :w]
    there = key.gather(1, by) > float("-inf")
    flat, score = flat.gather(1, by), score.gather(1, by)
    token = torch.where(there, flat % v, NO_TOKEN).flatten()
    beam = (flat // v + torch.arange(r, device=DEV)[:, None] * w).flatten()
    there = there.flatten()
    s["scores_out"].copy_(torch.where(there, score.flatten(), float("-inf")))
    s["tokens"].copy_(token)
    s["parents"].copy_(torch.where(there, beam, -1))
    done = s["finished"][beam]
    s["finished_out"].copy_(there & (done | (token == s["eos"])))
    # the histories move with their beams, and get the token
    most = s["history"].shape[1]
    was = s["lengths"].long()[beam]
    grows = there & ~done & (was < most)
    j = torch.arange(most, device=DEV)[None]
    ids = torch.where(token < 32768, token, token - 65536).to(torch.int16)
    moved = torch.where(j < was[:, None], s["history"][beam], s["history"])
    moved = torch.where(grows[:, None] & (j == was[:, None]), ids[:, None], moved)
    s["history"].copy_(torch.where(there[:, None], moved, s["history"]))
    s["lengths"].copy_(torch.where(there, was + grows, 0))


def _copy_pages(src, dst, a, b, tokens):
    """Pages a[i] of src to pages b[i] of dst: the 16-token units that hold the first tokens[i]."""
    kvh, page = src[0]["k"].shape[1:3]
    unit = torch.arange(page // 16, device=DEV)[None] < (tokens[:, None] + 15) // 16
    for x, y in zip(src, dst):
        for name in ("k", "v"):
            shape = (-1, kvh, page // 16, 16 * x["k"].shape[3])
            p, q = x[name].view(torch.uint8).reshape(shape), y[name].view(torch.uint8).view(shape)
            q[b] = torch.where(unit[:, None, :, None], p[a], q[b])
            y[name + "_exp"][b] = x[name + "_exp"][a]


def _fork_plain(s):
    page, table, refs = s["case"]["page"], s["table"], s["refs"]
    pages, (nseq, width) = refs.shape[0], table.shape
    seq, j = torch.arange(nseq, device=DEV), torch.arange(width, device=DEV)
    parent = s["parents"].long()
    lives = (parent >= 0) & (parent < nseq)
    parent = parent.clamp(0, nseq - 1)
    start = torch.where(lives, s["start"].long().clamp(0, width * page)[parent], 0)
    new = torch.ones_like(start).minimum(width * page - start)
    held = (start + page - 1) // page
    old = torch.where((table >= 0) & (table < pages), table.long(), -1)
    mid = torch.where(j[None] < held[:, None], old[parent], -1)
    count = torch.zeros(pages + 1, device=DEV, dtype=torch.int64)  # the last for entries that name no page
    count[:pages] = refs

    def add(ids, by):
        ids = torch.where(ids < 0, pages, ids).flatten()
        return count.scatter_add_(0, ids, torch.full_like(ids, by))

    add(mid, 1)
    add(old, -1)
    # the page that the first new token goes to, where it holds tokens from before
    at = (start // page).clamp(max=width - 1)
    writes = (new > 0) & (start % page != 0)
    last = torch.where(writes, mid[seq, at], -1)
    slot = torch.where(last < 0, pages, last)
    writers = torch.zeros_like(count).scatter_add_(0, slot, torch.ones_like(slot))
    lowest = torch.full_like(count, nseq).scatter_reduce_(0, slot, seq, "amin")
    keeps = (last >= 0) & (count[slot] == writers[slot]) & (lowest[slot] == seq)
    copies = (last >= 0) & ~keeps
    add(torch.where(copies, last, -1), -1)
    fresh = (j[None] >= held[:, None]) & (j[None] * page < (start + new)[:, None])
    need = fresh | (copies[:, None] & (j[None] == at[:, None]))
    rank = need.flatten().cumsum(0).view(nseq, width) - 1
    free, ids = torch.sort((count[:pages] > 0).to(torch.uint8), stable=True)
    got = torch.where(need & (rank < (free == 0).sum()), ids[rank.clamp(0, pages - 1)], -1)
    add(got, 1)
    table.copy_(torch.where(need, got, mid))
    refs.copy_(count[:pages])
    s["start"].copy_(start)
    moves = copies & (got[seq, at] >= 0)
    _copy_pages(s["layers"], s["layers"], last[moves], got[seq, at][moves], (start % page)[moves])
    return ((need & (got < 0)).sum() + (writes & (last < 0)).sum()).to(torch.int32).reshape(1)


def _compact_plain(s):
    refs, table = s["refs"], s["table"]
    pages = refs.shape[0]
    ids = torch.arange(pages, device=DEV)
    used = refs > 0
    total = used.sum()
    goes, hole = used & (ids >= total), ~used & (ids < total)
    holes = torch.sort((~hole).to(torch.uint8), stable=True)[1]
    to = torch.where(goes, holes[(goes.cumsum(0) - 1).clamp(min=0)], ids)
    moved = torch.where(used, to, -1)
    src = ids[goes]
    dst = to[goes]
    _copy_pages(s["layers"], s["layers"], src, dst, torch.full_like(src, s["case"]["page"]))
    refs[dst] = refs[src]
    refs[src] = 0
    there = (table >= 0) & (table < pages)
    table.copy_(torch.where(there, moved[table.long().clamp(0, pages - 1)], table.long()))
    return moved.to(torch.int32)


def _unit(amax):
    """The smallest exponent from B_MIN on at which amax <= 127 * 2^e."""
    m, e = torch.frexp(amax)
    return torch.where(amax > 0, (e - 7 + (m > 0.9921875)).clamp(min=B_MIN), B_MIN)


def _bound_plain(s, ids, tokens):
    """The bounds of pages `ids`, whose first `tokens` rows hold keys."""
    k = s["k"].view(torch.uint8)[ids].view(torch.float8_e4m3fn).float()
    k = torch.ldexp(k, s["k_exp"][ids].int()[:, :, None, None])
    there = torch.arange(k.shape[2], device=DEV)[None, None, :, None] < tokens[:, None, None, None]
    there = there & ~torch.isnan(k)
    lo = torch.where(there, k, float("inf")).amin(2)
    hi = torch.where(there, k, float("-inf")).amax(2)
    none = lo > hi
    lo, hi = lo.masked_fill(none, 0.0), hi.masked_fill(none, 0.0)
    e = _unit(torch.maximum(-lo, hi).amax(-1))
    lo, hi = torch.floor(torch.ldexp(lo, -e[..., None])), torch.ceil(torch.ldexp(hi, -e[..., None]))
    s["bounds"][ids] = torch.stack([hi, lo], 2).to(torch.int8)
    s["unit"][ids] = e.to(torch.int8)


def _sparse_plain(s):
    c = s["case"]
    h, kvh, dh, page, nseq = (c[k] for k in ("heads", "kv_heads", "head_dim", "page", "nseq"))
    g, most, new, rows, width = h // kvh, s["max_len"], s["max_new"], s["rows"], s["table"].shape[1]
    start, offsets, table = s["start"].long(), s["offsets"].long(), s["table"].long()
    count = offsets[1:] - offsets[:-1]
    # the pages that the new tokens went to; a page twice gets the same bounds twice
    j = (start // page)[:, None] + torch.arange((new - 1) // page + 2, device=DEV)
    j = torch.minimum(j, ((start + count - 1) // page)[:, None])
    held = ((start + count)[:, None] - j * page).clamp(max=page)
    _bound_plain(s, table.gather(1, j).flatten(), held.flatten())

    row = torch.arange(rows, device=DEV)
    seq = torch.searchsorted(offsets, row, right=True) - 1
    pos = start[seq] + row - offsets[seq]
    # queries in whole numbers of a power of two; products and sums of whole numbers below 2^24 are exact in fp32
    q = s["q"].float().clamp(-65504, 65504)
    e = _unit(q.abs().amax(-1))
    q = torch.round(torch.ldexp(q, -e[..., None]))
    q = torch.cat([q.clamp(min=0), q.clamp(max=0)], -1).view(rows, kvh, g, 2 * dh)
    e = e.view(rows, kvh, g, 1)
    pages = (most + page - 1) // page
    blocks = torch.empty((rows, kvh, c["count"]), device=DEV, dtype=torch.int32)
    for i in range(nseq):
        a, b = (0, rows) if new == 1 else (int(s["offsets"][i]), int(s["offsets"][i + 1]))
        who = seq[a:b] if new == 1 else torch.full((b - a,), i, device=DEV)
        at = table[who if new == 1 else who[:1], :pages]
        box = s["bounds"][at].flatten(-2).float().permute(0, 2, 3, 1)  # [rows or 1, kvh, 2 dh, pages]
        x = torch.matmul(q[a:b], box.contiguous())
        x = torch.ldexp(x, e[a:b]).amax(2)
        x = torch.ldexp(x, s["unit"][at].int().transpose(1, 2))  # [rows, kvh, pages]
        p = torch.arange(pages, device=DEV)
        own_page = (pos[a:b] // page)[:, None, None]
        x = torch.where((p < c["first"]) | (p > own_page - c["recent"]), float("inf"), x + 0.0)
        bits = x.view(torch.int32)
        bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
        key = torch.where(p > own_page, -(1 << 62), (bits << 32) | (pages - 1 - p))
        n = min(c["count"], pages)
        key = torch.topk(key, n, -1)[0]
        best = torch.where(key == -(1 << 62), width, pages - 1 - (key & 0xFFFFFFFF))
        best = torch.sort(best, -1)[0]
        blocks[a:b] = -1
        blocks[a:b, :, :n] = torch.where(best == width, -1, best).int()
        if new == 1:
            break
    _attend_blocks_plain(s, blocks, seq, pos)
    return blocks


def _attend_blocks_plain(s, blocks, seq, pos):
    c = s["case"]
    h, kvh, dh, page = (c[k] for k in ("heads", "kv_heads", "head_dim", "page"))
    g, n = h // kvh, c["count"]
    some = max(1, 100_000_000 // (kvh * n * page * dh))
    head = torch.arange(kvh, device=DEV)[None, :, None]
    for a in range(0, s["rows"], some):
        b = min(s["rows"], a + some)
        r = b - a
        j = blocks[a:b].long()
        at = s["table"].long()[seq[a:b, None, None], j.clamp(min=0)]  # [rows, kvh, n]
        k = s["k"].view(torch.uint8)[at, head].view(torch.float8_e4m3fn).float()  # [rows, kvh, n, page, dh]
        k = torch.ldexp(k, s["k_exp"][at, head].int()[..., None, None]).reshape(r, kvh, n * page, dh)
        v = s["v"].view(torch.uint8)[at, head].view(torch.float8_e4m3fn).float()
        v = v.permute(0, 1, 2, 3, 4, 7, 6, 5).reshape(r, kvh, n, page, dh)
        v = torch.ldexp(v, s["v_exp"][at, head].int()[..., None, None]).reshape(r, kvh, n * page, dh)
        t = j[..., None] * page + torch.arange(page, device=DEV)
        hidden = ((t > pos[a:b, None, None, None]) | (j < 0)[..., None]).reshape(r, kvh, 1, n * page)
        x = torch.matmul(s["q"][a:b].float().view(r, kvh, g, dh) * dh ** -0.5, k.transpose(-1, -2).contiguous())
        x.masked_fill_(hidden, float("-inf"))
        x = torch.exp(x - x.amax(-1, keepdim=True))
        o = torch.matmul(x, v) / x.sum(-1, keepdim=True)
        s["out"][a:b] = o.reshape(r, h, dh)


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------


def exact(case, seed):
    if case["kind"] not in ("beam", "sparse"):
        return None  # tables and copies: nothing is computed
    s = prepare(case, seed)
    return _beam_exact(s) if case["kind"] == "beam" else _sparse_exact(s)


def _beam_exact(s):
    c = s["case"]
    w, v = c["beams"], c["vocab"]
    scores = torch.full((c["requests"] * w,), float("-inf"), device=DEV, dtype=torch.float64)
    for r in range(c["requests"]):
        found = []
        for i in range(r * w, r * w + w):
            base, weight = float(s["scores"][i]), float(s["weights"][i])
            if bool(s["finished"][i]):
                found.append((base * weight, base))
                continue
            p = torch.log_softmax(s["logits"][i].double(), -1)
            for x in torch.sort(p, descending=True)[0][:w].tolist():
                if x > float("-inf"):
                    found.append(((base + x) * weight, base + x))
        found.sort(key=lambda f: -f[0])
        for i, (_, x) in enumerate(found[:w]):
            scores[r * w + i] = x
    return {"tokens": None, "parents": None, "history": None, "lengths": None, "scores": scores, "finished": None}


def _token_rows(x):
    """V's pages [..., P/16, 4, 16, dh/16, 4] as rows [..., P, dh]."""
    return x.movedim(-1, -3).transpose(-1, -2).flatten(-2).flatten(-4, -2)


def _sparse_exact(s):
    c = s["case"]
    h, kvh, dh, page = (c[k] for k in ("heads", "kv_heads", "head_dim", "page"))
    g = h // kvh
    out = torch.zeros((s["rows"], h, dh), device=DEV, dtype=torch.float64)
    if s["rows"] * kvh > 20000:
        return None
    row = 0
    for i, (held, n) in enumerate(_lengths(c)):
        ids = s["table"][i, :_up(held + n, page)].long()
        k = s["k"].view(torch.uint8)[ids].view(torch.float8_e4m3fn).double()
        k *= torch.exp2(s["k_exp"][ids].double())[:, :, None, None]
        v = _token_rows(s["v"].view(torch.uint8)[ids].view(torch.float8_e4m3fn).double())
        v *= torch.exp2(s["v_exp"][ids].double())[:, :, None, None]
        # a page's box, in whole numbers of its unit, of the keys that are there
        t = torch.arange(ids.shape[0] * page, device=DEV).view(-1, 1, page, 1)
        lo = torch.where(t < held + n, k, math.inf).amin(2)
        hi = torch.where(t < held + n, k, -math.inf).amax(2)
        step = torch.exp2(torch.ceil(torch.log2(torch.maximum(lo.abs(), hi.abs()).amax(-1) / 127)).clamp(min=B_MIN))
        lo, hi = torch.floor(lo / step[..., None]), torch.ceil(hi / step[..., None])
        for r in range(n):
            last = (held + r) // page
            for head in range(kvh):
                q = s["q"][row + r, head * g:head * g + g].double()
                fine = torch.exp2(torch.ceil(torch.log2(q.abs().amax(-1, keepdim=True) / 127)).clamp(min=B_MIN))
                z = torch.round(q / fine)[:, None]
                x = torch.where(z > 0, z * hi[None, :last + 1, head], z * lo[None, :last + 1, head]).sum(-1)
                x = (x * fine).amax(0) * step[:last + 1, head]
                x[:c["first"]] = math.inf
                x[max(0, last + 1 - c["recent"]):] = math.inf
                best = torch.sort(x, descending=True, stable=True)[1][:c["count"]]
                kk, vv = k[best, head].flatten(0, 1), v[best, head].flatten(0, 1)
                at = (best[:, None] * page + torch.arange(page, device=DEV)).flatten()
                y = torch.where(at <= held + r, q @ kk.t().contiguous() / math.sqrt(dh), -math.inf)
                out[row + r, head * g:head * g + g] = torch.softmax(y, -1) @ vv
        row += n
    return {"out": out, "blocks": None, "bounds": None, "unit": None}
