"""The serving operators as cases that can be timed and compared: appending rotated keys and values to a paged 8-bit
cache, attention over that cache, and the controls on logits before the next token is chosen.

Where `own` is false, `run` computes an operator with elementary torch operations in fp32; where it is true, it makes
the calls that a serving program makes of this framework.  `exact` is the definition in 64 bits.

The cache: pages of P tokens, e4m3 codes with one exponent for each page and key/value head (value = code * 2^e,
e in [-15, 8]).  K is [pages, kv_heads, P, head_dim].  V keeps four tokens of a dimension side by side:
[pages, kv_heads, P/16, 4, 16, head_dim/16, 4], token s and dimension d at [s//16, s%16//4, d%16, d//16, s%4].
"""
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
E_MIN, E_MAX = -15, 8
HALF_MAX = 65504.0
NO_TOKEN = 65535


def listed():
    return [
        # One user's next token: what the shortest append costs (latency).  The decoder's model: 12 query heads over 4
        # key/value heads of 64.
        _append("append_one", nseq=1, ctx=(200, 200), new=(1, 1)),
        # One decoding step of a full batch at the decode benchmark's lengths.
        _append("append_step_b64", nseq=64, ctx=(1024, 1100), new=(1, 1)),
        # Ragged prompts behind nothing: the prefill of a batch.
        _append("append_prompts", nseq=24, ctx=(0, 0), new=(100, 1400)),
        # Odd chunks of prompts behind odd contexts, small pages, wide heads.
        _append("append_chunks_d128", nseq=7, ctx=(1, 900), new=(33, 700), heads=16, kv_heads=2, head_dim=128, page=16),
        # One user's next token over a short context: latency.
        _attend("attend_one", nseq=1, ctx=(776, 776), new=(1, 1)),
        # One decoding step of a full batch at the decode benchmark's lengths.
        _attend("attend_step_b64", nseq=64, ctx=(1024, 1100), new=(1, 1)),
        # Long ragged contexts, where the cache's bytes are all of it.
        _attend("attend_step_long", nseq=40, ctx=(2000, 40000), new=(1, 1), heads=16, kv_heads=2, head_dim=128, page=32),
        # One long prompt: the products count.
        _attend("attend_prompt", nseq=1, ctx=(0, 0), new=(8192, 8192)),
        # Chunks of prompts, a few tokens to some hundred, on contexts that are there already; eight heads a group.
        _attend("attend_chunks", nseq=9, ctx=(0, 6000), new=(2, 300), heads=32, kv_heads=4, page=16),
        # One user's logits with a grammar's mask and penalties: latency.
        _control("control_one", rows=1, vocab=32000, history=300, mask=True, bias=False),
        # A full batch's logits.
        _control("control_step_b64", rows=64, vocab=32000, history=1100, mask=True, bias=True),
        # Many rows of a large odd vocabulary, long histories.
        _control("control_many", rows=400, vocab=60011, history=8000, mask=True, bias=False),
    ]


def _append(name, nseq, ctx, new, heads=12, kv_heads=4, head_dim=64, page=64, mix=1):
    return dict(name=name, kind="append", nseq=nseq, ctx_lo=ctx[0], ctx_hi=ctx[1], new_lo=new[0], new_hi=new[1],
                heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page, mix=mix)


def _attend(name, nseq, ctx, new, heads=12, kv_heads=4, head_dim=64, page=64, mix=2):
    return dict(_append(name, nseq, ctx, new, heads, kv_heads, head_dim, page, mix), kind="attend")


def _control(name, rows, vocab, history, mask, bias, mix=3):
    return dict(name=name, kind="control", rows=rows, vocab=vocab, history=history, mask=mask, bias=bias, mix=mix)


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    mix = rng.randrange(1 << 30)
    kind = rng.choice(["append", "attend", "attend", "control"])
    if kind == "control":
        rows, vocab = _log(rng, 1, 400), _log(rng, 500, 60011)
        c = _control("", rows, vocab, _log(rng, 1, 8000), rng.random() < 0.7, rng.random() < 0.5, mix)
    else:
        kv_heads = rng.choice([1, 2, 4, 8])
        head_dim = rng.choice([64, 128])
        group = rng.choice([1, 2, 3, 4, 6, 8, 16])
        page = rng.choice([16, 32, 64, 128])
        nseq = _log(rng, 1, 64)
        # the tokens of a call and the bytes of its cache stay within the largest listed cases
        tokens = 18000 * 20 // ((group + 2) * kv_heads * head_dim // 64)
        if rng.random() < 0.5:
            lo = hi = 1
        else:
            hi = max(1, min(4000, tokens // nseq))
            hi = _log(rng, 1, hi)
            lo = max(1, hi // 5)
        if kind == "append":
            most = 2000
        else:
            most = min(40000, 400_000_000 // (nseq * 2 * kv_heads * head_dim))
            most = min(most, max(1, 25_600_000_000 // (head_dim * nseq * hi * group * kv_heads)))
        top = _log(rng, 1, max(2, most - hi))
        ctx = (rng.randrange(top // 2 + 1), top)
        c = _append("", nseq, ctx, (lo, hi), group * kv_heads, kv_heads, head_dim, page, mix)
        c["kind"] = kind
    del c["name"]
    return c


def _lengths(case):
    """Tokens held before and new ones, of each sequence."""
    rng = random.Random(case["mix"])
    return [(rng.randint(case["ctx_lo"], case["ctx_hi"]), rng.randint(case["new_lo"], case["new_hi"]))
            for _ in range(case["nseq"])]


def work(case):
    if case["kind"] == "control":
        n, v = case["rows"], case["vocab"]
        b = n * v * 8 + _history_len(case)[0] * 2 + n * 2 + (n * ((v + 31) // 32) * 4 if case["mask"] else 0)
        return {"bytes": b + (v * 4 if case["bias"] else 0), "flops": 5 * n * v}
    h, kvh, dh = case["heads"], case["kv_heads"], case["head_dim"]
    lens = _lengths(case)
    rows = sum(n for _, n in lens)
    if case["kind"] == "append":
        touched = sum((s + n - 1) // case["page"] - s // case["page"] + 1 for s, n in lens)
        return {"bytes": rows * dh * (2 * h + 2 * 2 * kvh + 2 * h + 2 * kvh) + touched * kvh * 2
                + sum(n for _, n in lens) * 4 * dh, "flops": rows * 3 * dh * (h + kvh) + rows * 2 * kvh * dh}
    held = sum(s + n for s, n in lens)
    pairs = sum(n * s + n * (n + 1) // 2 for s, n in lens)
    pages = sum((s + n + case["page"] - 1) // case["page"] for s, n in lens)
    return {"bytes": rows * h * dh * 4 + held * kvh * dh * 2 + pages * (kvh * 2 + 4), "flops": 4 * h * dh * pairs}


def _history_len(case):
    rng = random.Random(case["mix"])
    lens = [rng.randint(min(1, case["history"]), case["history"]) for _ in range(case["rows"])]
    return sum(lens), lens, [rng.randint(0, n) for n in lens]


def _codes(x):
    """fp32 -> e4m3 codes held in uint8."""
    return x.to(torch.float8_e4m3fn).view(torch.uint8)


def _rope_tables(n, dh):
    f = torch.arange(n, device=DEV, dtype=torch.float64)[:, None] / (
        10000.0 ** (torch.arange(0, dh, 2, device=DEV, dtype=torch.float64) / dh))
    return torch.cos(f).float(), torch.sin(f).float()


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    if case["kind"] == "control":
        return _prepare_control(case, g)
    h, kvh, dh, page, nseq = (case[k] for k in ("heads", "kv_heads", "head_dim", "page", "nseq"))
    lens = _lengths(case)
    rows = sum(n for _, n in lens)
    total = [s + n for s, n in lens]
    held = [(t + page - 1) // page for t in total]
    pages = sum(held) + 3
    # pages in the order in which a busy server hands them out: none
    order = torch.randperm(pages, device=DEV, generator=g).to(torch.int32)
    width = max(held) + 1
    at = [[sum(held[:i]) + min(j, held[i] - 1) for j in range(width)] for i in range(nseq)]
    table = order[torch.tensor(at, device=DEV)].contiguous()
    offsets = [0]
    for _, n in lens:
        offsets.append(offsets[-1] + n)
    s = dict(case=case, table=table, start=torch.tensor([a for a, _ in lens], device=DEV, dtype=torch.int32),
             offsets=torch.tensor(offsets, device=DEV, dtype=torch.int32), rows=rows, max_len=max(total),
             max_new=max(n for _, n in lens))
    # what earlier calls left: normal values near the top of each page's range
    def codes(*shape):
        x = torch.empty(shape, device=DEV, dtype=torch.uint8)
        for a in range(0, shape[0], 4096):  # in parts: the fp32 numbers of a whole pool are many
            b = min(shape[0], a + 4096)
            x[a:b] = _codes(torch.randn((b - a, *shape[1:]), device=DEV, generator=g).mul_(60.0).clamp_(-448, 448))
        return x

    s["k"] = codes(pages, kvh, page, dh).view(torch.float8_e4m3fn)
    s["v"] = codes(pages, kvh, page // 16, 4, 16, dh // 16, 4).view(torch.float8_e4m3fn)
    s["k_exp"] = torch.randint(-7, -4, (pages, kvh), device=DEV, generator=g).to(torch.int8)
    s["v_exp"] = torch.randint(-8, -5, (pages, kvh), device=DEV, generator=g).to(torch.int8)
    if case["kind"] == "append":
        # the packed rows of the projection, q | k | v
        qkv = torch.randn((rows, h + 2 * kvh, dh), device=DEV, generator=g)
        qkv *= torch.exp(0.5 * torch.randn((1, h + 2 * kvh, dh), device=DEV, generator=g))
        s["qkv"] = qkv.half()
        s["cos"], s["sin"] = _rope_tables(width * page, dh)
        s["q_out"] = torch.zeros((rows, h, dh), device=DEV, dtype=torch.half)
    else:
        s["q"] = torch.randn((rows, h, dh), device=DEV, generator=g).half()
        s["out"] = torch.zeros((rows, h, dh), device=DEV, dtype=torch.half)
    if own:
        # the cache object of the program, and the step's batch, which all layers share
        ane = _package()
        s["cache"] = ane.KVCache8(s["k"], s["v"], s["k_exp"], s["v_exp"])
        s["batch"] = ane.KVBatch(s["table"], s["start"], s["offsets"], rows, max_len=s["max_len"], max_new=s["max_new"])
    return s


def _prepare_control(case, g):
    n, v = case["rows"], case["vocab"]
    _, lens, prompts = _history_len(case)
    wide = max(max(lens), 1)
    # text repeats its own words: ids crowd at small ranks
    ids = (torch.rand((n, wide), device=DEV, generator=g).pow_(3) * v).to(torch.int32).clamp_(max=v - 1)
    s = dict(case=case, logits=torch.randn((n, v), device=DEV, generator=g) * 3,
             history=torch.where(ids < 32768, ids, ids - 65536).to(torch.int16).contiguous(),
             lengths=torch.tensor(lens, device=DEV, dtype=torch.int32),
             prompts=torch.tensor(prompts, device=DEV, dtype=torch.int32),
             repetition=1.0 + 0.3 * torch.rand(n, device=DEV, generator=g),
             frequency=0.2 * torch.rand(n, device=DEV, generator=g),
             presence=0.5 * torch.rand(n, device=DEV, generator=g), bias=None, mask=None,
             out=torch.empty((n, v), device=DEV), tokens=torch.zeros(n, device=DEV, dtype=torch.int32))
    if case["bias"]:
        some = torch.rand(v, device=DEV, generator=g) < 0.01
        s["bias"] = torch.where(some, 4 * torch.randn(v, device=DEV, generator=g), torch.zeros(v, device=DEV))
    if case["mask"]:
        w = (v + 31) // 32
        words = torch.randint(-2**31, 2**31, (n, w), device=DEV, generator=g, dtype=torch.int64)
        words &= torch.randint(-2**31, 2**31, (n, w), device=DEV, generator=g, dtype=torch.int64)
        s["mask"] = words.to(torch.int32)
    if own:
        # the parameters of the requests in the batch, which stay for all their steps
        s["controls"] = _package().LogitControls(v, repetition=s["repetition"], frequency=s["frequency"],
                                                 presence=s["presence"], bias=s["bias"], mask=s["mask"])
    return s


def _package():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "autoresearch-go-ane_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import ane
    return ane


def run(s):
    kind = s["case"]["kind"]
    if kind == "append":
        return _append_own(s) if own else _append_plain(s)
    if kind == "attend":
        return _attend_own(s) if own else _attend_plain(s)
    return _control_own(s) if own else _control_plain(s)


def _append_own(s):
    c = s["case"]
    q, k, v = s["qkv"].split([c["heads"], c["kv_heads"], c["kv_heads"]], 1)
    s["cache"].Append(s["batch"], q, k, v, s["cos"], s["sin"], s["q_out"])
    return {"q": s["q_out"], "k": s["k"], "v": s["v"], "k_exp": s["k_exp"], "v_exp": s["v_exp"]}


def _attend_own(s):
    s["cache"].Attend(s["batch"], s["q"], s["out"])
    return s["out"]


def _control_own(s):
    s["controls"].Apply(s["logits"], s["history"], s["lengths"], s["prompts"], out=s["out"], tokens=s["tokens"])
    return {"logits": s["out"], "tokens": s["tokens"]}


# ---- plain forms -----------------------------------------------------------------------------------------------------


def _rotate(x, cos, sin):
    e, o = x[..., 0::2], x[..., 1::2]
    return torch.stack([e * cos - o * sin, o * cos + e * sin], -1).flatten(-2)


def _exponent(amax):
    m, x = torch.frexp(amax)
    e = (x - 9 + (m > 0.875)).clamp(E_MIN, E_MAX)
    return torch.where(amax > 0, e, torch.full_like(e, E_MIN))


def _quantised(x, e):
    """Codes of x at exponents e (fp32 holds 2^-e and the products exactly)."""
    y = torch.ldexp(x, -e)
    return _codes(torch.where(e == E_MAX, y.clamp(-240, 240), y))


def _append_plain(s):
    c = s["case"]
    h, kvh, dh, page, nseq = (c[k] for k in ("heads", "kv_heads", "head_dim", "page", "nseq"))
    start, offsets, table = s["start"].long(), s["offsets"].long(), s["table"].long()
    row = torch.arange(s["rows"], device=DEV)
    seq = torch.searchsorted(offsets, row, right=True) - 1
    pos = start[seq] + row - offsets[seq]
    at, slot = table[seq, pos // page], pos % page
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    q, k, v = s["qkv"].float().split([h, kvh, kvh], 1)
    s["q_out"].copy_(_rotate(q, cos, sin))
    head, d = torch.arange(kvh, device=DEV), torch.arange(dh, device=DEV)
    fresh = torch.zeros(s["k"].shape[0], device=DEV, dtype=torch.bool)
    fresh.index_put_((at,), slot == 0, accumulate=True)
    part = table[torch.arange(nseq, device=DEV), start // page]  # the page that holds the rows just before
    kept = torch.arange(page, device=DEV)[None] < (start % page)[:, None]  # [nseq, page]
    for name, x in (("k", _rotate(k, cos, sin)), ("v", v)):
        codes, exp = s[name].view(torch.uint8), s[name + "_exp"]
        x = x.clamp(-HALF_MAX, HALF_MAX)
        amax = torch.full((codes.shape[0], kvh), -1.0, device=DEV)
        amax.index_reduce_(0, at, torch.nan_to_num(x, nan=0.0).abs().amax(-1), "amax")
        old = exp.int()
        e = _exponent(amax)
        e = torch.where(amax < 0, old, torch.where(fresh[:, None], e, torch.maximum(old, e)))
        held = s[name][part].float()
        down = (old - e)[part].reshape(nseq, kvh, *[1] * (held.dim() - 2))
        again = _codes(torch.ldexp(held, down))
        if name == "k":
            keep = kept[:, None, :, None]
        else:
            keep = kept.reshape(nseq, page // 16, 4, 1, 1, 4)[:, None]
        codes[part] = torch.where(keep, again, codes[part])
        new = _quantised(x, e[at][:, :, None])
        if name == "k":
            codes[at, :, slot] = new
        else:
            t = slot[:, None, None]
            codes[at[:, None, None], head[:, None], t // 16, t % 16 // 4, d % 16, d // 16, t % 4] = new
        exp.copy_(e)
    return {"q": s["q_out"], "k": s["k"], "v": s["v"], "k_exp": s["k_exp"], "v_exp": s["v_exp"]}


def _attend_plain(s):
    c = s["case"]
    h, kvh, dh, page, nseq = (c[k] for k in ("heads", "kv_heads", "head_dim", "page", "nseq"))
    g, most, new = h // kvh, s["max_len"], s["max_new"]
    start, offsets, table = s["start"].long(), s["offsets"].long(), s["table"].long()
    p = torch.arange(most, device=DEV)
    at, slot = table[:, p // page], p % page  # [nseq, most]
    scale = torch.ldexp(torch.ones((), device=DEV), s["k_exp"].int())[at]  # [nseq, most, kvh]
    k = s["k"].view(torch.uint8)[at, :, slot].view(torch.float8_e4m3fn).float() * scale[..., None]
    head, d = torch.arange(kvh, device=DEV), torch.arange(dh, device=DEV)
    t = slot[:, None, None]
    v = s["v"].view(torch.uint8)[at[:, :, None, None], head[:, None], t // 16, t % 16 // 4, d % 16, d // 16, t % 4]
    v = v.view(torch.float8_e4m3fn).float()
    v *= torch.ldexp(torch.ones((), device=DEV), s["v_exp"].int())[at][..., None]
    j = torch.arange(new, device=DEV)
    count = offsets[1:] - offsets[:-1]
    rows = (offsets[:-1, None] + j).clamp(max=s["rows"] - 1)  # [nseq, new]
    q = s["q"].float()[rows] * (dh ** -0.5)
    q = q.reshape(nseq, new, kvh, g, dh).permute(0, 2, 3, 1, 4).reshape(nseq, kvh, g * new, dh)
    x = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()).reshape(nseq, kvh, g, new, most)
    hidden = p[None, None] > (start[:, None] + j)[..., None]  # [nseq, new, most]
    x.masked_fill_(hidden[:, None, None], float("-inf"))
    x -= x.amax(-1, keepdim=True)
    x.exp_()
    total = x.sum(-1)
    v = v.permute(0, 2, 1, 3) * (p[None] < (start + count)[:, None])[:, None, :, None]
    o = torch.matmul(x.reshape(nseq, kvh, g * new, most), v.contiguous()).reshape(nseq, kvh, g, new, dh)
    o = (o / total[..., None]).permute(0, 3, 1, 2, 4).reshape(nseq, new, h, dh)
    row = torch.arange(s["rows"], device=DEV)
    seq = torch.searchsorted(offsets, row, right=True) - 1
    s["out"].copy_(o[seq, row - offsets[seq]])
    return s["out"]


def _control_plain(s):
    n, v = s["case"]["rows"], s["case"]["vocab"]
    ids = s["history"].long() & 0xFFFF
    j = torch.arange(ids.shape[1], device=DEV)[None]
    there = j < s["lengths"][:, None]
    said = there & (j >= s["prompts"][:, None])
    every = torch.zeros((n, v), device=DEV).scatter_add_(1, ids, there.float())
    output = torch.zeros((n, v), device=DEV).scatter_add_(1, ids, said.float())
    x, rep = s["logits"], s["repetition"][:, None]
    x = torch.where(every > 0, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][:, None] * output
    x = torch.where(output > 0, x - s["presence"][:, None], x)
    if s["bias"] is not None:
        x = x + s["bias"]
    if s["mask"] is not None:
        w = torch.arange(v, device=DEV)
        x = torch.where((s["mask"][:, w // 32] >> (w % 32)) & 1 != 0, x, float("-inf"))
    s["out"].copy_(x)
    x = torch.nan_to_num(x, nan=float("-inf"), posinf=float("inf"), neginf=float("-inf"))
    top = x.amax(-1, keepdim=True)
    first = torch.where(x == top, torch.arange(v, device=DEV), v).amin(-1)
    s["tokens"].copy_(torch.where(top[:, 0] == float("-inf"), NO_TOKEN, first))
    return {"logits": s["out"], "tokens": s["tokens"]}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------


def _near(x):
    """x (64 bits, at most 448 in magnitude) rounded to the nearest e4m3 value, ties to even; NaN stays."""
    a = x.abs()
    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
    return torch.sign(x) * torch.round(a / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _append_exact, "attend": _attend_exact, "control": _control_exact}[case["kind"]](s)


def _token_rows(x):
    """V's pages [..., P/16, 4, 16, dh/16, 4] as rows [..., P, dh]."""
    return x.movedim(-1, -3).transpose(-1, -2).flatten(-2).flatten(-4, -2)


def _append_exact(s):
    c = s["case"]
    h, kvh, dh, page = (c[k] for k in ("heads", "kv_heads", "head_dim", "page"))
    x = s["qkv"].double()
    table, k_all, v_all = s["table"].tolist(), s["k"].double(), _token_rows(s["v"].double()).clone()
    exps = {"k": s["k_exp"].clone(), "v": s["v_exp"].clone()}
    turned = []
    row = 0
    for i, (held, n) in enumerate(_lengths(c)):
        block = x[row:row + n]
        z = torch.view_as_complex(block[:, :h + kvh].reshape(n, h + kvh, dh // 2, 2).contiguous())
        w = torch.complex(s["cos"][held:held + n].double(), s["sin"][held:held + n].double())
        z = torch.view_as_real(z * w[:, None]).reshape(n, h + kvh, dh)
        turned.append(z[:, :h])
        sides = (("k", z[:, h:], k_all), ("v", block[:, h + kvh:], v_all))
        row += n
        a = held
        while a < held + n:
            b = min(held + n, (a // page + 1) * page)
            at, r = table[i][a // page], a % page
            for name, new, pool in sides:
                part = new[a - held:b - held].transpose(0, 1)  # [kvh, tokens, dh]
                top = part.abs().flatten(1).amax(1)
                e = torch.ceil(torch.log2((top / 448).clamp(min=2.0 ** E_MIN))).clamp(max=E_MAX)
                if r:
                    old = exps[name][at].double()
                    e = torch.maximum(old, e)
                    pool[at, :, :r] = _near(pool[at, :, :r] * torch.exp2(old - e)[:, None, None])
                y = part * torch.exp2(-e)[:, None, None]
                y = torch.where((e == E_MAX)[:, None, None], y.clamp(-240, 240), y)
                pool[at, :, r:r + b - a] = _near(y)
                exps[name][at] = e.to(torch.int8)
            a = b
    v = v_all.reshape(*v_all.shape[:2], page // 16, 4, 4, dh // 16, 16).permute(0, 1, 2, 3, 6, 5, 4)
    return {"q": torch.cat(turned), "k": k_all, "v": v.contiguous(), "k_exp": exps["k"], "v_exp": exps["v"]}


def _attend_exact(s):
    c = s["case"]
    h, kvh, dh, page = (c[k] for k in ("heads", "kv_heads", "head_dim", "page"))
    g = h // kvh
    out = torch.zeros((s["rows"], h, dh), device=DEV, dtype=torch.float64)
    row = 0
    for i, (held, n) in enumerate(_lengths(c)):
        ids = s["table"][i, :(held + n + page - 1) // page].long()
        for name in ("k", "v"):
            x = s[name].view(torch.uint8)[ids].view(torch.float8_e4m3fn).double()
            x = _token_rows(x) if name == "v" else x
            x = x * torch.exp2(s[name + "_exp"][ids].double())[:, :, None, None]
            x = x.transpose(1, 2).flatten(0, 1)[:held + n]  # [tokens, kvh, dh]
            k, v = (x, None) if name == "k" else (k, x)
        for a in range(0, n, 2048):
            b = min(n, a + 2048)
            seen = torch.arange(held + n, device=DEV)[None] <= held + torch.arange(a, b, device=DEV)[:, None]
            for head in range(h):
                y = s["q"][row + a:row + b, head].double() @ k[:, head // g].t().contiguous() / math.sqrt(dh)
                y = torch.softmax(torch.where(seen, y, float("-inf")), -1)
                out[row + a:row + b, head] = y @ v[:, head // g].contiguous()
        row += n
    return out


def _control_exact(s):
    v = s["case"]["vocab"]
    x = s["logits"].double()
    for r, (n, p) in enumerate(zip(s["lengths"].tolist(), s["prompts"].tolist())):
        ids = s["history"][r, :n].long() & 0xFFFF
        seen = torch.unique(ids)
        rep = s["repetition"][r].double()
        x[r, seen] = torch.where(x[r, seen] > 0, x[r, seen] / rep, x[r, seen] * rep)
        count = torch.bincount(ids[p:], minlength=v).double()
        x[r] -= s["frequency"][r].double() * count + s["presence"][r].double() * (count > 0)
    if s["bias"] is not None:
        x += s["bias"].double()
    if s["mask"] is not None:
        bits = (s["mask"].unsqueeze(-1) >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1
        x[bits.flatten(1)[:, :v] == 0] = float("-inf")
    return {"logits": x, "tokens": None}
