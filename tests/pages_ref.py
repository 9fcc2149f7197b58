"""Plain implementations of beam search's step, of the tables of the cache's
pages and of the choice of pages, in numpy, one row, page and entry at a time
(64 bits, and whole numbers)."""
import math

import numpy as np

NO_TOKEN = 65535
UNIT_MIN = -30


def beam_select(logits, scores, beams, weights=None, finished=None, eos=-1, history=None, lengths=None):
    """-> dict of tokens, parents, scores (64 bits), tol, finished, history,
    lengths.  tol: what the kernel's arithmetic leaves of a score: fp32
    exponentials of differences rounded to fp32 (half a step, 2^-24, of |x -
    max|), scaled by log2(e) as it is held in fp32 (2^-24 each for the constant
    and the product), with 2^-23 for the instruction; fp32 sums of at most 16
    terms a lane (2^-24 each); and the score's own rounding."""
    rows, vocab = logits.shape
    out = dict(tokens=np.full(rows, NO_TOKEN, np.int32), parents=np.full(rows, -1, np.int32),
               scores=np.full(rows, -np.inf), tol=np.zeros(rows), finished=np.zeros(rows, bool))
    if history is not None:
        out["history"], out["lengths"] = history.copy(), np.zeros(rows, np.int32)
        most = history.shape[1]
        held = np.clip(lengths, 0, most)
    for r0 in range(0, rows, beams):
        found = []
        for w in range(beams):
            r = r0 + w
            base = float(scores[r])
            weight = 1.0 if weights is None else float(weights[r])
            if not base > -math.inf or not weight > 0:
                continue
            if finished is not None and finished[r]:
                found.append((base * weight, w * vocab + eos, base, 0.0))
                continue
            x = logits[r].astype(np.float64)
            x = np.where(np.isnan(x), -np.inf, x)
            m = x.max()
            if not np.isfinite(m):
                continue
            e = np.exp(x - m)
            lse = m + math.log(e.sum())
            p = e / e.sum()
            err = (p[p > 0] * np.abs(x - m)[p > 0]).sum() * 3 * 2.0 ** -24 + 2.0 ** -23 + 17 * 2.0 ** -24
            s = base + (x - lse)
            order = np.lexsort((np.arange(vocab), -s))[:beams]
            found += [(s[v] * weight, w * vocab + int(v), s[v], err) for v in order if s[v] > -np.inf]
        found.sort(key=lambda f: (-f[0], f[1]))
        for k, (_, flat, s, err) in enumerate(found[:beams]):
            r, w, v = r0 + k, flat // vocab, flat % vocab
            out["tokens"][r], out["parents"][r], out["scores"][r] = v, r0 + w, s
            out["tol"][r] = err + (abs(s) * 2.0 ** -24 if np.isfinite(s) else 0.0)
            done = finished is not None and bool(finished[r0 + w])
            out["finished"][r] = done or (eos >= 0 and v == eos)
            if history is not None:
                n = int(held[r0 + w])
                out["history"][r, :n] = history[r0 + w, :n]
                if not done and n < most:
                    out["history"][r, n] = v
                    n += 1
                out["lengths"][r] = n
    return out


def valid(i, pages):
    return int(i) if 0 <= int(i) < pages else -1


def fork(table, start, refs, P, parents, news):
    """-> (table, start, refs, missing, copies [(src, dst, tokens)])."""
    nseq, width = table.shape
    pages = len(refs)
    cap = width * P
    refs = refs.astype(np.int64).copy()
    out = np.full_like(table, -1)
    st = np.zeros(nseq, np.int64)
    for i in range(nseq):
        p = i if parents is None else int(parents[i])
        if 0 <= p < nseq:
            st[i] = min(max(int(start[p]), 0), cap)
            held = -(-int(st[i]) // P)
            out[i, :held] = [valid(x, pages) for x in table[p, :held]]
    for t, by in ((table, -1), (out, 1)):
        for x in t.ravel():
            if valid(x, pages) >= 0:
                refs[x] += by
    n = np.array([min(max(int(news[i]), 0), cap - int(st[i])) for i in range(nseq)])
    last = np.full(nseq, -2)
    for i in range(nseq):
        if n[i] > 0 and st[i] % P:
            last[i] = out[i, st[i] // P]
    writers = {}
    for i in range(nseq):
        if last[i] >= 0:
            writers.setdefault(int(last[i]), []).append(i)
    copies, missing = [], int((last == -1).sum())
    moves = np.zeros(nseq, bool)
    for p, who in writers.items():
        refs[p] -= len(who)
        if refs[p] <= 0:
            refs[p] = 1
            who = who[1:]
        moves[who] = True
    free = [i for i in range(pages) if refs[i] <= 0]
    for i in range(nseq):
        want = [int(st[i]) // P] if moves[i] else []
        want += range(-(-int(st[i]) // P), -(-int(st[i] + n[i]) // P))
        for j in want:
            src = int(out[i, j])
            if free:
                d = free.pop(0)
                refs[d] = 1
                out[i, j] = d
                if moves[i] and j == st[i] // P:
                    copies.append((src, d, int(st[i]) % P))
            else:
                out[i, j] = -1
                missing += 1
    return out, st.astype(np.int32), refs.astype(np.int32), missing, copies


def copy_units(k, v, ke, ve, src, into, dst, tokens, box=None, into_box=None):
    """Page src of byte arrays (k [pages, kvh, P, dh], v in its own order) to
    page dst of `into` (k, v, ke, ve), the 16-token units of `tokens` tokens."""
    u = -(-tokens // 16)
    if u == 0:
        return
    ik, iv, ike, ive = into
    ik[dst, :, :16 * u] = k[src, :, :16 * u]
    iv[dst, :, :u] = v[src, :, :u]
    ike[dst], ive[dst] = ke[src], ve[src]
    if box is not None and into_box is not None:
        for a, b in zip(box, into_box):
            b[dst] = a[src]


def compact(refs, table=None):
    """-> (moved, refs, table, copies [(src, dst)])."""
    pages = len(refs)
    held = int((refs > 0).sum())
    holes = [i for i in range(held) if refs[i] <= 0]
    moved = np.full(pages, -1, np.int32)
    out = refs.copy()
    copies = []
    for i in range(pages):
        if refs[i] > 0:
            moved[i] = i if i < held else holes.pop(0)
            if i >= held:
                copies.append((i, int(moved[i])))
                out[moved[i]], out[i] = refs[i], 0
    if table is not None:
        table = np.array([[moved[x] if 0 <= x < pages else x for x in row] for row in table], np.int32).reshape(table.shape)
    return moved, out, table, copies


def unit(amax):
    """The smallest e >= -30 with amax <= 127 * 2^e."""
    e = UNIT_MIN
    while amax > 127 * 2.0 ** e:
        e += 1
    return e


def bound(k):
    """k [tokens, dh], 64 bits -> (box [2, dh], unit)."""
    some = ~np.isnan(k)
    hi = np.where(some, k, -np.inf).max(0)
    lo = np.where(some, k, np.inf).min(0)
    none = ~some.any(0)
    hi[none] = lo[none] = 0.0
    e = unit(max(abs(hi).max(), abs(lo).max()))
    return np.stack([np.ceil(hi * 2.0 ** -e), np.floor(lo * 2.0 ** -e)]).astype(np.int8), e


def page_scores(q, box, units):
    """q [group, dh], box [n, 2, dh], units [n] -> scores [n], exact."""
    best = np.full(len(units), -np.inf)
    for x in q.astype(np.float64):
        x = np.nan_to_num(np.clip(x, -65504, 65504), nan=0.0)
        f = unit(abs(x).max())
        z = np.rint(x * 2.0 ** -f).astype(np.int64)
        s = (z * np.where(z > 0, box[:, 0], box[:, 1]).astype(np.int64)).sum(1)
        best = np.maximum(best, s * 2.0 ** f)
    return best * 2.0 ** units.astype(np.float64)


def select(q, box, units, there, count, first, recent):
    """The places of one row and head among its context's pages (box, units and
    `there` by place)."""
    n = len(units)
    s = page_scores(q, box, np.where(there, units, 0))
    s = np.where((np.arange(n) < first) | (np.arange(n) >= n - recent), np.inf, s)
    order = [int(i) for i in np.lexsort((np.arange(n), -s)) if there[i]][:count]
    return np.array(sorted(order) + [-1] * (count - len(order)), np.int32)
