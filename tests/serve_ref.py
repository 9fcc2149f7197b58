"""Plain 64-bit implementations of the serving operators, in numpy, one
sequence, page and row at a time, and the tolerances that the kernels'
arithmetic leaves."""
import numpy as np

E_MIN, E_MAX = -15, 8
HALF_MAX = 65504.0


def code_values():
    """The value of every e4m3 code."""
    b = np.arange(256)
    s, e, m = np.where(b & 128, -1.0, 1.0), b >> 3 & 15, b & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    v = np.where((b & 127) == 127, np.nan, v)
    return s * v


VALUES = code_values()


def near(x):
    """x, at most 448 in magnitude, to the nearest e4m3 value, ties to even."""
    a = np.abs(x)
    step = 2.0 ** (np.floor(np.log2(np.maximum(a, 2.0 ** -6))) - 3)
    return np.sign(x) * np.rint(a / step) * step


def exponent(x):
    """Smallest e in [-15, 8] with max |x| <= 448 * 2^e; NaN not counted."""
    top = np.nanmax(np.abs(x)) if np.isfinite(x).any() or np.isinf(x).any() else 0.0
    e = E_MIN
    while e < E_MAX and top > 448 * 2.0 ** e:
        e += 1
    return e


def limit(x):
    return np.where(np.isnan(x), x, np.clip(x, -HALF_MAX, HALF_MAX))


def quantise(x, e):
    y = limit(x) * 2.0 ** -e
    if e == E_MAX:
        y = np.where(np.isnan(y), y, np.clip(y, -240, 240))
    return near(y)


def rope(x, cos, sin):
    """x [tokens, heads, dh], cos and sin [tokens, dh/2]."""
    a, b = x[..., 0::2], x[..., 1::2]
    c, s = cos[:, None], sin[:, None]
    return np.stack([a * c - b * s, b * c + a * s], -1).reshape(x.shape)


def v_rows(v):
    """[pages, kvh, P/16, 4, 16, dh/16, 4] -> [pages, kvh, P, dh]."""
    p, h, u, _, _, t, _ = v.shape
    return v.transpose(0, 1, 2, 3, 6, 5, 4).reshape(p, h, u * 16, t * 16)


def append(k, v, k_exp, v_exp, table, start, offsets, xk, xv, cos, sin):
    """Pools as code values (k and v [pages, kvh, P, dh], float64, changed in
    place with their exponents); xk, xv [rows, kvh, dh] before the rotation."""
    pages, kvh, P, _ = k.shape
    cap = table.shape[1] * P
    for i in range(len(start)):
        a0, n = int(offsets[i]), int(offsets[i + 1] - offsets[i])
        n = min(n, cap - int(start[i]))
        pos = int(start[i])
        end = pos + n
        while pos < end:
            stop = min(end, (pos // P + 1) * P)
            row = a0 + pos - int(start[i])
            cnt, r0 = stop - pos, pos % P
            page = int(table[i, pos // P])
            if 0 <= page < pages:
                turned = rope(xk[row:row + cnt], cos[pos:stop], sin[pos:stop])
                for pool, exps, x in ((k, k_exp, turned), (v, v_exp, xv[row:row + cnt])):
                    for h in range(kvh):
                        e = exponent(limit(x[:, h]))
                        if r0:
                            old = int(exps[page, h])
                            e = max(e, old)
                            pool[page, h, :r0] = near(pool[page, h, :r0] * 2.0 ** (old - e))
                        pool[page, h, r0:r0 + cnt] = quantise(x[:, h], e)
                        exps[page, h] = e
            pos = stop


def attend(k, v, k_exp, v_exp, table, start, offsets, q, scale):
    """-> (out [rows, heads, dh], tolerance) in 64 bits; rows of no sequence
    are NaN in both.  k, v: code values [pages, kvh, P, dh].

    The tolerance counts, per row: fp32 sums of the dh products of a score
    (each addition half a step of at most the sum of magnitudes, 2^-24), the
    score's scaling and the exponential (arguments off by 2^-23 of the largest
    score's magnitude, 2^-23 for the instruction), which move a weight by that
    much relatively; fp16 weights (2^-11 of each, or half of 2^-24 where they
    are tiny); fp32 sums over the keys (2^-24 times their number, times two for
    the parts that are joined); the output's rounding to fp16 (2^-11, or half
    of 2^-24)."""
    pages, kvh, P, dh = k.shape
    rows, heads, _ = q.shape
    g = heads // kvh
    cap = table.shape[1] * P
    out = np.full(q.shape, np.nan)
    tol = np.full(q.shape, np.nan)
    for i in range(len(start)):
        a0, n, st = int(offsets[i]), int(offsets[i + 1] - offsets[i]), int(start[i])
        n = min(n, cap - st)
        if n <= 0:
            continue
        ids = table[i, :(st + n + P - 1) // P]
        there = np.repeat((ids >= 0) & (ids < pages), P)[:st + n]
        ids = np.where((ids >= 0) & (ids < pages), ids, 0)
        kk = (k[ids] * 2.0 ** k_exp[ids][:, :, None, None]).transpose(0, 2, 1, 3).reshape(-1, kvh, dh)[:st + n]
        vv = (v[ids] * 2.0 ** v_exp[ids][:, :, None, None]).transpose(0, 2, 1, 3).reshape(-1, kvh, dh)[:st + n]
        for t in range(n):
            m = there[:st + t + 1]
            for h in range(heads):
                K, V = kk[:st + t + 1, h // g][m], vv[:st + t + 1, h // g][m]
                if not len(K):
                    out[a0 + t, h], tol[a0 + t, h] = 0.0, 0.0
                    continue
                x = q[a0 + t, h].astype(np.float64)
                s = scale * (K @ x)
                w = np.exp(s - s.max())
                w /= w.sum()
                o = w @ V
                ds = scale * (np.abs(K) @ np.abs(x)).max() * (dh + 1) * 2.0 ** -24
                ds += (np.abs(s).max() + 1) * 2.0 ** -22 + 2.0 ** -23
                rel = 2 * ds + 2.0 ** -11 + len(K) * 2.0 ** -23
                out[a0 + t, h] = o
                tol[a0 + t, h] = rel * (w @ np.abs(V)) + 2.0 ** -25 * np.abs(V).sum(0) + np.abs(o) * 2.0 ** -11 + 2.0 ** -25
    return out, tol


def control(logits, history, lengths, prompts, repetition, frequency, presence, bias, mask):
    """fp32, every step rounded, as the operator is defined: (logits, tokens)."""
    f = np.float32
    x = logits.astype(f).copy()
    rows, vocab = x.shape
    tokens = np.full(rows, 65535, np.int32)
    with np.errstate(invalid="ignore", over="ignore"):
        for r in range(rows):
            if history is not None:
                n = int(np.clip(lengths[r], 0, history.shape[1]))
                p = 0 if prompts is None else int(np.clip(prompts[r], 0, n))
                ids = history[r, :n].astype(np.int64)
                ids[ids >= vocab] = vocab
                every = np.bincount(ids, minlength=vocab + 1)[:vocab]
                said = np.bincount(ids[p:], minlength=vocab + 1)[:vocab]
                rep = f(1) if repetition is None else repetition[r]
                fr = f(0) if frequency is None else frequency[r]
                pr = f(0) if presence is None else presence[r]
                a, o = every > 0, said > 0
                x[r, a] = np.where(x[r, a] > 0, x[r, a] / rep, x[r, a] * rep)
                x[r, o] = (x[r, o] - fr * said[o].astype(f)) - pr
            if bias is not None:
                x[r] = x[r] + (bias if bias.ndim == 1 else bias[r])
            if mask is not None:
                words = (mask if mask.ndim == 1 else mask[r]).astype(np.uint32)
                bits = words[np.arange(vocab) // 32] >> (np.arange(vocab) % 32).astype(np.uint32) & 1
                x[r, bits == 0] = -np.inf
            y = np.where(np.isnan(x[r]), -np.inf, x[r])
            if y.max() > -np.inf:
                tokens[r] = y.argmax()
    return x, tokens
