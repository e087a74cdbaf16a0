"""Plain 64-bit forms of the serving operators (numpy), written from their
definitions: cache plan, 8-bit cache writes, attention, log probabilities."""

import numpy as np

QMAX = {"e4m3": 448.0, "int8": 127.0}
EXP_LO, EXP_HI = -40, 40


def plan(lens, new, table, free, cursor, page, n_tokens):
    """(kv_lens, cu, positions, slots, cursor, table) by walking the requests."""
    table = table.copy()
    cu, pos, slots = [0], [], []
    for b, (a, n) in enumerate(zip(lens, new)):
        for col in range(-(-a // page), -(-(a + n) // page)):
            p = free[cursor] if cursor < len(free) else -1
            cursor += cursor < len(free)
            if col < table.shape[1]:
                table[b, col] = p
        for t in range(a, a + n):
            pg = table[b, t // page] if t // page < table.shape[1] else -1
            pos.append(t)
            slots.append(pg * page + t % page if pg >= 0 else -1)
        cu.append(cu[-1] + n)
    pos, slots = pos[:n_tokens], slots[:n_tokens]
    pad = n_tokens - len(pos)
    return (np.add(lens, new), np.minimum(cu, n_tokens), np.array(pos + [0] * pad), np.array(slots + [-1] * pad),
            cursor, table)


def scale_exponent(amax, code):
    """The smallest e in [EXP_LO, EXP_HI] with amax <= QMAX * 2^e (EXP_HI if none)."""
    for e in range(EXP_LO, EXP_HI):
        if amax <= QMAX[code] * 2.0 ** e:
            return e
    return EXP_HI


def round_code(y, code):
    """Round to nearest even on the codes' grid; the range's ends beyond it."""
    y = np.asarray(y, np.float64)
    if code == "int8":
        return np.clip(np.rint(np.nan_to_num(y, nan=0.0, posinf=1e9, neginf=-1e9)), -127, 127)
    mag = np.minimum(np.abs(y), 1e9)
    e = np.maximum(np.frexp(np.maximum(mag, 2.0 ** -30))[1] - 1, -6)
    step = 2.0 ** (e - 3)
    return np.where(np.isnan(y), np.nan, np.sign(y) * np.minimum(np.rint(mag / step) * step, 448.0))


def append(x, slots, codes, scale, code, v=None):
    """One of K and V: x [T, heads, dim], codes [pages, heads, page, dim] as numbers, scale [pages, heads].
    For K in e4m3, `v` is V: a token's NaN there makes its whole key NaN; for V it is not given, and NaN becomes 0."""
    codes, scale = codes.astype(np.float64).copy(), scale.astype(np.float64).copy()
    P = codes.shape[2]
    t = 0
    while t < len(slots):
        if slots[t] < 0 or slots[t] >= codes.shape[0] * P:
            t += 1
            continue
        n = 1
        while t + n < len(slots) and slots[t + n] >= 0 and slots[t + n] // P == slots[t] // P:
            n += 1
        pg, off = slots[t] // P, slots[t] % P
        for h in range(codes.shape[1]):
            rows = x[t:t + n, h].astype(np.float64)
            mag = np.abs(rows)
            e = scale_exponent(np.max(np.where(np.isnan(mag), 0.0, mag)), code)
            if off:
                was = int(np.log2(scale[pg, h]))
                e = max(e, was)
                if e > was:
                    codes[pg, h, :off] = round_code(codes[pg, h, :off] * 2.0 ** (was - e), code)
            scale[pg, h] = 2.0 ** e
            for i in range(n):
                got = round_code(rows[i] * 2.0 ** -e, code)
                if v is None:
                    got = np.nan_to_num(got)
                elif code == "e4m3" and np.isnan(v[t + i, h]).any():
                    got = np.full_like(got, np.nan)
                codes[pg, h, slots[t + i] % P] = got
        t += n
    return codes, scale


def attend(q, kv, table, kv_lens, cu, scale, window):
    """q [rows, heads, dim]; kv = (k, v) values [pages, kv_heads, page, dim].

    Returns out, lse and, for the error bounds, sum p |v|, max |v| and the
    largest sum |q k| * scale of each row."""
    k, v = kv
    rows, heads, D = q.shape
    G, P = heads // k.shape[1], k.shape[2]
    out, lse = np.zeros((rows, heads, D)), np.full((rows, heads), -np.inf)
    amp, vmax, smax = np.zeros_like(out), np.zeros_like(out), np.zeros_like(lse)
    for b, n in enumerate(kv_lens):
        new = cu[b + 1] - cu[b]
        for i in range(new):
            pos = n - new + i
            lo = max(0, pos - window + 1) if window else 0
            js = np.arange(lo, pos + 1)
            js = js[[0 <= table[b, j // P] < k.shape[0] for j in js]] if len(js) else js
            if not len(js):
                continue
            pg = table[b, js // P]
            for h in range(heads):
                kk, vv = k[pg, h // G, js % P], v[pg, h // G, js % P]
                qq = q[cu[b] + i, h]
                s = scale * (kk @ qq)
                m = s.max()
                p = np.exp(s - m)
                r = cu[b] + i
                out[r, h] = p @ vv / p.sum()
                lse[r, h] = m + np.log(p.sum())
                amp[r, h] = p @ np.abs(vv) / p.sum()
                vmax[r, h] = np.abs(vv).max()
                smax[r, h] = abs(scale) * (np.abs(kk) @ np.abs(qq)).max()
    return out, lse, amp, vmax, smax


def logprobs(x, tokens, top):
    """x [rows, vocab] float64; (logprob, entropy, rank, top values, top ids)."""
    lp, ent, rank, vals, ids = [], [], [], [], []
    for row, t in zip(x, tokens):
        m = row.max()
        with np.errstate(invalid="ignore"):
            e = np.exp(row - (m if m > -np.inf else 0.0))
            s = e.sum()
            logp = row - m - np.log(s) if s > 0 else np.full_like(row, -np.inf)
            p = e / s if s > 0 else e
            ent.append(-np.sum(np.where(p > 0, p * np.where(p > 0, logp, 0.0), 0.0)))
        order = np.lexsort((np.arange(len(row)), -row))
        vals.append(logp[order[:top]])
        ids.append(order[:top])
        ok = 0 <= t < len(row)
        lp.append(logp[t] if ok else -np.inf)
        rank.append(1 + int(np.sum(row > row[t]) + np.sum(row[:t] == row[t])) if ok else 0)
    return np.array(lp), np.array(ent), np.array(rank), np.array(vals).reshape(len(x), top), np.array(ids).reshape(len(x), top)
