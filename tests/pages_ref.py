"""Plain 64-bit forms of the paged cache's operators (include/kv_pages.h) in numpy, and
how far a kernel with f32 scores, statistics and sums may be from them.

Bounds of the attention.  A score is scale times a sum of D exact products (f16 times f16,
or times an 8-bit code), summed in f32 in any order: off by at most D 2^-24 scale sum |q
k|; scaling, the row's k scale and the conversion to base 2 add 6 roundings of the
score itself, so e_s = (D scale sum |q k| + 6 |s|) 2^-24.  exp and log are good to 4
ulp, a sum of N non-negative terms in at least 16 chains to (N / 16 + 32) 2^-24
relative.  With e = max_j e_s of the row:
  lse:    e + (N / 16 + 40) 2^-24 + 2^-23 |lse|
  a weight, relative: 2 e + (N / 16 + 48) 2^-24; where it is multiplied with v it is
  the sum of two f16 values, off by 2^-22 of itself, or by 2^-25 where the second
  is subnormal; the largest weight (times its v scale) of a row is 2^6 at least, so N
  of them add N 2^-31 of the largest
  out:    that, times sum p |v|, and half a step of f16: 2^-11 |out| + 2^-25.
"""
from __future__ import annotations

import numpy as np

EPS = 2.0 ** -24


def rows_of(start, seqs, rows, max_rows):
    """(first row, rows) of every sequence, rows 0 for those left out."""
    if start is None:
        return [(s, 1) for s in range(seqs)]
    out = []
    for s in range(seqs):
        lo, hi = int(start[s]), int(start[s + 1])
        out.append((lo, hi - lo if 0 <= lo <= hi <= rows and hi - lo <= max_rows else 0))
    return out


def place(table, s, slot, pages, page_size):
    """(page, entry) of a slot, None for one that stands for nothing."""
    if not 0 <= slot < table.shape[1] * page_size:
        return None
    page = int(table[s, slot // page_size])
    return (page, slot % page_size) if 0 <= page < pages else None


def gather(pool, scale, table, s, count, h):
    """Slots 0 .. count - 1 of head h of a layer's pool [pages, kvh, page, D] in f64, and
    which of them stand for something."""
    pages, _, page_size, d = pool.shape
    x, ok = np.zeros((count, d)), np.zeros(count, bool)
    w = np.ones(count)
    for j in range(count):
        at = place(table, s, j, pages, page_size)
        if at is not None:
            ok[j] = True
            x[j] = pool[at[0], h, at[1]].astype(np.float64)
            if scale is not None:
                w[j] = np.float64(scale[at[0], h, at[1]])
    return x, w, ok


def attention(q, pools, table, length, start, max_rows, scale):
    """q [rows, qh, D] f16; pools (k, v, k_scale, v_scale) of one layer.  out, lse, their
    bounds, and which rows belong to a sequence."""
    k, v, ks, vs = pools
    rows, qh, d = q.shape
    kvh = k.shape[1]
    g = qh // kvh
    slots = table.shape[1] * k.shape[2]
    out, lse = np.zeros((rows, qh, d)), np.full((rows, qh), -np.inf)
    out_tol, lse_tol = np.zeros_like(out), np.zeros_like(lse)
    mine = np.zeros(rows, bool)
    for s, (lo, m) in enumerate(rows_of(start, len(length), rows, max_rows)):
        mine[lo:lo + m] = m > 0
        top = min(max(int(length[s]), 0), slots)
        if m == 0 or top == 0:
            continue
        for h in range(kvh):
            kx, kw, ok = gather(k, ks, table, s, top, h)
            vx, vw, _ = gather(v, vs, table, s, top, h)
            for i in range(m):
                see = ok & (np.arange(top) < int(length[s]) - m + 1 + i)
                if not see.any():
                    continue
                kk, vv = kx[see], vx[see]
                for j in range(h * g, (h + 1) * g):
                    qq = q[lo + i, j].astype(np.float64)
                    sc = scale * (kk @ qq) * kw[see]
                    e = ((d * scale * (np.abs(kk) @ np.abs(qq)) * np.abs(kw[see])
                          + 6 * np.abs(sc)) * EPS).max()
                    mx = sc.max()
                    w = np.exp(sc - mx)
                    tot = w.sum()
                    p = w / tot
                    N = int(see.sum())
                    lse[lo + i, j] = mx + np.log(tot)
                    lse_tol[lo + i, j] = e + (N / 16 + 40) * EPS + 2 * EPS * abs(lse[lo + i, j])
                    pv = p * vw[see]
                    o = pv @ vv
                    out[lo + i, j] = o
                    rel = 2 * e + (N / 16 + 48) * EPS + 2.0 ** -22
                    small = N * 2.0 ** -31 * np.abs(pv).max() * np.abs(vv).max(0)
                    out_tol[lo + i, j] = (rel * (np.abs(pv) @ np.abs(vv)) + small
                                          + 2.0 ** -11 * np.abs(o) + 2.0 ** -25)
    return out, lse, out_tol, lse_tol, mine


def turned(x, norm, eps, theta, position):
    """x [heads, D] f16 of one row: norm and rotation in f64."""
    y = x.astype(np.float64)
    d = y.shape[-1]
    with np.errstate(invalid="ignore", over="ignore"):
        if norm is not None:
            y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * norm.astype(np.float64)
        if theta:
            a = position * theta ** (-2.0 * np.arange(d // 2) / d)
            lo, hi = y[..., :d // 2], y[..., d // 2:]
            y = np.concatenate([lo * np.cos(a) - hi * np.sin(a), hi * np.cos(a) + lo * np.sin(a)], -1)
    return y


def check_codes(y, code, scale):
    """y [.., D] f64 against int8 codes and their f32 scales: the scale the f32 nearest to
    max / 127, every code the nearest, a border within 2^-40 either way."""
    for idx in np.ndindex(y.shape[:-1]):
        if not np.isfinite(y[idx]).all():
            assert np.isnan(scale[idx]), idx
            continue
        want = np.abs(y[idx]).max() / 127.0
        s = np.float64(scale[idx])
        assert abs(s - want) <= (0.5 + 2.0 ** -20) * np.spacing(np.float32(want)), (idx, s, want)
        if s == 0.0:
            assert (code[idx] == 0).all(), idx
            continue
        x = y[idx] / s
        assert (np.abs(x - code[idx]) <= 0.5 + 2.0 ** -40).all(), (idx, x, code[idx])


def verify(logits, tokens, start, seqs, max_rows, uniform, temperature=None, draft=None):
    """out [seqs, max_rows], accepted [seqs], logprob, and the least relative distance of a
    random number from a border it could have fallen on the other side of."""
    rows, vocab = logits.shape
    out = np.full((seqs, max_rows), -1, np.int64)
    accepted = np.zeros(seqs, np.int64)
    logprob = np.zeros((seqs, max_rows))
    margin = np.inf
    for s, (lo, m) in enumerate(rows_of(start, seqs, rows, max_rows)):
        if m == 0:
            continue
        heat = 1.0 if temperature is None else float(np.float32(temperature[s]))
        n = 0
        while True:
            x = logits[lo + n].astype(np.float64)
            x[np.isnan(x)] = -np.inf
            top = x.max()
            p = np.zeros(vocab)
            if top > -np.inf:
                if not heat > 0:
                    p[np.argmax(x)] = 1.0
                else:
                    with np.errstate(invalid="ignore", over="ignore"):
                        p = np.where(x == top, 1.0, np.exp((x - top) / heat))
                    p = p / p.sum()
            w = p
            if n < m - 1:
                t = int(tokens[lo + n + 1])
                inside = 0 <= t < vocab
                if draft is None:
                    q = np.zeros(vocab)
                    if inside:
                        q[t] = 1.0
                else:
                    q = draft[lo + n].astype(np.float64)
                    q[~(q > 0)] = 0.0
                u = float(np.float32(uniform[lo + n]))
                if inside:
                    margin = min(margin, abs(u * q[t] - p[t]) / max(p[t], 1e-300))
                if inside and u * q[t] < p[t]:
                    out[s, n], logprob[s, n] = t, np.log(p[t])
                    n += 1
                    continue
                rest = np.maximum(p - q, 0.0)
                if rest.sum() > 0:
                    w = rest
            accepted[s] = n
            c = np.cumsum(w)
            if c[-1] > 0:
                goal = float(np.float32(uniform[lo + m - 1])) * c[-1]
                above = np.nonzero(c > goal)[0]
                some = np.nonzero(w > 0)[0]
                j = int(above[0]) if above.size else int(some[-1])
                margin = min(margin, np.abs(c[some] - goal).min() / c[-1])
                out[s, n], logprob[s, n] = j, np.log(p[j])
            break
    return out, accepted, logprob, margin
