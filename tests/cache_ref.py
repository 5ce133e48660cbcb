"""Plain 64-bit forms of the cache operators (include/f16_cache.h) in numpy, and
how far a kernel with f32 scores, statistics and sums may be from them.

Bounds.  A score is scale times a sum of D exact products of f16 values, summed
in f32 in any order: off by at most D 2^-24 scale sum |q k|, and scaling and the
conversion to base 2 add 4 roundings of the score itself, so
  e_s = (D scale sum |q k| + 4 |s|) 2^-24.
exp and log are good to 4 ulp, and a sum of N non-negative terms in at least 16
chains to (N / 16 + 32) 2^-24 relative.  With e = max_j e_s of the row:
  lse:    e + (N / 16 + 40) 2^-24 + 2^-23 |lse|
  a weight, relative: 2 e + (N / 16 + 48) 2^-24; where it is multiplied with v it
  has been rounded to f16, at most half a step, 2^-11 of itself (the kernels keep
  weights below 2^-14 of 2^6 or more, whose step is 2^-24, so N of them add
  N 2^-25 / 2^6 of the row's largest)
  out:    that, times sum p |v|, and half a step of f16: 2^-11 |out| + 2^-25.
"""
from __future__ import annotations

import numpy as np

EPS = 2.0 ** -24


def tree_see(parents) -> np.ndarray:
    n = len(parents)
    see = np.zeros((n, n), bool)
    for i, p in enumerate(parents):
        if p == -1:
            see[i, i] = True
        elif 0 <= p < i and see[p].any():
            see[i] = see[p]
            see[i, i] = True
    return see


def pack_mask(see: np.ndarray) -> np.ndarray:
    n = see.shape[0]
    words = (n + 31) // 32
    bits = np.zeros((n, words * 32), np.uint64)
    bits[:, :n] = see
    w = (bits.reshape(n, words, 32) << np.arange(32, dtype=np.uint64)).sum(-1)
    return w.astype(np.uint32)


def random_tree(rng, n: int, pad: int = 0) -> np.ndarray:
    p = np.array([-1] + [i - 1 if rng.random() < 0.5 else int(rng.integers(0, i))
                         for i in range(1, n)], np.int32)
    if pad:
        p[n - pad:] = -2
    return p


def scores(q, k, scale):
    """q [n, qh, D], k [S, kvh, D] -> s [n, qh, S] and the bound e_s, in f64."""
    n, qh, d = q.shape
    g = qh // k.shape[1]
    q, k = q.astype(np.float64), k.astype(np.float64)
    s = np.empty((n, qh, k.shape[0]))
    e = np.empty_like(s)
    for h in range(qh):
        s[:, h] = scale * (q[:, h] @ k[:, h // g].T)
        e[:, h] = (d * scale * (np.abs(q[:, h]) @ np.abs(k[:, h // g]).T) + 4 * np.abs(s[:, h])) * EPS
    return s, e


def attention(q, k, v, see, length, scale):
    """out [n, qh, D], lse [n, qh] in f64 and the bounds of both.  k, v hold
    slots 0 .. length + n - 1; masked entries are never read."""
    n, qh, d = q.shape
    g = qh // k.shape[1]
    out = np.zeros((n, qh, d))
    lse = np.full((n, qh), -np.inf)
    out_tol, lse_tol = np.full_like(out, 0.0), np.zeros_like(lse)
    for i in range(n):
        if not see[i].any():
            continue
        at = np.concatenate([np.arange(length), length + np.nonzero(see[i])[0]])
        s, e = scores(q[i:i + 1], k[at], scale)
        s, e = s[0], e[0].max(-1)
        top = s.max(-1, keepdims=True)
        w = np.exp(s - top)
        tot = w.sum(-1, keepdims=True)
        lse[i] = (top + np.log(tot))[:, 0]
        p = w / tot
        N = len(at)
        lse_tol[i] = e + (N / 16 + 40) * EPS + 2 * EPS * np.abs(lse[i])
        rel = 2 * e + (N / 16 + 48) * EPS + 2.0 ** -11
        small = N * 2.0 ** -31 * p.max(-1)  # of weights that are subnormal in f16
        for h in range(qh):
            vv = v[at, h // g].astype(np.float64)
            out[i, h] = p[h] @ vv
            out_tol[i, h] = rel[h] * (p[h] @ np.abs(vv)) + small[h] * np.abs(vv).max(0) + 2.0 ** -11 * np.abs(out[i, h]) + 2.0 ** -25
    return out, lse, out_tol, lse_tol


def weights_add(w, q, lse, k, path, length, n, scale):
    """w [kvh, max_seq] f32 of one layer -> the sums in f64 and their bound."""
    kvh = k.shape[1]
    rows, qh, d = q.shape
    g = qh // kvh
    out = w.astype(np.float64)
    out[:, length:length + n] = 0.0
    add = np.zeros((kvh, length + n))
    err = np.zeros_like(add)
    for i in range(n):
        r = int(path[i])
        if not 0 <= r < rows:
            continue
        S = length + i + 1
        s, e = scores(q[r:r + 1], k[:S], scale)
        with np.errstate(over="ignore"):
            x = np.where(np.isneginf(lse[r])[:, None], 0.0,
                         np.exp(s[0] - np.where(np.isneginf(lse[r]), 0.0, lse[r]).astype(np.float64)[:, None]))
        rel = e[0] + 2 * EPS * np.abs(np.where(np.isneginf(lse[r]), 0, lse[r]))[:, None] + 8 * EPS
        for h in range(qh):
            add[h // g, :S] += x[h]
            err[h // g, :S] += x[h] * rel[h]
    out[:, :length + n] += add
    tol = np.zeros_like(out)
    # n g positive terms in any order, then one addition
    tol[:, :length + n] = err + (n * g + 2) * EPS * add + EPS * np.abs(out[:, :length + n]) + 1e-38
    return out, tol


def select(w, length, budget, sinks, recent):
    """kept slots [.., budget] of w [.., max_seq], equal weights lowest first,
    NaN below every number."""
    lead = w.shape[:-1]
    flat = w.reshape(-1, w.shape[-1])
    keep = np.empty((flat.shape[0], budget), np.int32)
    for r, row in enumerate(flat):
        mid = row[sinks:length - recent].astype(np.float64)
        # finite stand-ins that order NaN below -inf
        key = np.where(np.isnan(mid), -np.inf, np.where(np.isneginf(mid), -1e300, mid))
        order = np.argsort(-key, kind="stable")[:budget - sinks - recent]
        keep[r] = np.concatenate([np.arange(sinks), np.sort(order) + sinks,
                                  np.arange(length - recent, length)])
    return keep.reshape(*lead, budget)
