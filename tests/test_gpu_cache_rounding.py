"""How far tree attention (f16_attn_tree) may be from its 64-bit form, at every
number of rows: a softmax weight enters the product with v to 2^-22 of itself, so
that the output's own rounding to f16 is what is left.

Bounds as in cache_ref, but with 2^-22 for a weight (a sum of two f16 values, each
off by half a step) in place of 2^-11.  An output is the f16 nearest to a value
within that bound of the exact one: rounding keeps order, so it lies between the
roundings of both ends.  Queries are small, so that the scores' own bound, which
grows with them, stays far below a step of f16."""
from __future__ import annotations

import numpy as np
import pytest

import cache_ref as R
from test_gpu_cache import C, make, normal, run_tree  # noqa: F401 (C: the fixture)

pytestmark = pytest.mark.gpu

WEIGHT = 2.0 ** -22


def check_rows(got, lse, q, k, v, see, length, scale, rows, weight=WEIGHT):
    """Rows `rows` of got [n, qh, d] and lse [n, qh] against the 64-bit form."""
    g = q.shape[1] // k.shape[1]
    for i in rows:
        if not see[i].any():
            assert (got[i] == 0).all() and np.isneginf(lse[i]).all()
            continue
        own = length + np.nonzero(see[i])[0]
        kk, vv = (np.concatenate([a[:length], a[own]]) for a in (k, v))
        s, e = R.scores(q[i:i + 1], kk, scale)
        s, e = s[0], e[0].max(-1)
        top = s.max(-1, keepdims=True)
        w = np.exp(s - top)
        tot = w.sum(-1)
        N = len(kk)
        want = top[:, 0] + np.log(tot)
        assert (np.abs(lse[i] - want) <= e + (N / 16 + 40) * R.EPS + 2 * R.EPS * np.abs(want)).all()
        p = w / tot[:, None]
        rel = 2 * e + (N / 16 + 48) * R.EPS + weight
        small = N * 2.0 ** -31 * p.max(-1)
        for h in range(q.shape[1]):
            x = vv[:, h // g].astype(np.float64)
            out = p[h] @ x
            tol = rel[h] * (p[h] @ np.abs(x)) + small[h] * np.abs(x).max(0)
            lo, hi = (out - tol).astype(np.float16), (out + tol).astype(np.float16)
            bad = ~((lo <= got[i, h]) & (got[i, h] <= hi))
            assert not bad.any(), (i, h, int(bad.sum()), got[i, h][bad][:4], out[bad][:4], tol[bad][:4])


@pytest.mark.parametrize("qh,kvh,d,n,length", [
    (16, 8, 128, 1, 300), (16, 8, 128, 8, 77), (16, 8, 128, 16, 500), (16, 8, 128, 17, 40),
    (16, 8, 128, 32, 200), (16, 8, 128, 32, 1000), (16, 8, 128, 33, 90), (16, 8, 128, 61, 700),
    (16, 8, 128, 130, 30), (16, 8, 128, 256, 200), (64, 2, 64, 1, 200), (64, 2, 64, 2, 100),
    (64, 2, 64, 9, 500), (14, 2, 64, 5, 60), (14, 2, 64, 40, 33), (9, 3, 64, 100, 400)])
def test_outputs_are_rounded_once(gpu, C, qh, kvh, d, n, length):  # noqa: F811
    rng = np.random.default_rng(n + length + qh)
    k, v = make(rng, kvh, d, length, n)
    q = normal(rng, (n, qh, d), 0.02)
    see = R.tree_see(R.random_tree(rng, n, pad=n // 8))
    got, lse = run_tree(gpu, C, k, v, q, see, length, d ** -0.5)
    check_rows(got, lse, q, k[0], v[0], see, length, d ** -0.5, range(0, n, max(1, n // 40)))


@pytest.mark.parametrize("qh,kvh,d,n,length,std", [
    (16, 8, 128, 256, 8400, 0.02),   # two row tiles a wave, 16 splits
    (16, 8, 128, 256, 9001, 1.5),
    (256, 128, 64, 256, 500, 0.02),  # and no split at all: outputs straight from the tiles
    (256, 128, 64, 255, 411, 1.5)])
def test_large_trees(gpu, C, qh, kvh, d, n, length, std):  # noqa: F811
    """Where each CU has much to do; rows of every wave and tile, padding at the end."""
    rng = np.random.default_rng(length)
    k, v = make(rng, kvh, d, length, n)
    q = normal(rng, (n, qh, d), std)
    parents = R.random_tree(rng, n, pad=20)
    parents[100] = n
    see = R.tree_see(parents)
    got, lse = run_tree(gpu, C, k, v, q, see, length, d ** -0.5)
    dead = ~see.any(1)
    assert dead.sum() >= 21 and (got[dead] == 0).all() and np.isneginf(lse[dead]).all()
    check_rows(got, lse, q, k[0], v[0], see, length, d ** -0.5,
               [0, 7, 8, 15, 16, 63, 64, 99, 101, 160, 200, n - 21, n - 20, n - 1])
