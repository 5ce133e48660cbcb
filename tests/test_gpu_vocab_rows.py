"""f16_gemm_argmax with more 128-row tiles than workgroups: sums, argmax and copies that
run on from one tile into the next, and a ragged last tile behind whole ones.  Rows,
tokens and bounds as in test_vocab_rows."""
from __future__ import annotations

import numpy as np
import pytest

import cache_ref as R
from test_gpu_cache import first_max, normal, run_vocab

pytestmark = pytest.mark.gpu

ROUND = 256 * 128  # rows between a workgroup's tiles


@pytest.fixture(scope="module")
def matrix():
    return normal(np.random.default_rng(1), (70003, 1024), 0.02)


@pytest.mark.parametrize("rows", [ROUND, ROUND + 1, 33001, 2 * ROUND + 130, 70003])
@pytest.mark.parametrize("n", [13, 64, 100, 256])
def test_tiles_of_one_workgroup(gpu, matrix, rows, n):
    w, x = matrix[:rows], normal(np.random.default_rng(rows + n), (n, 1024))
    got, tok = run_vocab(gpu, w, x)
    assert np.array_equal(tok, [first_max(r) for r in got])
    for r0 in range(0, rows, 8192):
        part = w[r0:r0 + 8192].astype(np.float64)
        ref = x.astype(np.float64) @ part.T
        mag = np.abs(x.astype(np.float64)) @ np.abs(part).T
        tol = 1024 * R.EPS * mag + 2.0 ** -11 * np.abs(ref) + 2.0 ** -25
        assert (np.abs(got[:, r0:r0 + 8192].astype(np.float64) - ref) <= tol).all(), r0
    _, tok2 = run_vocab(gpu, w, x, logits=False)
    assert np.array_equal(tok, tok2)


@pytest.mark.parametrize("n", [13, 100, 256])
def test_ties_between_tiles(gpu, matrix, n):
    """Equal maxima in different tiles of one workgroup and in tiles of others: the
    lowest row wins, wherever it is."""
    rng = np.random.default_rng(n)
    w = matrix.copy()
    x = normal(rng, (n, 1024))
    want = []
    for i in range(n):
        base = int(rng.integers(0, 70003 - 2 * ROUND))
        spots = [base, base + ROUND, base + 2 * ROUND, int(rng.integers(0, 70003))]
        spots = sorted(rng.permutation(spots)[:int(rng.integers(1, 5))])
        row = (x[i].astype(np.float32) * 0.1).astype(np.float16)
        w[spots] = row
        want.append(spots)
    got, tok = run_vocab(gpu, w, x)
    assert np.array_equal(tok, [first_max(r) for r in got])
    # a later token's copies may have taken a spot over
    for i, spots in enumerate(want):
        left = [s for s in spots if np.array_equal(w[s], (x[i].astype(np.float32) * 0.1).astype(np.float16))]
        if left:
            assert tok[i] == left[0]
