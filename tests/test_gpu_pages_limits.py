"""The paged cache's operators (include/kv_pages.h) on the GPU where their numbers come near
the limits of what holds them: temperatures and logits of every size.  Against the plain
64-bit forms (pages_ref), with the tolerances of test_gpu_pages."""
from __future__ import annotations

import numpy as np
import pytest

import test_gpu_pages as T

pytestmark = pytest.mark.gpu

P = T.P

HEATS = [1e-6, 1e-5, 1e-4, 1e-3, 1e-2, 0.1, 10.0, 1e6]
TOPS = [-1000.0, -10.0, -1.0, 0.0, 0.06, 10.0, 40.0, 1000.0]


def shifted(heat, top, masked):
    """Logits whose rows have their maximum at `top`, some of a row -inf, one temperature."""
    def spoil(logits, tokens, temperature, draft):
        x = logits.astype(np.float32)
        logits[:] = (x - x.max(1, keepdims=True) + np.float32(top)).astype(np.float16)
        if masked:
            logits[:, 1::3] = -np.inf
            logits[::2, :100] = np.nan
        temperature[:] = np.float32(heat)

    return spoil


@pytest.mark.parametrize("drafted", [True, False])
@pytest.mark.parametrize("heat", HEATS)
def test_verify_temperatures(gpu, P, heat, drafted):
    """Cold rows, in which all but the maxima vanish, and hot ones, in both chunk sizes (9001
    logits of 11 rows, of 130) and with one row a sequence."""
    for i, top in enumerate(TOPS):
        for masked in (False, True):
            spoil = shifted(heat, top, masked)
            T.verify_case(gpu, P, 40 + i, 9001, [3, 2, 1, 5], drafted=drafted, heat="warm", spoil=spoil)
    for top in (-10.0, 40.0):
        T.verify_case(gpu, P, 50, 9001, [5] * 26, drafted=drafted, heat="warm", spoil=shifted(heat, top, True))
        T.verify_case(gpu, P, 51, 9001, None, rows=9, drafted=drafted, heat="warm",
                      spoil=shifted(heat, top, True))


@pytest.mark.parametrize("drafted", [True, False])
@pytest.mark.parametrize("heat", [1e25, 1e36, 3e38, np.inf])
def test_verify_hottest_rows(gpu, P, heat, drafted):
    """All finite logits alike, and -inf and NaN among them without any probability."""
    for i, top in enumerate((-1000.0, 0.0, 40.0)):
        T.verify_case(gpu, P, 60 + i, 9001, [3, 2, 1, 5], drafted=drafted, heat="warm",
                      spoil=shifted(heat, top, heat < np.inf))


@pytest.mark.parametrize("drafted", [True, False])
@pytest.mark.parametrize("vocab", [524288, 524289, 1100003])
def test_verify_large_vocabularies(gpu, P, vocab, drafted):
    """More parts of a row than a workgroup has threads, the token in the first of them, in the
    last and between."""
    for i, uniform in enumerate((None, 0.0, 1.0 - 2.0 ** -24)):
        T.verify_case(gpu, P, 80 + i, vocab, [2, 1, 3], drafted=drafted, uniform=uniform, heat="warm",
                      spoil=shifted(10.0, 5.0, False))
        T.verify_case(gpu, P, 90 + i, vocab, None, rows=2, drafted=drafted, uniform=uniform)


def far_case(Q, P, heads, counts, gap, scale_far, other):
    """8-bit pages whose slots have scores 0 but for some whose v is nothing (codes or scale 0,
    or a scale of 2^-120) `gap` above in units of log 2, and, with other, a few ordinary ones as
    far up, in the same blocks of 32 slots and in others."""
    rng = np.random.default_rng(70)
    qh, kvh, d = heads
    lengths = [900, 70, 3000]
    need = sum((n + 15) // 16 for n in lengths) + 1
    pool = T.Pool(Q, P, rng, 1, need, 16, kvh, d, 8)
    batch = T.Batch(Q, P, rng, pool, lengths, counts)
    (k, v), (ks, vs) = pool.host, pool.scales
    q = T.normal(rng, (batch.rows, qh, d))
    q[..., 0] = 1
    k[..., 0] = 0  # scores within about 1 of 0, by the other dims; dim 0 says how far up
    ks[:] *= np.float32(0.1)
    for s, n in enumerate(lengths):
        for j in range(n):
            page, entry = T.R.place(batch.table, s, j, need, 16)
            up = 130 <= j < 155 or 400 <= j < 640 or j == 20
            if not (up or (other and j in (35, 68, 140, 500, 700, 2900))):
                continue
            k[0, page, :, entry] = 0
            k[0, page, :, entry, 0] = 127
            ks[0, page, :, entry] = np.float32(gap * np.log(2.0) / 127 / 0.125)
            if up and j != 140:
                if scale_far is None:
                    v[0, page, :, entry] = 0
                    vs[0, page, :, entry] = 0
                else:
                    vs[0, page, :, entry] = scale_far
    pool.upload(P)
    got = T.run_attn(Q, P, pool, batch, q, 0.125)
    T.check_attn(*got, T.R.attention(q, pool.layer(0), batch.table, batch.length, batch.start,
                                     batch.max_rows, 0.125))


@pytest.mark.parametrize("heads", [(2, 1, 64), (4, 2, 128)])
@pytest.mark.parametrize("gap", [50, 65, 75, 100, 108, 112, 115, 118, 121, 124, 126, 128, 131, 140, 300])
def test_attn_weights_far_above_that_add_nothing(gpu, P, heads, gap):
    """The sum of the weights stays finite where slots of no v have scores far above the
    others': one row a sequence, and the tiles of 20 and 40 rows of a kv head."""
    for counts in (None, [10, 1, 2], [1, 1, 20]):
        for scale_far in (None, np.float32(2.0 ** -120)):
            for other in (False, True):
                far_case(gpu, P, heads, counts, gap, scale_far, other)
