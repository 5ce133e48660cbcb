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
