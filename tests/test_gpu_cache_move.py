"""f16_cache_compact in place over lists with entries outside the cache: strictly
ascending, so negative entries come first, and behind enough of them a slot moves up
instead of down.  Held to the plain form, which reads the cache as it was."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_cache import C, Dev, move, normal  # noqa: F401 (C: the fixture)

pytestmark = pytest.mark.gpu


def ascending(rng, count, slots, negative, beyond):
    """count strictly ascending entries, `negative` of them below 0 and `beyond` at or
    past `slots`."""
    low = np.sort(rng.choice(np.arange(-3 * count - 3, 0), negative, replace=False))
    mid = np.sort(rng.permutation(slots)[:count - negative - beyond])
    high = slots + np.sort(rng.choice(np.arange(3 * count + 3), beyond, replace=False))
    return np.concatenate([low, mid, high]).astype(np.int32)


@pytest.mark.parametrize("count,slots,negative,beyond", [
    (1, 5, 1, 0), (2, 5, 1, 0), (300, 299, 1, 0), (540, 500, 40, 0), (540, 500, 40, 17),
    (256, 700, 0, 20), (257, 257, 1, 0), (700, 400, 300, 0), (700, 900, 350, 50), (900, 901, 899, 0),
    (2500, 2500, 1, 0), (4500, 2400, 2100, 0), (4500, 6000, 1000, 30)])
@pytest.mark.parametrize("kvh,d,base,per_head", [(2, 128, 0, True), (3, 64, 5, False)])
def test_in_place_with_entries_outside(gpu, C, count, slots, negative, beyond, kvh, d, base,  # noqa: F811
                                       per_head):
    layers = 2
    rng = np.random.default_rng(count + 7 * negative + d)
    seq = base + max(slots, count)
    k, v = (normal(rng, (layers, seq, kvh, d)) for _ in range(2))
    w = rng.random((layers, kvh, seq), dtype=np.float32)
    shape = (layers, kvh, count) if per_head else (count,)
    keep = np.array([ascending(rng, count, seq - base, negative, beyond)
                     for _ in range(int(np.prod(shape[:-1])))]).reshape(shape)
    assert (np.diff(keep, axis=-1) > 0).all()
    dev = Dev(gpu, C, k, v, w)
    kb = gpu.DeviceBuffer.from_array(keep)
    print(f"in place {count} of {slots}, {negative} below, {beyond} beyond", flush=True)
    C.cache_compact(dev.c, dev.c, kb, per_head, base, count)
    gpu.synchronize()
    for a, b in zip(dev.get(), move(k, v, w, k, v, w, keep, base)):
        assert np.array_equal(a, b)


def test_a_list_of_one_slot_up(gpu, C):  # noqa: F811
    """-1, 0, 1 .. 298: every slot moves one up and slot 0 stays."""
    rng = np.random.default_rng(1)
    k, v = (normal(rng, (1, 310, 2, 64)) for _ in range(2))
    dev = Dev(gpu, C, k, v)
    keep = gpu.DeviceBuffer.from_array(np.arange(-1, 299, dtype=np.int32))
    C.cache_compact(dev.c, dev.c, keep, False, 0, 300)
    gpu.synchronize()
    got = dev.get()
    for a, b in ((got[0], k), (got[1], v)):
        assert np.array_equal(a[:, 1:300], b[:, :299])
        assert np.array_equal(a[:, 0], b[:, 0]) and np.array_equal(a[:, 300:], b[:, 300:])
