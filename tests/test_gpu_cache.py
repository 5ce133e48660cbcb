"""The cache operators (include/f16_cache.h) on the GPU against plain 64-bit
forms (cache_ref): every head layout, lengths around the kernels' blocks, masks
that leave rows empty, NaN and infinities in masked places, strides, guards
around the outputs, captured and replayed calls, and the operators run together
as a serving program uses them."""
from __future__ import annotations

import numpy as np
import pytest

import cache_ref as R

pytestmark = pytest.mark.gpu

GUARD = 256  # sentinel bytes before and behind an output


class Guarded:
    """A device buffer with sentinel bytes around (and in) it."""

    def __init__(self, Q, nbytes):
        self.n = nbytes
        self.buf = Q.DeviceBuffer(nbytes + 2 * GUARD)
        self.buf.fill(0xA5)
        self.ptr = self.buf.ptr + GUARD

    def get(self, dtype):
        raw = self.buf.download(np.uint8)
        assert (raw[:GUARD] == 0xA5).all() and (raw[GUARD + self.n:] == 0xA5).all(), "guard"
        return raw[GUARD:GUARD + self.n].view(dtype)


@pytest.fixture(scope="module")
def C(gpu):
    from qwen3_iree_amd import cache

    return cache


def normal(rng, shape, std=1.0):
    return (rng.standard_normal(shape, dtype=np.float32) * np.float32(std)).astype(np.float16)


def make(rng, kvh, d, length, n, slack=7, layers=1):
    """k, v [layers, max_seq, kvh, d]; NaN behind slot length + n."""
    k = normal(rng, (layers, length + n + slack, kvh, d))
    v = normal(rng, (layers, length + n + slack, kvh, d))
    k[:, length + n:] = np.nan
    v[:, length + n:] = np.inf
    return k, v


class Dev:
    """A cache on the device."""

    def __init__(self, Q, C, k, v, w=None):
        self.bufs = [Q.DeviceBuffer.from_array(a) if a is not None else None for a in (k, v, w)]
        layers, max_seq, kvh, d = k.shape
        self.shape, self.wshape = k.shape, None if w is None else w.shape
        self.c = C.Cache(self.bufs[0], self.bufs[1], max_seq, layers, kvh, d, self.bufs[2])

    def get(self):
        k, v = (b.download(np.float16).reshape(self.shape) for b in self.bufs[:2])
        w = None if self.bufs[2] is None else self.bufs[2].download(np.float32).reshape(self.wshape)
        return k, v, w


def run_tree(Q, C, k, v, q, see, length, scale, layer=0, fused=0, mask="pack", want_lse=True,
             stream=None, out_pad=0):
    """q [n, qh, d]; returns out [n, qh, d] f16 and lse."""
    n, qh, d = q.shape
    dev = Dev(Q, C, k, v)
    rows = np.full((n, qh * d + fused), np.nan, np.float16)
    rows[:, :qh * d] = q.reshape(n, -1)
    qb = Q.DeviceBuffer.from_array(rows)
    if isinstance(mask, str):
        mask = R.pack_mask(see)
    mb = None if mask is None else Q.DeviceBuffer.from_array(mask)
    stride = qh * d + out_pad
    out = Guarded(Q, 2 * (n * stride - out_pad))
    lse = Guarded(Q, 4 * n * qh)
    nbytes = C.attn_tree_workspace_bytes(dev.c, length, n, qh)
    ws = Guarded(Q, nbytes)
    ws.buf.fill(0xA5)
    print(f"attn_tree n={n} len={length} qh={qh} kvh={k.shape[2]} d={d} ws={nbytes}", flush=True)
    C.attn_tree(dev.c, layer, length, qb, qh * d + fused, qh, mb, n, scale, out.ptr, stride,
                lse.ptr if want_lse else None, ws.ptr if nbytes else None, nbytes, stream)
    Q.synchronize()
    ws.get(np.uint8)
    got = np.zeros(n * stride, np.float16)
    got[:n * stride - out_pad] = out.get(np.float16)
    got = got.reshape(n, stride)
    if out_pad:
        assert (got[:-1, qh * d:].view(np.uint16) == 0xA5A5).all()
    got_lse = lse.get(np.float32).reshape(n, qh)
    if not want_lse:
        assert (got_lse.view(np.uint32) == 0xA5A5A5A5).all()
    return got[:, :qh * d].reshape(n, qh, d), got_lse


def check_tree(got, got_lse, ref, want_lse=True):
    out, lse, out_tol, lse_tol = ref
    g = got.astype(np.float64)
    bad = ~(np.abs(g - out) <= out_tol)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:5], g[bad][:5], out[bad][:5], out_tol[bad][:5])
    if want_lse:
        assert np.array_equal(np.isneginf(got_lse), np.isneginf(lse))
        ok = np.isfinite(lse)
        assert (np.abs(got_lse.astype(np.float64)[ok] - lse[ok]) <= lse_tol[ok]).all(), \
            np.abs(got_lse[ok] - lse[ok]).max()


HEADS = [(16, 8, 128), (14, 2, 64), (9, 3, 64), (16, 1, 128), (8, 8, 128), (64, 2, 64),
         (28, 4, 128), (1, 1, 128), (32, 1, 64)]


@pytest.mark.parametrize("n,length", [
    (1, 0), (1, 1), (1, 15), (1, 31), (1, 32), (1, 33), (1, 127), (1, 1000), (1, 5000),
    (2, 0), (2, 300), (8, 64), (9, 63), (13, 1024), (16, 129), (17, 95), (32, 32), (33, 700),
    (61, 2047), (64, 1000), (65, 33), (127, 1), (128, 0), (129, 511), (200, 1500), (256, 0),
    (256, 700)])
def test_tree_lengths(gpu, C, n, length):
    rng = np.random.default_rng(1000 * n + length)
    k, v = make(rng, 8, 128, length, n)
    q = normal(rng, (n, 16, 128), 1.5)
    see = R.tree_see(R.random_tree(rng, n))
    ref = R.attention(q, k[0], v[0], see, length, 128 ** -0.5)
    check_tree(*run_tree(gpu, C, k, v, q, see, length, 128 ** -0.5), ref)


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("n,length", [(1, 77), (5, 129), (30, 400), (100, 65)])
def test_tree_head_layouts(gpu, C, heads, n, length):
    qh, kvh, d = heads
    rng = np.random.default_rng(n + 7 * length + qh)
    k, v = make(rng, kvh, d, length, n)
    q = normal(rng, (n, qh, d), 1.5)
    see = R.tree_see(R.random_tree(rng, n, pad=n // 4))
    ref = R.attention(q, k[0], v[0], see, length, d ** -0.5)
    check_tree(*run_tree(gpu, C, k, v, q, see, length, d ** -0.5, fused=2 * kvh * d, out_pad=8), ref)


@pytest.mark.parametrize("n,length", [(3, 50), (40, 0), (70, 333)])
def test_tree_padding_and_masked_values(gpu, C, n, length):
    """Padding nodes whose q, k and v hold NaN and infinities; a node whose v is
    infinite reaches the rows that see it and no other."""
    rng = np.random.default_rng(n)
    k, v = make(rng, 8, 128, length, n)
    q = normal(rng, (n, 16, 128), 1.5)
    parents = R.random_tree(rng, n)
    parents[1] = -7
    parents[n // 2] = n  # not before it
    see = R.tree_see(parents)
    dead = ~see.any(1)
    assert dead.sum() >= 2
    q[dead] = np.nan
    k[0, length:length + n][dead] = np.nan
    v[0, length:length + n][dead] = np.where(rng.random(v[0, 0].shape) < 0.5, np.inf, np.nan)
    leaf = n - 1 if not dead[n - 1] else int(np.nonzero(~dead)[0][-1])
    v[0, length + leaf, 3, 5] = np.inf
    v[0, length + leaf, 4, 6] = np.nan
    got, lse = run_tree(gpu, C, k, v, q, see, length, 128 ** -0.5)
    assert (got[dead] == 0).all() and np.isneginf(lse[dead]).all()
    sees_leaf = see[:, leaf]
    assert np.isposinf(got[sees_leaf][:, 6:8, 5]).all()
    assert np.isnan(got[sees_leaf][:, 8:10, 6]).all()
    v[0, length + leaf, 3, 5] = v[0, length + leaf, 4, 6] = 0
    q[dead] = 0
    ref = R.attention(q, k[0], v[0], see, length, 128 ** -0.5)
    got[np.ix_(sees_leaf, [6, 7], [5])] = ref[0][np.ix_(sees_leaf, [6, 7], [5])]
    got[np.ix_(sees_leaf, [8, 9], [6])] = ref[0][np.ix_(sees_leaf, [8, 9], [6])]
    check_tree(got, lse, ref)


@pytest.mark.parametrize("kvh,d,n,length,kind", [
    (64, 128, 100, 1210, "tree"), (64, 128, 100, 1210, "padded"), (64, 64, 100, 1210, "tree"),
    (64, 64, 100, 1210, "chain"), (128, 64, 65, 1405, "padded")])
def test_tree_many_rows_over_many_blocks(gpu, C, kvh, d, n, length, kind):
    """Work enough for two row tiles a wave: several row blocks, ragged at both ends."""
    qh = 256
    rng = np.random.default_rng(n + d)
    k, v = make(rng, kvh, d, length, n)
    q = normal(rng, (n, qh, d), 1.5)
    parents = R.random_tree(rng, n, pad=n // 4 if kind == "padded" else 0)
    see = np.tril(np.ones((n, n), bool)) if kind == "chain" else R.tree_see(parents)
    if kind == "padded":
        dead = ~see.any(1)
        assert dead.any()
        q[dead] = np.nan
        k[0, length:length + n][dead] = np.nan
        v[0, length:length + n][dead] = np.inf
    got = run_tree(gpu, C, k, v, q, see, length, d ** -0.5, mask=None if kind == "chain" else "pack")
    if kind == "padded":
        q[dead] = 0
        k[0, length:length + n][dead] = 0
        v[0, length:length + n][dead] = 0
    check_tree(*got, R.attention(q, k[0], v[0], see, length, d ** -0.5))


@pytest.mark.parametrize("n,length", [(1, 40), (33, 200), (90, 31)])
def test_chain_without_a_mask(gpu, C, n, length):
    rng = np.random.default_rng(n)
    k, v = make(rng, 8, 128, length, n)
    q = normal(rng, (n, 16, 128), 1.5)
    see = np.tril(np.ones((n, n), bool))
    ref = R.attention(q, k[0], v[0], see, length, 128 ** -0.5)
    got = run_tree(gpu, C, k, v, q, see, length, 128 ** -0.5, mask=None)
    check_tree(*got, ref)
    same = run_tree(gpu, C, k, v, q, see, length, 128 ** -0.5)
    assert np.array_equal(got[0], same[0]) and np.array_equal(got[1], same[1])


def test_any_mask_and_bits_behind_n(gpu, C):
    rng = np.random.default_rng(5)
    n, length = 45, 70
    k, v = make(rng, 8, 128, length, n)
    q = normal(rng, (n, 16, 128), 1.5)
    see = rng.random((n, n)) < 0.3
    see[[0, 17, 44]] = False
    mask = R.pack_mask(see)
    mask[:, -1] |= np.uint32(0xFFFFFFFF << (n % 32) & 0xFFFFFFFF)
    ref = R.attention(q, k[0], v[0], see, length, 0.1)
    check_tree(*run_tree(gpu, C, k, v, q, see, length, 0.1, mask=mask), ref)


@pytest.mark.parametrize("n,length", [(4, 100), (40, 300)])
def test_large_and_equal_scores(gpu, C, n, length):
    """Scores far apart, and rows where one early or late key takes all."""
    rng = np.random.default_rng(9)
    k, v = make(rng, 8, 128, length, n)
    q = normal(rng, (n, 16, 128), 12.0)
    k[0, 0] *= np.float16(6)
    k[0, length - 1, 3] *= np.float16(9)
    k[0, 10:20] = k[0, 10]
    see = R.tree_see(R.random_tree(rng, n))
    ref = R.attention(q, k[0], v[0], see, length, 128 ** -0.5)
    check_tree(*run_tree(gpu, C, k, v, q, see, length, 128 ** -0.5), ref)


def test_many_small_weights_beside_a_large_one(gpu, C):
    """One weight of about 1 and 16,000 of about 2^-18: the small ones together
    still count."""
    n, length = 1, 16000
    k = np.zeros((1, length + 8, 1, 128), np.float16)
    v = np.full((1, length + 8, 1, 128), 1.0, np.float16)
    q = np.full((n, 2, 128), 1.0, np.float16)
    k[0, 5, 0] = np.float16(12.476 / 128)
    v[0, 5] = 0
    see = np.ones((1, 1), bool)
    ref = R.attention(q, k[0], v[0], see, length, 1.0)
    assert 0.01 < ref[0].max() < 0.1
    check_tree(*run_tree(gpu, C, k, v, q, see, length, 1.0), ref)


def test_tree_layers_and_no_lse(gpu, C):
    rng = np.random.default_rng(3)
    k, v = make(rng, 2, 64, 90, 6, layers=3)
    q = normal(rng, (6, 4, 64))
    see = R.tree_see([-1, 0, 0, 1, -1, 4])
    for layer in (0, 2):
        ref = R.attention(q, k[layer], v[layer], see, 90, 0.125)
        got = run_tree(gpu, C, k, v, q, see, 90, 0.125, layer=layer, want_lse=False)
        check_tree(*got, ref, want_lse=False)


def test_offsets_past_32_bits(gpu, C):
    """A cache of 4.3 GB a side: zero keys and values but for the last slots."""
    n, length, kvh, d = 3, (1 << 21) + 1500, 8, 128
    max_seq = length + n
    rng = np.random.default_rng(1)
    kb, vb = gpu.DeviceBuffer(max_seq * kvh * d * 2), gpu.DeviceBuffer(max_seq * kvh * d * 2)
    wb = gpu.DeviceBuffer(kvh * max_seq * 4)
    for b in (kb, vb, wb):
        b.fill(0)
    tail = 40
    k, v = normal(rng, (tail, kvh, d)), normal(rng, (tail, kvh, d), 1000.0)
    at = (max_seq - tail) * kvh * d * 2
    kb.upload(k, at)
    vb.upload(v, at)
    q = normal(rng, (n, 16, d), 3.0)
    qb = gpu.DeviceBuffer.from_array(q)
    c = C.Cache(kb, vb, max_seq, 1, kvh, d, wb)
    out, lse = gpu.DeviceBuffer(q.nbytes), gpu.DeviceBuffer(n * 16 * 4)
    ws = gpu.DeviceBuffer(C.attn_tree_workspace_bytes(c, length, n, 16))
    C.attn_tree(c, 0, length, qb, 16 * d, 16, None, n, d ** -0.5, out, 16 * d, lse, ws, ws.nbytes)
    C.attn_weights_add(c, length, qb, 0, 16 * d, 16, lse, 0, n, None, n, d ** -0.5)
    gpu.synchronize()
    got = out.download(np.float16).reshape(n, 16, d).astype(np.float64)
    got_lse = lse.download(np.float32).reshape(n, 16)
    w = wb.download(np.float32).reshape(kvh, max_seq)
    zeros = max_seq - tail
    sums = np.zeros((kvh, tail))
    for i in range(n):
        m = tail - n + i + 1
        s, e = R.scores(q[i:i + 1], k[:m], d ** -0.5)
        tot = zeros + np.exp(s[0]).sum(-1)
        assert np.abs(got_lse[i] - np.log(tot)).max() < 2e-5 * 15
        for h in range(16):
            p = np.exp(s[0, h]) / tot[h]
            want = p @ v[:m, h // 2].astype(np.float64)
            # N / 16 chains of equal weights: (N / 16 + 48) 2^-24 relative
            tol = (zeros / 16 + 48) * R.EPS * (p @ np.abs(v[:m, h // 2].astype(np.float64))) + \
                2.0 ** -11 * np.abs(want) + 2.0 ** -25
            assert (np.abs(got[i, h] - want) <= tol).all()
            sums[h // 2, :m] += np.exp(s[0, h] - got_lse[i, h])
    assert np.allclose(w[:, zeros:], sums, rtol=1e-5, atol=0)
    each = np.exp(-got_lse.astype(np.float64)).reshape(n, kvh, 2).sum((0, 2))
    assert np.allclose(w[:, [0, 5, 1 << 20, zeros - 1]], each[:, None], rtol=1e-5, atol=0)
    # the last slots to the front: rows past 2^31 elements into a small cache
    keep = gpu.DeviceBuffer.from_array(np.arange(max_seq - tail, max_seq, dtype=np.int32))
    small = Dev(gpu, C, np.zeros((1, tail, kvh, d), np.float16),
                np.zeros((1, tail, kvh, d), np.float16), np.zeros((1, kvh, tail), np.float32))
    C.cache_compact(c, small.c, keep, False, 0, tail)
    gpu.synchronize()
    sk, sv, sw = small.get()
    assert np.array_equal(sk[0], k) and np.array_equal(sv[0], v)
    assert np.array_equal(sw[0], w[:, zeros:])
    for b in (kb, vb, wb):
        b.free()


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 64, 100, 255, 256])
@pytest.mark.parametrize("kind", ["random", "chain", "star", "bad"])
def test_tree_mask(gpu, C, n, kind):
    rng = np.random.default_rng(n)
    parents = R.random_tree(rng, n, pad=n // 5)
    if kind == "chain":
        parents = np.arange(-1, n - 1, dtype=np.int32)
    elif kind == "star":
        parents = np.full(n, -1, np.int32)
    elif kind == "bad":
        bad = rng.random(n) < 0.1
        parents[bad] = rng.choice([-2, -(2 ** 31), n, 2 ** 31 - 1, 300], int(bad.sum()))
        parents[n - 1] = n - 1
    see = R.tree_see(parents)
    words = (n + 31) // 32
    pb = gpu.DeviceBuffer.from_array(parents)
    mask, depth = Guarded(gpu, 4 * n * words), Guarded(gpu, 4 * n)
    C.tree_mask(pb, n, mask.ptr, depth.ptr)
    gpu.synchronize()
    assert np.array_equal(mask.get(np.uint32).reshape(n, words), R.pack_mask(see))
    assert np.array_equal(depth.get(np.int32), see.sum(1) - 1)
    C.tree_mask(pb, n, mask.ptr, None)
    gpu.synchronize()
    assert np.array_equal(mask.get(np.uint32).reshape(n, words), R.pack_mask(see))


# ------------------------------------------------------------- weights ----

@pytest.mark.parametrize("heads", [(16, 8, 128), (14, 2, 64), (64, 2, 64), (16, 1, 128), (9, 3, 64)])
@pytest.mark.parametrize("n,nodes,length,layers", [
    (1, 1, 0, 1), (1, 1, 33, 2), (1, 5, 1000, 3), (5, 24, 300, 2), (17, 17, 15, 1), (33, 40, 128, 1),
    (256, 256, 100, 1), (100, 120, 0, 2)])
def test_weights_add(gpu, C, heads, n, nodes, length, layers):
    qh, kvh, d = heads
    rng = np.random.default_rng(n + 3 * length + qh)
    k, v = make(rng, kvh, d, length, n, layers=layers)
    w = rng.random((layers, kvh, k.shape[1]), dtype=np.float32)
    w[:, :, length:] = np.nan  # new slots hold nothing yet
    q = normal(rng, (layers, nodes, qh, d), 1.5)
    path = np.sort(rng.permutation(nodes)[:n]).astype(np.int32)
    scale = d ** -0.5
    lse = rng.standard_normal((layers, nodes, qh), dtype=np.float32) + 6
    if n > 4:
        path[2], path[3] = -1, nodes  # out of range: add nothing
        lse[:, path[4], 1] = -np.inf
    dev = Dev(gpu, C, k, v, w)
    qb, lb = gpu.DeviceBuffer.from_array(q), gpu.DeviceBuffer.from_array(lse)
    pb = gpu.DeviceBuffer.from_array(path)
    print(f"weights n={n} nodes={nodes} len={length} heads={heads}", flush=True)
    C.attn_weights_add(dev.c, length, qb, nodes * qh * d, qh * d, qh, lb, nodes * qh, nodes, pb, n,
                       scale)
    gpu.synchronize()
    got = dev.get()[2]
    for l in range(layers):
        ref, tol = R.weights_add(w[l], q[l], lse[l], k[l], path, length, n, scale)
        S = length + n
        assert (np.abs(got[l, :, :S] - ref[:, :S]) <= tol[:, :S]).all(), \
            (np.abs(got[l, :, :S] - ref[:, :S]) / tol[:, :S]).max()
        assert np.array_equal(got[l, :, S:], w[l, :, S:], equal_nan=True)


@pytest.mark.parametrize("heads", [(16, 8, 128), (64, 2, 64), (16, 1, 128)])
@pytest.mark.parametrize("layers,length,n", [(40, 250, 70), (2, 33, 130), (300, 100, 40)])
def test_weights_add_many_rows_and_layers(gpu, C, heads, layers, length, n):
    """Above 64 rows, on both sides of the number of workgroups where the kernel
    changes; a few layers are checked."""
    qh, kvh, d = heads
    rng = np.random.default_rng(layers + n)
    k, v = make(rng, kvh, d, length, n, layers=layers)
    w = rng.random((layers, kvh, k.shape[1]), dtype=np.float32)
    nodes = n + 5
    q = normal(rng, (layers, nodes, qh, d), 1.5)
    path = np.sort(rng.permutation(nodes)[:n]).astype(np.int32)
    lse = rng.standard_normal((layers, nodes, qh), dtype=np.float32) + 6
    path[n // 2], lse[:, path[3], 0] = nodes, -np.inf
    dev = Dev(gpu, C, k, v, w)
    qb, lb = gpu.DeviceBuffer.from_array(q), gpu.DeviceBuffer.from_array(lse)
    pb = gpu.DeviceBuffer.from_array(path)
    print(f"weights n={n} layers={layers} len={length} heads={heads}", flush=True)
    C.attn_weights_add(dev.c, length, qb, nodes * qh * d, qh * d, qh, lb, nodes * qh, nodes, pb, n,
                       d ** -0.5)
    gpu.synchronize()
    got = dev.get()[2]
    for l in sorted({0, 1, layers // 2, layers - 1}):
        ref, tol = R.weights_add(w[l], q[l], lse[l], k[l], path, length, n, d ** -0.5)
        S = length + n
        assert (np.abs(got[l, :, :S] - ref[:, :S]) <= tol[:, :S]).all()
        assert np.array_equal(got[l, :, S:], w[l, :, S:], equal_nan=True)


def test_weights_without_a_path_and_row_stride(gpu, C):
    rng = np.random.default_rng(2)
    n, length, qh, kvh, d = 6, 50, 4, 2, 64
    k, v = make(rng, kvh, d, length, n)
    w = np.zeros((1, kvh, k.shape[1]), np.float32)
    rows = normal(rng, (n, qh * d + 128), 1.5)
    q = rows[:, :qh * d].reshape(n, qh, d)
    rows[:, qh * d:] = np.nan
    lse = rng.standard_normal((n, qh), dtype=np.float32) + 4
    dev = Dev(gpu, C, k, v, w)
    qb, lb = gpu.DeviceBuffer.from_array(rows), gpu.DeviceBuffer.from_array(lse)
    C.attn_weights_add(dev.c, length, qb, 0, qh * d + 128, qh, lb, 0, n, None, n, 0.125)
    gpu.synchronize()
    ref, tol = R.weights_add(w[0], q, lse, k[0], np.arange(n), length, n, 0.125)
    assert (np.abs(dev.get()[2][0] - ref) <= tol)[:, :length + n].all()


# ------------------------------------------------------------- eviction ----

@pytest.mark.parametrize("length,budget,sinks,recent", [
    (1, 1, 0, 0), (2, 1, 0, 0), (2, 1, 1, 0), (2, 1, 0, 1), (5, 5, 1, 1), (33, 20, 4, 8),
    (600, 512, 4, 64), (1024, 1, 0, 0), (1025, 1024, 0, 0), (3000, 1500, 0, 1500),
    (5000, 1250, 16, 300), (20000, 7000, 3, 11)])
@pytest.mark.parametrize("kind", ["random", "ties", "special"])
def test_select(gpu, C, length, budget, sinks, recent, kind):
    layers, kvh = 2, 3
    rng = np.random.default_rng(length + budget)
    max_seq = length + 5
    w = np.exp(2 * rng.standard_normal((layers, kvh, max_seq))).astype(np.float32)
    if kind == "ties":
        w = rng.integers(0, 4, w.shape).astype(np.float32)
        w[0, 0] = 1.0
    elif kind == "special":
        pick = rng.random(w.shape)
        for i, x in enumerate([np.nan, np.inf, -np.inf, 0.0, -0.0, -1.0, 1e-42, -np.nan, 1e30]):
            w[(pick > 0.1 * i) & (pick <= 0.1 * (i + 1))] = x
    w[:, :, length:] = np.inf
    wb = gpu.DeviceBuffer.from_array(w)
    c = C.Cache(None, None, max_seq, layers, kvh, 128, wb)
    keep = Guarded(gpu, 4 * layers * kvh * budget)
    print(f"select {length} -> {budget} ({sinks}, {recent}) {kind}", flush=True)
    C.cache_select(c, length, budget, sinks, recent, keep.ptr)
    gpu.synchronize()
    got = keep.get(np.int32).reshape(layers, kvh, budget)
    assert np.array_equal(got, R.select(w, length, budget, sinks, recent))


@pytest.mark.parametrize("slots", [1023, 1025, 4096, 4097, 16384, 16385, 20481, 49152, 49153, 70000])
@pytest.mark.parametrize("kind", ["random", "ties", "equal", "nan", "mixed"])
def test_select_on_both_sides_of_each_size(gpu, C, slots, kind):
    """Slots between the first and last kept ones where the number a thread holds
    changes; budgets of one, about a third, all but one and all of them."""
    sinks, recent, kvh = 3, 7, 2
    length = sinks + slots + recent
    rng = np.random.default_rng(slots)
    w = np.exp(2 * rng.standard_normal((1, kvh, length + 1))).astype(np.float32)
    if kind == "ties":
        w = rng.integers(-1, 2, w.shape).astype(np.float32)
    elif kind == "equal":
        w[:] = 0.25
    elif kind == "nan":
        w[:] = np.nan
    elif kind == "mixed":
        w[rng.random(w.shape) < 0.5] = np.nan
        w[rng.random(w.shape) < 0.2] = -np.inf
    w[:, :, length:] = np.inf
    wb = gpu.DeviceBuffer.from_array(w)
    c = C.Cache(None, None, length + 1, 1, kvh, 128, wb)
    print(f"select of {slots} {kind}", flush=True)
    for middle in (1, slots // 3, slots - 1, slots):
        budget = sinks + middle + recent
        keep = Guarded(gpu, 4 * kvh * budget)
        C.cache_select(c, length, budget, sinks, recent, keep.ptr)
        gpu.synchronize()
        got = keep.get(np.int32).reshape(1, kvh, budget)
        assert np.array_equal(got, R.select(w, length, budget, sinks, recent)), middle


def move(k, v, w, k_to, v_to, w_to, keep, base):
    """numpy form of cache_compact; keep [layers, kvh, count] or [count]."""
    layers, seq, kvh, _ = k.shape
    k_to, v_to = k_to.copy(), v_to.copy()
    w_to = None if w_to is None else w_to.copy()
    for l in range(layers):
        for h in range(kvh):
            ks = keep if keep.ndim == 1 else keep[l, h]
            for j, p in enumerate(ks):
                if 0 <= p < seq - base:
                    k_to[l, base + j, h] = k[l, base + p, h]
                    v_to[l, base + j, h] = v[l, base + p, h]
                    if w_to is not None and w is not None:
                        w_to[l, h, base + j] = w[l, h, base + p]
    return k_to, v_to, w_to


@pytest.mark.parametrize("kvh,d", [(8, 128), (3, 64)])
@pytest.mark.parametrize("length,count,base", [(1, 1, 0), (40, 31, 0), (300, 33, 0), (700, 256, 0),
                                               (700, 699, 0), (1300, 1000, 0), (90, 7, 64)])
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("per_head", [True, False])
def test_compact(gpu, C, kvh, d, length, count, base, in_place, per_head):
    layers = 2
    rng = np.random.default_rng(length + count + base)
    seq = length + 9
    k, v = (normal(rng, (layers, seq, kvh, d)) for _ in range(2))
    w = rng.random((layers, kvh, seq), dtype=np.float32)
    shape = (layers, kvh, count) if per_head else (count,)
    lists = [np.sort(rng.permutation(length - base)[:count]) for _ in range(int(np.prod(shape[:-1])))]
    keep = np.array(lists, np.int32).reshape(shape)
    if not in_place:  # any order, repeats, and entries outside the cache
        flat = keep.reshape(-1)
        rng.shuffle(flat)
        flat[0] = flat[-1]
        if count > 20:
            flat[3], flat[7], flat[11] = -1, seq - base, 2 ** 31 - 1
    src = Dev(gpu, C, k, v, w)
    if in_place:
        dst, to = src, (k, v, w)
    else:
        n2 = base + count + 3
        to = (normal(rng, (layers, n2, kvh, d)), normal(rng, (layers, n2, kvh, d)),
              rng.random((layers, kvh, n2), dtype=np.float32))
        dst = Dev(gpu, C, *to)
    kb = gpu.DeviceBuffer.from_array(keep)
    print(f"compact {length}/{count}+{base} kvh={kvh} d={d} {in_place} {per_head}", flush=True)
    C.cache_compact(src.c, dst.c, kb, per_head, base, count)
    gpu.synchronize()
    want = move(k, v, w, *to, keep, base)
    for a, b in zip(dst.get(), want):
        assert np.array_equal(a, b)
    if not in_place:
        for a, b in zip(src.get(), (k, v, w)):
            assert np.array_equal(a, b)


def test_compact_without_weights_and_nothing(gpu, C):
    rng = np.random.default_rng(0)
    k, v = (normal(rng, (2, 50, 2, 64)) for _ in range(2))
    src = Dev(gpu, C, k, v)
    keep = gpu.DeviceBuffer.from_array(np.array([0, 3, 9, 40], np.int32))
    C.cache_compact(src.c, src.c, None, False, 5, 0)
    C.cache_compact(src.c, src.c, keep, False, 5, 4)
    gpu.synchronize()
    want = move(k, v, None, k, v, None, np.array([0, 3, 9, 40]), 5)
    got = src.get()
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


def test_many_layers_and_heads(gpu, C):
    """The most layers and a wide row of heads: more (layer, head) pairs than a
    grid's second dimension holds."""
    layers, kvh, d, seq = 1024, 80, 64, 4
    rng = np.random.default_rng(6)
    k, v = (normal(rng, (layers, seq, kvh, d)) for _ in range(2))
    w = rng.random((layers, kvh, seq), dtype=np.float32)
    dev = Dev(gpu, C, k, v, w)
    keep = gpu.DeviceBuffer(4 * layers * kvh * 2)
    C.cache_select(dev.c, 4, 2, 0, 0, keep)
    C.cache_compact(dev.c, dev.c, keep, True, 0, 2)
    gpu.synchronize()
    want = R.select(w, 4, 2, 0, 0)
    assert np.array_equal(keep.download(np.int32).reshape(want.shape), want)
    li, hi = np.arange(layers)[:, None, None], np.arange(kvh)[None, :, None]
    gk, gv, gw = dev.get()
    assert np.array_equal(gk[:, :2], k[li, want, hi].transpose(0, 2, 1, 3))
    assert np.array_equal(gv[:, :2], v[li, want, hi].transpose(0, 2, 1, 3))
    assert np.array_equal(gw[:, :, :2], np.take_along_axis(w, want.astype(np.int64), 2))
    assert np.array_equal(gk[:, 2:], k[:, 2:]) and np.array_equal(gw[:, :, 2:], w[:, :, 2:])
    q = normal(rng, (layers, 1, kvh, d))
    lse = np.full((layers, 1, kvh), 3.0, np.float32)
    qb, lb = gpu.DeviceBuffer.from_array(q), gpu.DeviceBuffer.from_array(lse)
    C.attn_weights_add(dev.c, 2, qb, kvh * d, kvh * d, kvh, lb, kvh, 1, None, 1, 0.125)
    gpu.synchronize()
    got = dev.get()[2]
    for l in (0, 500, 1023):
        ref, tol = R.weights_add(gw[l], q[l], lse[l], gk[l], [0], 2, 1, 0.125)
        assert (np.abs(got[l] - ref) <= tol)[:, :3].all()
        assert np.array_equal(got[l, :, 3], gw[l, :, 3])


# ------------------------------------------------------ vocabulary rows ----

def run_vocab(Q, w, x, logits=True, stream=None):
    n, rows = x.shape[0], w.shape[0]
    wb, xb = Q.DeviceBuffer.from_array(w), Q.DeviceBuffer.from_array(x)
    ws = Guarded(Q, Q.gemm_argmax_workspace_bytes(n))
    tok, lg = Guarded(Q, 4 * n), Guarded(Q, 2 * n * rows)
    print(f"gemm_argmax rows={rows} n={n}", flush=True)
    Q.f16_gemm_argmax(wb, rows, xb, n, lg.ptr if logits else None, tok.ptr, ws.ptr, stream)
    Q.synchronize()
    ws.get(np.uint8)
    got = lg.get(np.float16).reshape(n, rows)
    if not logits:
        assert (got.view(np.uint16) == 0xA5A5).all()
    return got, tok.get(np.int32)


def first_max(row):
    v = np.where(np.isnan(row), -np.inf, row.astype(np.float32))
    return int(np.argmax(v)) if v.max() > -np.inf else -1


@pytest.mark.parametrize("rows", [1, 3, 16, 63, 64, 65, 127, 129, 1000, 4099])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 33, 64, 65, 130, 256])
def test_vocab_rows(gpu, rows, n):
    rng = np.random.default_rng(rows + n)
    w, x = normal(rng, (rows, 1024), 0.02), normal(rng, (n, 1024))
    got, tok = run_vocab(gpu, w, x)
    ref = x.astype(np.float64) @ w.astype(np.float64).T
    mag = np.abs(x.astype(np.float64)) @ np.abs(w.astype(np.float64)).T
    # 1024 exact products summed in f32 in any order, one rounding to f16
    tol = 1024 * R.EPS * mag + 2.0 ** -11 * np.abs(ref) + 2.0 ** -25
    assert (np.abs(got.astype(np.float64) - ref) <= tol).all()
    assert np.array_equal(tok, [first_max(r) for r in got])
    _, tok2 = run_vocab(gpu, w, x, logits=False)
    assert np.array_equal(tok, tok2)


def test_vocab_ties_nan_and_infinities(gpu):
    rng = np.random.default_rng(4)
    rows, n = 5000, 40
    w = normal(rng, (rows, 1024), 0.02)
    x = normal(rng, (n, 1024))
    w[[7, 70, 4999]] = w[7]
    x[0] = (w[7].astype(np.float32) * 50).astype(np.float16)  # three equal maxima
    x[1] = np.nan
    x[2, 0] = np.inf
    x[3] = 0  # all zero: the first row
    w[100] = np.nan
    got, tok = run_vocab(gpu, w, x)
    assert np.array_equal(tok, [first_max(r) for r in got])
    assert tok[0] == 7 and tok[1] == -1 and tok[3] == 0
    assert np.isnan(got[:, 100]).all() and np.isnan(got[1]).all()


def test_vocab_one_row_agrees_with_the_single_row_call(gpu):
    rng = np.random.default_rng(8)
    w = normal(rng, (3001, 1024), 0.02)
    x = (normal(rng, (3, 1024)).astype(np.float32) + 20 * w[[5, 2999, 77]]).astype(np.float16)
    _, tok = run_vocab(gpu, w, x)
    assert list(tok) == [5, 2999, 77]
    wb = gpu.DeviceBuffer.from_array(w)
    one, ws = gpu.DeviceBuffer(16), gpu.DeviceBuffer(gpu.vocab_workspace_bytes())
    gpu.vocab_workspace_reset(ws)
    for i in range(3):
        xb = gpu.DeviceBuffer.from_array(x[i])
        gpu.f16_gemv_argmax_rows(wb, 3001, xb, None, one, ws)
        gpu.synchronize()
        assert int(one.download(np.int32, 1)[0]) == tok[i]


# ------------------------------------------------------ used as a whole ----

class Serve:
    """Buffers of a small serving loop, and the loop's steps."""

    def __init__(self, Q, C, rng, n, length, qh=16, kvh=8, d=128, layers=2):
        self.Q, self.C, self.rng = Q, C, rng
        self.n, self.qh, self.kvh, self.d, self.layers = n, qh, kvh, d, layers
        self.k, self.v = make(rng, kvh, d, length, n, slack=40, layers=layers)
        self.w = rng.random((layers, kvh, self.k.shape[1]), dtype=np.float32)
        self.dev = Dev(Q, C, self.k, self.v, self.w)
        self.parents = R.random_tree(rng, n, pad=1)
        self.q = normal(rng, (layers, n, qh, d), 1.5)
        words = (n + 31) // 32
        self.pb, self.qb = Q.DeviceBuffer.from_array(self.parents), Q.DeviceBuffer.from_array(self.q)
        self.mask, self.depth = Q.DeviceBuffer(4 * n * words), Q.DeviceBuffer(4 * n)
        self.out, self.lse = Q.DeviceBuffer(self.q.nbytes), Q.DeviceBuffer(4 * layers * n * qh)
        self.ws = Q.DeviceBuffer(C.attn_tree_workspace_bytes(self.dev.c, self.k.shape[1] - n, n, qh))
        self.keep = Q.DeviceBuffer(4 * layers * kvh * self.k.shape[1])
        self.path = Q.DeviceBuffer(4 * n)

    def attend(self, length, stream=None):
        C, n, qh, d = self.C, self.n, self.qh, self.d
        C.tree_mask(self.pb, n, self.mask, self.depth, stream)
        for l in range(self.layers):
            C.attn_tree(self.dev.c, l, length, self.qb.ptr + 2 * l * n * qh * d, qh * d, qh, self.mask,
                        n, d ** -0.5, self.out.ptr + 2 * l * n * qh * d, qh * d,
                        self.lse.ptr + 4 * l * n * qh, self.ws, self.ws.nbytes, stream)

    def got(self):
        return (self.out.download(np.float16).reshape(self.q.shape),
                self.lse.download(np.float32).reshape(self.layers, self.n, self.qh))

    def check(self, length):
        got, lse = self.got()
        see = R.tree_see(self.parents)
        for l in range(self.layers):
            ref = R.attention(self.q[l], self.k[l], self.v[l], see, length, self.d ** -0.5)
            check_tree(got[l], lse[l], ref)
        return lse


@pytest.mark.parametrize("heads", [(16, 8, 128), (14, 2, 64)])
def test_verify_commit_weigh_evict_verify(gpu, C, heads):
    """The operators as a serving program runs them, on one stream with nothing
    waited for between: a tree, its accepted path moved to the front, the weights
    of that path, eviction in place, and the next tree over what is left."""
    rng = np.random.default_rng(12)
    n, length = 11, 150
    S = Serve(gpu, C, rng, n, length, *heads)
    stream = gpu.Stream()
    path = np.array([0, 2, 5, 9], np.int32)
    S.path.upload(path)
    m, budget, sinks, recent = len(path), 100, 4, 30
    qh, d = S.qh, S.d
    S.attend(length, stream)
    C.cache_compact(S.dev.c, S.dev.c, S.path, False, length, m, stream)
    C.attn_weights_add(S.dev.c, length, S.qb, n * qh * d, qh * d, qh, S.lse, n * qh, n, S.path, m,
                       d ** -0.5, stream)
    C.cache_select(S.dev.c, length + m, budget, sinks, recent, S.keep, stream)
    C.cache_compact(S.dev.c, S.dev.c, S.keep, True, 0, budget, stream)
    stream.synchronize()
    lse = S.check(length)
    # the path's k and v, but not its weights, which weights_add replaces
    S.k, S.v, _ = move(S.k, S.v, None, S.k, S.v, None, path, length)
    _, _, w_dev = S.dev.get()
    keep = S.keep.download(np.int32, S.layers * S.kvh * budget).reshape(S.layers, S.kvh, budget)
    for l in range(S.layers):
        ref, tol = R.weights_add(S.w[l], S.q[l], lse[l], S.k[l], path, length, m, d ** -0.5)
        S.w[l, :, :length + m] = ref[:, :length + m]
        rows = np.take_along_axis(ref, keep[l].astype(np.int64), 1)
        assert (np.abs(w_dev[l, :, :budget] - rows) <= np.take_along_axis(tol, keep[l].astype(np.int64), 1)).all()
        # what was kept is at least as heavy as what was not, up to the bound
        for h in range(S.kvh):
            mid = np.setdiff1d(np.arange(sinks, length + m - recent), keep[l, h])
            inside = keep[l, h, sinks:budget - recent]
            assert ref[h, inside].min() >= ref[h, mid].max() - 2 * tol[h].max()
    S.k, S.v, _ = move(S.k, S.v, None, S.k, S.v, None, keep, 0)
    got = S.dev.get()
    assert np.array_equal(got[0][:, :budget], S.k[:, :budget])
    assert np.array_equal(got[1][:, :budget], S.v[:, :budget])
    # the next tree, written behind what is left
    for a, b in ((S.k, S.dev.bufs[0]), (S.v, S.dev.bufs[1])):
        a[:, budget:budget + n] = normal(rng, a[:, :n].shape)
        b.upload(a)
    S.attend(budget, stream)
    stream.synchronize()
    S.check(budget)


def test_captured_and_replayed(gpu, C):
    """One graph of the whole round, replayed over changing inputs with eager
    calls between; every replay gives the eager result's bits."""
    rng = np.random.default_rng(21)
    n, length = 20, 333
    S = Serve(gpu, C, rng, n, length)
    w, x = normal(rng, (700, 1024), 0.02), normal(rng, (n, 1024))
    wb, xb = gpu.DeviceBuffer.from_array(w), gpu.DeviceBuffer.from_array(x)
    tok, lg = gpu.DeviceBuffer(4 * n), gpu.DeviceBuffer(2 * n * 700)
    vws = gpu.DeviceBuffer(gpu.gemm_argmax_workspace_bytes(n))
    stream = gpu.Stream()
    qh, d = S.qh, S.d

    def work():
        S.attend(length, stream)
        gpu.f16_gemm_argmax(wb, 700, xb, n, lg, tok, vws, stream)
        C.attn_weights_add(S.dev.c, length, S.qb, n * qh * d, qh * d, qh, S.lse, n * qh, n, None, n,
                           d ** -0.5, stream)
        C.cache_select(S.dev.c, length + n, 200, 4, 16, S.keep, stream)

    def state():
        stream.synchronize()
        return [S.out.download(np.uint16), S.lse.download(np.uint32), tok.download(np.int32),
                lg.download(np.uint16), S.dev.bufs[2].download(np.uint32),
                S.keep.download(np.int32, S.layers * S.kvh * 200)]

    def reset(step):
        r = np.random.default_rng(step)
        S.qb.upload(normal(r, S.q.shape, 1.5))
        S.pb.upload(R.random_tree(r, n, pad=step))
        xb.upload(normal(r, x.shape))
        S.dev.bufs[2].upload(S.w)

    graph = gpu.Graph(stream, work)
    for step in range(4):
        reset(step)
        work()
        eager = state()
        reset(step)
        graph.launch(stream)
        for a, b in zip(eager, state()):
            assert np.array_equal(a, b)
    graph.destroy()


def test_two_streams_at_once(gpu, C):
    rng = np.random.default_rng(31)
    a, b = Serve(gpu, C, rng, 30, 900), Serve(gpu, C, rng, 7, 2000)
    sa, sb = gpu.Stream(), gpu.Stream()
    for _ in range(3):
        a.attend(900, sa)
        b.attend(2000, sb)
    sa.synchronize()
    sb.synchronize()
    a.check(900)
    b.check(2000)


def test_same_inputs_same_bits(gpu, C):
    rng = np.random.default_rng(41)
    S = Serve(gpu, C, rng, 61, 4000)
    S.attend(4000)
    gpu.synchronize()
    first = S.got()
    S.ws.fill(0xFF)
    S.attend(4000)
    gpu.synchronize()
    for x, y in zip(first, S.got()):
        assert np.array_equal(x.view(np.uint8), y.view(np.uint8))
