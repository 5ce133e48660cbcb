"""The paged cache's operators (include/kv_pages.h) on the GPU against plain 64-bit forms
(pages_ref): page types and sizes, head layouts, ragged batches, lengths from none on,
slots that stand for nothing, NaN and infinities in places a row does not see, strides,
guards, rows that belong to nobody, captured calls, and the operators run together."""
from __future__ import annotations

import numpy as np
import pytest

import pages_ref as R

pytestmark = pytest.mark.gpu

GUARD = 256


@pytest.fixture(scope="module")
def P(gpu):
    from qwen3_iree_amd import pages

    return pages


class Guarded:
    """A device buffer with sentinel bytes around (and in) it."""

    def __init__(self, Q, nbytes, fill=0xA5):
        self.n = nbytes
        self.buf = Q.DeviceBuffer(nbytes + 2 * GUARD)
        self.buf.fill(0xA5)
        if fill == 0:
            self.buf.upload(np.zeros(nbytes, np.uint8), GUARD)
        self.ptr = self.buf.ptr + GUARD

    def get(self, dtype):
        raw = self.buf.download(np.uint8)
        assert (raw[:GUARD] == 0xA5).all() and (raw[GUARD + self.n:] == 0xA5).all(), "guard"
        return raw[GUARD:GUARD + self.n].view(dtype)


def normal(rng, shape, std=1.0):
    return (rng.standard_normal(shape, dtype=np.float32) * np.float32(std)).astype(np.float16)


def quantised(x):
    x = x.astype(np.float32)
    scale = (np.abs(x).max(-1) / 127).astype(np.float32)
    safe = np.where(scale > 0, scale, 1)
    return np.rint(x / safe[..., None]).astype(np.int8), scale


class Pool:
    """Pages of every layer on host and device."""

    def __init__(self, Q, P, rng, layers, pages, page, kvh, d, bits, fill=None):
        self.Q, self.bits, self.shape = Q, bits, (layers, pages, kvh, page, d)
        k, v = (normal(rng, self.shape) for _ in range(2))
        self.scales = [None, None]
        if bits == 8:
            k, ks = quantised(k)
            v, vs = quantised(v)
            self.scales = [ks, vs]
        self.host = [k, v]
        self.upload(P)

    def upload(self, P):
        layers, pages, kvh, page, d = self.shape
        self.dev = [self.Q.DeviceBuffer.from_array(x) for x in self.host]
        self.dev_scale = [None if x is None else self.Q.DeviceBuffer.from_array(x) for x in self.scales]
        self.c = P.Pages(self.dev[0], self.dev[1], pages, page, layers, kvh, d,
                         self.dev_scale[0], self.dev_scale[1])

    def layer(self, l):
        return (self.host[0][l], self.host[1][l], *(None if x is None else x[l] for x in self.scales))

    def get(self):
        dtype = np.int8 if self.bits == 8 else np.float16
        data = [b.download(dtype).reshape(self.shape) for b in self.dev]
        return data, [None if b is None else b.download(np.float32).reshape(self.shape[:-1])
                      for b in self.dev_scale]


class Batch:
    """Sequences of given lengths and new rows over random pages of a pool."""

    def __init__(self, Q, P, rng, pool, lengths, counts=None, rows=None, spare=0, start=None,
                 max_rows=None, wide=None):
        page, pages = pool.shape[3], pool.shape[1]
        used = [(max(n, 0) + page - 1) // page for n in lengths]
        wide = wide or max(1, max(used) + spare)
        used = [min(u, wide) for u in used]
        self.table = np.full((len(lengths), wide), -1, np.int32)
        order = rng.permutation(pages)[:sum(used)].astype(np.int32)
        at = 0
        for s, u in enumerate(used):
            self.table[s, :u] = order[at:at + u]
            at += u
        self.length = np.array(lengths, np.int32)
        self.start = None
        if start is not None:
            self.start = np.array(start, np.int32)
        elif counts is not None:
            self.start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.rows = int(rows if rows is not None else len(lengths) if self.start is None else self.start[-1])
        self.max_rows = int(max_rows or (1 if self.start is None else max(1, np.diff(self.start).max())))
        self.Q = Q
        self.upload(P)

    def upload(self, P):
        Q = self.Q
        self.dev = [None if x is None else Q.DeviceBuffer.from_array(x)
                    for x in (self.table, self.length, self.start)]
        self.c = P.Batch(self.dev[0], self.dev[1], len(self.length), self.table.shape[1], self.rows,
                         self.max_rows, start=self.dev[2])

    def places(self, pool):
        """(row, sequence, slot, place) of every row of a sequence."""
        for s, (lo, m) in enumerate(R.rows_of(self.start, len(self.length), self.rows, self.max_rows)):
            for i in range(m):
                slot = int(self.length[s]) - m + i
                yield lo + i, s, slot, R.place(self.table, s, slot, pool.shape[1], pool.shape[3])


def workspace(Q, P, pool, batch, qh):
    n = P.attn_workspace_bytes(pool.c, batch.c, qh)
    return Guarded(Q, n, 0) if n else None


def run_attn(Q, P, pool, batch, q, scale, layer=0, pad=0, out_pad=0, stream=None, ws=None,
             want_lse=True):
    rows, qh, d = q.shape
    host = np.full((rows, qh * d + pad), np.nan, np.float16)
    host[:, :qh * d] = q.reshape(rows, -1)
    qb = Q.DeviceBuffer.from_array(host)
    stride = qh * d + out_pad
    out, lse = Guarded(Q, 2 * (rows * stride - out_pad)), Guarded(Q, 4 * rows * qh)
    ws = ws or workspace(Q, P, pool, batch, qh)
    print(f"attn rows={rows} qh={qh} kvh={pool.shape[2]} d={d} page={pool.shape[3]} bits={pool.bits} "
          f"len={batch.length.tolist()[:8]} max_rows={batch.max_rows}", flush=True)
    P.attn(pool.c, layer, batch.c, qb, qh * d + pad, qh, scale, out.ptr, stride,
           lse.ptr if want_lse else None, ws.ptr if ws else None, ws.n if ws else 0, stream)
    Q.synchronize()
    if ws:
        ws.get(np.uint8)
    got = np.zeros(rows * stride, np.float16)
    got[:rows * stride - out_pad] = out.get(np.float16)
    got = got.reshape(rows, stride)
    if out_pad:
        assert (got[:-1, qh * d:].view(np.uint16) == 0xA5A5).all()
    got_lse = lse.get(np.float32).reshape(rows, qh)
    if not want_lse:
        assert (got_lse.view(np.uint32) == 0xA5A5A5A5).all()
    return got[:, :qh * d].reshape(rows, qh, d), got_lse


def check_attn(got, got_lse, ref, want_lse=True):
    out, lse, out_tol, lse_tol, mine = ref
    g = got.astype(np.float64)
    bad = ~(np.abs(g - out) <= out_tol)
    bad[~mine] = False
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:5], g[bad][:5], out[bad][:5], out_tol[bad][:5])
    assert (got[~mine].view(np.uint16) == 0xA5A5).all()
    if want_lse:
        gl = got_lse[mine].astype(np.float64)
        assert np.array_equal(np.isneginf(gl), np.isneginf(lse[mine]))
        ok = np.isfinite(lse[mine])
        assert (np.abs(gl[ok] - lse[mine][ok]) <= lse_tol[mine][ok]).all(), np.abs(gl[ok] - lse[mine][ok]).max()
        assert (got_lse[~mine].view(np.uint32) == 0xA5A5A5A5).all()


# query heads, kv heads, head_dim
HEADS = [(16, 8, 128), (14, 2, 64), (9, 3, 64), (16, 1, 128), (8, 8, 128), (64, 2, 64), (1, 1, 128)]


def attn_case(Q, P, seed, heads, bits, page, lengths, counts=None, spoil=True, **kw):
    rng = np.random.default_rng(seed)
    qh, kvh, d = heads
    need = sum((max(n, 0) + page - 1) // page for n in lengths) + 2
    pool = Pool(Q, P, rng, 2, need, page, kvh, d, bits)
    batch = Batch(Q, P, rng, pool, lengths, counts)
    if spoil:  # slots that no row sees hold NaN and infinities
        seen = np.zeros((need, page), bool)
        for s, n in enumerate(lengths):
            for j in range(n):
                seen[R.place(batch.table, s, j, need, page)] = True
        at = np.nonzero(~seen)
        for i, x in enumerate(pool.host if bits == 16 else pool.scales):
            x[:, at[0], :, at[1]] = (np.nan, np.inf)[i]
        pool.upload(P)
    q = normal(rng, (batch.rows, qh, d), 1.2)
    scale = float(np.float32(d ** -0.5))
    got = run_attn(Q, P, pool, batch, q, scale, layer=1, **kw)
    check_attn(*got, R.attention(q, pool.layer(1), batch.table, batch.length, batch.start,
                                 batch.max_rows, scale), kw.get("want_lse", True))


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("lengths", [[1], [15, 16, 17], [31, 32, 33, 1], [0, 5], [63, 64, 65, 127],
                                     [300], [1000, 1], [128] * 9])
def test_attn_lengths(gpu, P, bits, lengths):
    attn_case(gpu, P, len(lengths) + lengths[0], HEADS[0], bits, 16, lengths)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("page", [16, 48, 64, 256])
def test_attn_heads_and_pages(gpu, P, bits, heads, page):
    attn_case(gpu, P, page, heads, bits, page, [77, 130, 3], [1, 3, 2])


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("lengths,counts", [
    ([40, 7, 90], [5, 7, 0]), ([100, 33, 12], [8, 1, 9]), ([64, 64], [16, 17]), ([50], [33]),
    ([70, 40], [64, 40]), ([256], [256]), ([2000, 100, 555], [5, 2, 4])])
def test_attn_new_rows(gpu, P, bits, lengths, counts):
    attn_case(gpu, P, sum(counts), HEADS[0], bits, 32, lengths, counts)
    attn_case(gpu, P, sum(counts), HEADS[5], bits, 32, lengths[:1], counts[:1])


@pytest.mark.parametrize("bits", [16, 8])
def test_attn_long(gpu, P, bits):
    attn_case(gpu, P, 5, (4, 2, 128), bits, 64, [9000, 12, 4097], [2, 1, 3])
    attn_case(gpu, P, 6, (2, 1, 64), bits, 16, [20011])


@pytest.mark.parametrize("bits", [16, 8])
def test_attn_strides_and_no_lse(gpu, P, bits):
    attn_case(gpu, P, 7, HEADS[0], bits, 32, [50, 20], pad=24, out_pad=40)
    attn_case(gpu, P, 8, HEADS[1], bits, 32, [50, 20], want_lse=False)


@pytest.mark.parametrize("bits", [16, 8])
def test_attn_many_sequences(gpu, P, bits):
    rng = np.random.default_rng(3)
    lengths = rng.integers(1, 90, 300).tolist()
    attn_case(gpu, P, 9, (4, 2, 64), bits, 16, lengths, spoil=False)
    counts = [int(min(n, c)) for n, c in zip(lengths, rng.integers(0, 4, 300))]
    attn_case(gpu, P, 10, (4, 2, 64), bits, 16, lengths, counts, spoil=False)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_attn_rows_do_not_see_later_rows(gpu, P, bits, bad):
    """A new row whose k and v are NaN or infinite reaches only the rows from it on."""
    rng = np.random.default_rng(12)
    pool = Pool(gpu, P, rng, 1, 8, 16, 2, 128, bits)
    batch = Batch(gpu, P, rng, pool, [45, 20], [6, 2])
    page, entry = R.place(batch.table, 0, 42, 8, 16)  # row 3 of the first sequence
    if bits == 16:
        pool.host[1][0, page, :, entry, 5:9] = bad
    else:
        pool.scales[1][0, page, :, entry] = np.nan
    pool.upload(P)
    q = normal(rng, (8, 4, 128), 1.2)
    got, lse = run_attn(gpu, P, pool, batch, q, 0.1)
    clean = pool.layer(0)
    clean = (clean[0], np.nan_to_num(clean[1], nan=0, posinf=0, neginf=0), clean[2],
             None if clean[3] is None else np.nan_to_num(clean[3]))
    ref = R.attention(q, clean, batch.table, batch.length, batch.start, batch.max_rows, 0.1)
    hit = np.zeros(got.shape, bool)
    hit[3:6, :, slice(5, 9) if bits == 16 else slice(None)] = True
    assert not np.isfinite(got[hit]).any()
    # a weight within the bound of its exact value: the others are as ever
    g = np.where(hit, 0, got.astype(np.float64))
    out = np.where(hit, 0, ref[0])
    assert (np.abs(g - out) <= ref[2]).all()
    assert (np.abs(lse - ref[1]) <= ref[3]).all()


@pytest.mark.parametrize("bits", [16, 8])
def test_attn_slots_that_stand_for_nothing(gpu, P, bits):
    rng = np.random.default_rng(13)
    pool = Pool(gpu, P, rng, 1, 20, 16, 2, 64, bits)
    batch = Batch(gpu, P, rng, pool, [70, 40, 16, 1000, 3], wide=5)
    batch.table[0, 1] = -1
    batch.table[0, 3] = 20
    batch.table[1, 0] = 2 ** 31 - 1
    batch.table[2, 0] = -(2 ** 31)  # its only page: an empty row
    batch.upload(P)
    q = normal(rng, (5, 2, 64), 1.2)
    got, lse = run_attn(gpu, P, pool, batch, q, 0.125)
    ref = R.attention(q, pool.layer(0), batch.table, batch.length, None, 1, 0.125)
    check_attn(got, lse, ref)
    assert (got[2] == 0).all() and np.isneginf(lse[2]).all()


@pytest.mark.parametrize("bits", [16, 8])
def test_attn_rows_left_out(gpu, P, bits):
    """Starts before, behind and over the rows or max_rows, lengths below the rows or
    below none."""
    rng = np.random.default_rng(14)
    pool = Pool(gpu, P, rng, 1, 40, 16, 2, 64, bits)
    for start, max_rows in (([0, 2, 2, 5, 9], 4), ([1, 1, 4, 6, 7], 4), ([-2, 1, 3, 50, 60], 4),
                            ([0, 5, 6, 8, 8], 4)):
        batch = Batch(gpu, P, rng, pool, [50, 40, 33, 20], rows=10, start=start, max_rows=max_rows)
        q = normal(rng, (10, 4, 64), 1.2)
        got = run_attn(gpu, P, pool, batch, q, 0.125)
        check_attn(*got, R.attention(q, pool.layer(0), batch.table, batch.length, batch.start,
                                     max_rows, 0.125))
    batch = Batch(gpu, P, rng, pool, [2, -5, 0], [4, 2, 1])
    q = normal(rng, (7, 4, 64), 1.2)
    got, lse = run_attn(gpu, P, pool, batch, q, 0.125)
    check_attn(got, lse, R.attention(q, pool.layer(0), batch.table, batch.length, batch.start, 4, 0.125))
    assert np.isneginf(lse[[0, 1, 4, 5, 6]]).all() and np.isfinite(lse[[2, 3]]).all()


@pytest.mark.parametrize("bits", [16, 8])
def test_attn_extremes(gpu, P, bits):
    """Scores far apart and equal ones, zero rows, values of the largest size."""
    rng = np.random.default_rng(15)
    for case in range(4):
        pool = Pool(gpu, P, rng, 1, 24, 16, 2, 128, bits)
        batch = Batch(gpu, P, rng, pool, [200, 33, 90], [2, 1, 3])
        q = normal(rng, (6, 4, 128), (30.0, 1.0, 0.0, 1.0)[case])
        if case == 1:  # some rows of v are zero, some far larger than others
            for x in ([pool.host[1]] if bits == 16 else [pool.host[1], pool.scales[1]]):
                x[0, :5] = 0
            if bits == 16:
                pool.host[1][0, 5:9] *= np.float16(2000)
            else:
                pool.scales[1][0, 5:9] *= np.float32(2000)
        if case == 3:
            (pool.host[1] if bits == 16 else pool.scales[1])[:] *= np.float16(1e-3)
        pool.upload(P)
        got = run_attn(gpu, P, pool, batch, q, 0.09)
        check_attn(*got, R.attention(q, pool.layer(0), batch.table, batch.length, batch.start, 3, 0.09))


# ---------------------------------------------------------------- append ----

def append_case(Q, P, seed, heads, bits, page, lengths, counts=None, norm=True, theta=1e6,
                given=False, with_q=True, in_place=False, rows=None, start=None, spoil=None,
                max_rows=None, table=None):
    rng = np.random.default_rng(seed)
    qh, kvh, d = heads
    need = sum((max(n, 0) + page - 1) // page for n in lengths) + 2
    pool = Pool(Q, P, rng, 2, need, page, kvh, d, bits)
    batch = Batch(Q, P, rng, pool, lengths, counts, rows=rows, start=start, max_rows=max_rows)
    if table is not None:
        table(batch.table)
        batch.upload(P)
    n, cols = batch.rows, (qh + 2 * kvh) * d + 8
    x = normal(rng, (n, cols), 2.0)
    x[:, (qh + kvh // 2) * d + 3] *= np.float16(9)
    if spoil is not None:
        spoil(x)
    qn, kn = (normal(rng, (d,), 0.2) + np.float16(1) for _ in range(2))
    pos = rng.integers(0, 1 << 17, n).astype(np.int32) if given else None
    xb = Q.DeviceBuffer.from_array(x)
    nb = [Q.DeviceBuffer.from_array(w) for w in (qn, kn)]
    pb = None if pos is None else Q.DeviceBuffer.from_array(pos)
    out = Guarded(Q, 2 * n * qh * d)
    print(f"append rows={n} qh={qh} kvh={kvh} d={d} page={page} bits={bits} len={lengths[:8]}", flush=True)
    P.append(pool.c, 1, batch.c, xb.ptr + 2 * qh * d, cols, xb.ptr + 2 * (qh + kvh) * d, cols,
             k_norm=nb[1] if norm else None, q=xb if with_q else None, q_stride=cols if with_q else 0,
             q_heads=qh if with_q else 0, q_norm=nb[0] if norm else None,
             q_out=(xb if in_place else out.ptr) if with_q else None,
             q_out_stride=(cols if in_place else qh * d) if with_q else 0, eps=1e-6, theta=theta,
             positions=pb)
    Q.synchronize()
    after = xb.download(np.float16).reshape(n, cols)
    got_q = out.get(np.float16).reshape(n, qh, d)
    if in_place:
        assert (got_q.view(np.uint16) == 0xA5A5).all()
        got_q = after[:, :qh * d].reshape(n, qh, d)
    keep = slice(qh * d, None) if in_place else slice(None)
    assert np.array_equal(after[:, keep].view(np.uint16), x[:, keep].view(np.uint16))
    data, scales = pool.get()
    want = [a.copy() for a in pool.host]
    want_scale = [None if a is None else a.copy() for a in pool.scales]
    written = np.zeros((need, page), bool)
    mine = np.zeros(n, bool)
    for r, s, slot, at in batch.places(pool):
        mine[r] = True
        p = slot if pos is None else int(pos[r])
        heads_of = x[r, :(qh + 2 * kvh) * d].reshape(-1, d)
        q = R.turned(heads_of[:qh], qn if norm else None, 1e-6, theta, p)
        if with_q:
            fine = np.isfinite(q)
            q = np.where(fine, q, 0)
            g = got_q[r].astype(np.float64)
            assert np.array_equal(np.isfinite(g), fine)
            # in f32, 2^-24 each: half of the squares' 12 sums and of eps' one, 2 for the root,
            # 2 products; cosine, product and sum: under 16 of the two values that are turned
            y = np.abs(np.nan_to_num(R.turned(heads_of[:qh], qn if norm else None, 1e-6, 0.0, p)))
            turned = y + np.roll(y, d // 2, -1)
            assert (np.abs(g - q) <= 2.0 ** -11 * np.abs(q) + 2.0 ** -20 * turned + 2.0 ** -25)[fine].all()
        if at is None:
            continue
        written[at] = True
        ys = (R.turned(heads_of[qh:qh + kvh], kn if norm else None, 1e-6, theta, p),
              heads_of[qh + kvh:].astype(np.float64))
        for i, y in enumerate(ys):
            cell = data[i][1, at[0], :, at[1]]
            if bits == 8:
                sc = scales[i][1, at[0], :, at[1]]
                R.check_codes(y, cell.astype(np.float64), sc)
                want[i][1, at[0], :, at[1]] = cell
                want_scale[i][1, at[0], :, at[1]] = sc
            else:
                fine = np.isfinite(y)
                assert np.array_equal(np.isfinite(cell), fine)
                y, cell0 = np.where(fine, y, 0), np.where(fine, cell, 0)
                assert (np.abs(cell0.astype(np.float64) - y)
                        <= (2.0 ** -11 + 2.0 ** -23) * np.abs(y) + 2.0 ** -25).all()
                if i == 1:
                    assert np.array_equal(cell[fine], y[fine].astype(np.float16))
                want[i][1, at[0], :, at[1]] = cell
    # nothing else has changed
    for i in range(2):
        assert np.array_equal(data[i].view(np.uint8), want[i].view(np.uint8))
        if bits == 8:
            assert np.array_equal(scales[i].view(np.uint32), want_scale[i].view(np.uint32))
    if with_q and not in_place:
        assert (got_q[~mine].view(np.uint16) == 0xA5A5).all()
    return written


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("heads", HEADS)
def test_append(gpu, P, bits, heads):
    append_case(gpu, P, 1, heads, bits, 16, [1, 50, 33], [1, 5, 33])
    append_case(gpu, P, 2, heads, bits, 48, [100, 7], given=True)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("kw", [dict(norm=False), dict(theta=0.0), dict(norm=False, theta=0.0),
                                dict(with_q=False), dict(in_place=True), dict(theta=10000.0)])
def test_append_forms(gpu, P, bits, kw):
    append_case(gpu, P, 3, (6, 2, 64), bits, 32, [40, 9], [7, 2], **kw)
    append_case(gpu, P, 4, (16, 8, 128), bits, 32, [40, 9], [7, 2], **kw)


@pytest.mark.parametrize("bits", [16, 8])
def test_append_special_values(gpu, P, bits):
    def spoil(x):
        x[0, 16 * 128 + 5] = np.nan    # a k
        x[1, 18 * 128 + 5] = np.inf    # a v: heads 16, 17 are k's, 18, 19 v's
        x[2, 16 * 128:] = 0            # zero rows
        x[3, 16 * 128:] = np.float16(6e-8)
        x[4, 16 * 128:] = np.float16(65504)
        x[5, 18 * 128:] = np.arange(x.shape[1] - 18 * 128) % 255 - 127  # codes' own values
        x[6, 18 * 128:] = 15
        x[6, 18 * 128] = 762           # 15 lies on a border of scale 6

    append_case(gpu, P, 5, (16, 2, 128), bits, 16, [60], [9], spoil=spoil)
    append_case(gpu, P, 6, (16, 2, 128), bits, 16, [60], [9], spoil=spoil, norm=False, theta=0.0)


@pytest.mark.parametrize("bits", [16, 8])
def test_append_rows_and_slots_left_out(gpu, P, bits):
    append_case(gpu, P, 7, (4, 2, 64), bits, 16, [30, 20], [3, 2], rows=9)
    append_case(gpu, P, 8, (4, 2, 64), bits, 16, [30, 20, 40], rows=12, start=[2, 3, 8, 10], max_rows=4)
    append_case(gpu, P, 12, (4, 2, 64), bits, 16, [30, 20, 40], rows=12, start=[-1, 3, 6, 13], max_rows=4)
    append_case(gpu, P, 9, (4, 2, 64), bits, 16, [2, -3, 500], [4, 1, 1], given=True, table=None)

    def bad(table):
        table[0, 1] = -1
        table[1, 0] = 1 << 30

    append_case(gpu, P, 10, (4, 2, 64), bits, 16, [30, 10], [20, 5], table=bad)


def test_append_many_sequences(gpu, P):
    rng = np.random.default_rng(2)
    lengths = rng.integers(1, 40, 1024).tolist()
    counts = [int(min(n, c)) for n, c in zip(lengths, rng.integers(0, 3, 1024))]
    append_case(gpu, P, 11, (2, 1, 64), 8, 16, lengths, counts)


# ------------------------------------------------------------------ read ----

def read_case(Q, P, seed, kvh, d, bits, page, lengths, counts, layers=3, pad=8, rows=None, table=None):
    rng = np.random.default_rng(seed)
    need = sum((n + page - 1) // page for n in lengths) + 2
    pool = Pool(Q, P, rng, layers, need, page, kvh, d, bits)
    if bits == 8:
        pool.scales[0][0, 0] = np.nan
        pool.upload(P)
    batch = Batch(Q, P, rng, pool, lengths, counts, rows=rows)
    if table is not None:
        table(batch.table)
        batch.upload(P)
    n, row = batch.rows, kvh * d + pad
    lstride = n * row + 16
    outs = [Guarded(Q, 2 * (layers - 1) * lstride) for _ in range(2)]
    print(f"read rows={n} kvh={kvh} d={d} page={page} bits={bits}", flush=True)
    P.read(pool.c, 1, layers - 1, batch.c, outs[0].ptr, outs[1].ptr, row, lstride)
    Q.synchronize()
    for i in range(2):
        got = outs[i].get(np.uint16).reshape(layers - 1, lstride)
        want = np.full((layers - 1, lstride), 0xA5A5, np.uint16)
        for r, s, slot, at in batch.places(pool):
            for l in range(layers - 1):
                x = np.zeros((kvh, d), np.float16)
                if at is not None:
                    x = pool.host[i][l + 1, at[0], :, at[1]]
                    if bits == 8:
                        sc = pool.scales[i][l + 1, at[0], :, at[1]]
                        x = (x.astype(np.float32) * sc[:, None]).astype(np.float16)
                want[l, r * row:r * row + kvh * d] = x.reshape(-1).view(np.uint16)
        assert np.array_equal(got, want)


@pytest.mark.parametrize("bits", [16, 8])
def test_read(gpu, P, bits):
    read_case(gpu, P, 1, 8, 128, bits, 16, [1], [1])
    read_case(gpu, P, 2, 8, 128, bits, 64, [200, 0, 31], [200, 0, 31])
    read_case(gpu, P, 3, 3, 64, bits, 48, [100, 50], [7, 50], rows=61)
    read_case(gpu, P, 4, 1, 64, bits, 16, [100, 50], None)

    def bad(table):
        table[0, 2] = 1 << 20

    read_case(gpu, P, 5, 2, 128, bits, 16, [100, 50], [100, 50], table=bad)


# ---------------------------------------------------------------- verify ----

def verify_case(Q, P, seed, vocab, counts, max_rows=None, heat="mixed", drafted=True, spoil=None,
                pad=0, rows=None, start=None, logprob=True, uniform=None, ws=None):
    rng = np.random.default_rng(seed)
    start = np.array(start, np.int32) if start is not None else None if counts is None else \
        np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    seqs = rows if start is None else start.size - 1
    rows = rows or int(start[-1])
    max_rows = max_rows or (1 if start is None else max(1, int(np.diff(start).max())))
    logits = normal(rng, (rows, vocab + pad), 2.0)
    likely = rng.integers(0, vocab, (rows, 4))
    logits[np.arange(rows)[:, None], likely] += np.float16(9)
    tokens = np.roll(likely[:, 0], 1).astype(np.int32)
    u = rng.random(rows, dtype=np.float32) if uniform is None else np.full(rows, uniform, np.float32)
    temperature = None
    if heat is not None:
        temperature = (0.5 + rng.random(seqs)).astype(np.float32)
        temperature[rng.random(seqs) < 0.3] = 0 if heat == "mixed" else 0.7
    draft = None
    if drafted:
        x = logits[:, :vocab].astype(np.float64) + rng.standard_normal((rows, vocab))
        draft = np.full((rows, vocab + pad), np.nan, np.float32)
        e = np.exp(x - x.max(1, keepdims=True))
        draft[:, :vocab] = e / e.sum(1, keepdims=True)
    if spoil is not None:
        spoil(logits, tokens, temperature, draft)
    up = lambda a: None if a is None else Q.DeviceBuffer.from_array(a)  # noqa: E731
    lb, tb, ub, hb, db, sb = map(up, (logits, tokens, u, temperature, draft, start))
    ostride = max_rows + 3
    out, acc, lp = Guarded(Q, 4 * seqs * ostride), Guarded(Q, 4 * seqs), Guarded(Q, 4 * seqs * ostride)
    ws = ws or Guarded(Q, P.verify_workspace_bytes(rows, seqs, vocab), 0)
    print(f"verify rows={rows} seqs={seqs} vocab={vocab} drafted={drafted}", flush=True)
    for _ in range(2):
        P.verify(lb, vocab + pad, vocab, rows, tb, seqs, max_rows, ub, out.ptr, ostride, acc.ptr,
                 start=sb, temperature=hb, draft=db, draft_stride=vocab + pad,
                 logprob=lp.ptr if logprob else None, workspace=ws.ptr, workspace_bytes=ws.n)
    Q.synchronize()
    ws.get(np.uint8)
    got = out.get(np.int32).reshape(seqs, ostride)
    got_lp = lp.get(np.float32).reshape(seqs, ostride)
    assert (got[:, max_rows:].view(np.uint32) == 0xA5A5A5A5).all()
    assert (got_lp[:, max_rows if logprob else 0:].view(np.uint32) == 0xA5A5A5A5).all()
    want, accepted, wlp, margin = R.verify(logits[:, :vocab], tokens, start, seqs, max_rows, u,
                                           temperature, None if draft is None else draft[:, :vocab])
    # the sums are good to about 2^-40 of their total: numbers nearer to a border than
    # that would say nothing
    assert margin > 2.0 ** -40 or uniform is not None, margin
    assert np.array_equal(acc.get(np.int32), accepted)
    assert np.array_equal(got[:, :max_rows], want)
    if logprob:
        assert (np.abs(got_lp[:, :max_rows] - wlp) <= 2.0 ** -24 * np.abs(wlp) + 2.0 ** -40).all()
    return got[:, :max_rows], accepted


@pytest.mark.parametrize("drafted", [True, False])
@pytest.mark.parametrize("vocab", [1, 2, 255, 8191, 8192, 8193, 20011, 151936])
def test_verify_vocabularies(gpu, P, vocab, drafted):
    verify_case(gpu, P, vocab, vocab, [1, 4, 0, 3, 2], drafted=drafted)


@pytest.mark.parametrize("drafted", [True, False])
def test_verify_batches(gpu, P, drafted):
    verify_case(gpu, P, 1, 1001, None, rows=9, drafted=drafted)
    verify_case(gpu, P, 2, 3001, [9] * 20, drafted=drafted, pad=7)
    verify_case(gpu, P, 3, 501, [256, 1, 30], drafted=drafted)
    verify_case(gpu, P, 4, 701, None, rows=6, start=[0, 2, 2, 4, 8], max_rows=3, drafted=drafted)
    verify_case(gpu, P, 14, 701, None, rows=9, start=[1, 3, 7, 8], max_rows=3, drafted=drafted)
    verify_case(gpu, P, 5, 701, [2, 2], rows=7, heat=None, drafted=drafted, logprob=False)
    verify_case(gpu, P, 6, 64, [1] * 1024, drafted=drafted)


@pytest.mark.parametrize("drafted", [True, False])
def test_verify_borders_of_the_random_numbers(gpu, P, drafted):
    verify_case(gpu, P, 7, 9001, [4, 1, 5], drafted=drafted, uniform=0.0)
    verify_case(gpu, P, 8, 9001, [4, 1, 5], drafted=drafted, uniform=1.0 - 2.0 ** -24)


@pytest.mark.parametrize("drafted", [True, False])
def test_verify_special_values(gpu, P, drafted):
    def spoil(logits, tokens, temperature, draft):
        logits[0, 5] = np.nan
        logits[1, [7, 70, 700]] = np.inf
        logits[3] = -np.inf           # no distribution
        logits[6] = np.nan
        logits[7, 1:] = -np.inf       # one token alone
        tokens[9] = -1                # a drafted token that is none
        tokens[12] = 9001
        logits[13] = 3.0              # all alike
        if draft is not None:
            draft[13, 10:20] = np.nan
            draft[13, 20:30] = -1.0
        temperature[4] = -1.0

    for seed in (9, 10, 11):
        verify_case(gpu, P, seed, 9001, [3, 2, 1, 5, 6], drafted=drafted, heat="warm", spoil=spoil)


def test_verify_a_drafter_that_is_the_model(gpu, P):
    """Equal probabilities: everything is accepted."""
    def spoil(logits, tokens, temperature, draft):
        temperature[:] = 1.0
        x = logits.astype(np.float64)
        e = np.exp(x - x.max(1, keepdims=True))
        draft[:] = (e / e.sum(1, keepdims=True) * (1 - 2.0 ** -20)).astype(np.float32)

    _, accepted = verify_case(gpu, P, 12, 5000, [6, 6, 6], spoil=spoil)
    assert (accepted == 5).all()


def test_verify_keeps_the_models_distribution(gpu, P):
    """Over many sequences with a bad drafter, the first token falls as the model's p says:
    a chi-squared sum over 6 tokens below 25.7 (a chance of 10^-4 of more)."""
    rng = np.random.default_rng(4)
    seqs, vocab = 1024, 6
    row = np.array([1.0, 0.2, -0.5, 0.7, -2.0, 0.0], np.float16)
    q = np.array([0.05, 0.3, 0.3, 0.05, 0.2, 0.1])
    counts = np.zeros(vocab)
    for rep in range(8):
        tokens = rng.choice(vocab, 2 * seqs, p=q).astype(np.int32)
        logits = np.tile(row, (2 * seqs, 1))
        draft = np.tile(q.astype(np.float32), (2 * seqs, 1))
        u = rng.random(2 * seqs, dtype=np.float32)
        start = (2 * np.arange(seqs + 1)).astype(np.int32)
        b = [gpu.DeviceBuffer.from_array(a) for a in (logits, tokens, u, start, draft)]
        out, acc = gpu.DeviceBuffer(8 * seqs), gpu.DeviceBuffer(4 * seqs)
        ws = gpu.DeviceBuffer(P.verify_workspace_bytes(2 * seqs, seqs, vocab))
        ws.fill(0)
        P.verify(b[0], vocab, vocab, 2 * seqs, b[1], seqs, 2, b[2], out, 2, acc, start=b[3],
                 draft=b[4], draft_stride=vocab, workspace=ws, workspace_bytes=ws.nbytes)
        gpu.synchronize()
        counts += np.bincount(out.download(np.int32).reshape(seqs, 2)[:, 0], minlength=vocab)
    p = np.exp(row.astype(np.float64))
    want = p / p.sum() * counts.sum()
    assert ((counts - want) ** 2 / want).sum() < 25.7


# -------------------------------------------------------------- together ----

class Round:
    """A layer's step as it is used: new rows appended, attended to and read back, then
    judged by their logits."""

    def __init__(self, Q, P, seed, bits, heads=(16, 8, 128), page=32, vocab=5000, pages=60, seqs=4):
        self.Q, self.P, self.heads, self.vocab = Q, P, heads, vocab
        qh, kvh, d = heads
        rng = np.random.default_rng(seed)
        self.pool = Pool(Q, P, rng, 2, pages, page, kvh, d, bits)
        self.pages, self.page, self.seqs, self.rows, self.max_rows = pages, page, seqs, 3 * seqs, 5
        self.wide = pages // seqs
        up, n = Q.DeviceBuffer, self.rows
        cols = self.cols = (qh + 2 * kvh) * d
        self.table, self.length, self.start = up(4 * seqs * self.wide), up(4 * seqs), up(4 * seqs + 4)
        self.x, self.logits, self.draft = up(2 * n * cols), up(2 * n * vocab), up(4 * n * vocab)
        self.norms = up(4 * d)
        self.tokens, self.u, self.heat = up(4 * n), up(4 * n), up(4 * seqs)
        self.outs = [up(s) for s in (2 * n * qh * d, 2 * n * qh * d, 4 * n * qh, 2 * n * kvh * d,
                                     2 * n * kvh * d, 4 * seqs * 5, 4 * seqs, 4 * seqs * 5)]
        self.b = P.Batch(self.table, self.length, seqs, self.wide, n, self.max_rows, start=self.start)
        self.ws = [up(P.attn_workspace_bytes(self.pool.c, self.b, qh)),
                   up(P.verify_workspace_bytes(n, seqs, vocab))]
        for w in self.ws:
            w.fill(0)
        self.put(seed)

    def put(self, seed):
        """Other inputs, tables, lengths and starts in the same buffers."""
        rng = np.random.default_rng(seed)
        counts = rng.integers(0, self.max_rows + 1, self.seqs)
        while counts.sum() > self.rows:
            counts[counts.argmax()] -= 1
        self.table.upload(rng.permutation(self.pages)[:self.seqs * self.wide].astype(np.int32))
        self.length.upload(rng.integers(6, self.wide * self.page + 1, self.seqs).astype(np.int32))
        self.start.upload(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32))
        self.x.upload(normal(rng, (self.rows, self.cols)))
        self.norms.upload(normal(rng, (2, self.heads[2])))
        self.logits.upload(normal(rng, (self.rows, self.vocab), 3.0))
        draft = rng.random((self.rows, self.vocab), dtype=np.float32)
        self.draft.upload(draft / draft.sum(1, keepdims=True))
        self.tokens.upload(rng.integers(0, self.vocab, self.rows).astype(np.int32))
        self.u.upload(rng.random(self.rows, dtype=np.float32))
        self.heat.upload(rng.integers(0, 3, self.seqs).astype(np.float32))
        for o in self.outs:
            o.fill(0xA5)

    def run(self, stream=None):
        qh, kvh, d = self.heads
        P, x, n, o = self.P, self.x.ptr, self.rows, self.outs
        P.append(self.pool.c, 1, self.b, x + 2 * qh * d, self.cols, x + 2 * (qh + kvh) * d, self.cols,
                 k_norm=self.norms.ptr, q=x, q_stride=self.cols, q_heads=qh,
                 q_norm=self.norms.ptr + 2 * d, q_out=o[0], q_out_stride=qh * d, theta=1e4,
                 stream=stream)
        P.attn(self.pool.c, 1, self.b, o[0], qh * d, qh, d ** -0.5, o[1], qh * d, o[2], self.ws[0],
               self.ws[0].nbytes, stream)
        P.read(self.pool.c, 1, 1, self.b, o[3], o[4], kvh * d, stream=stream)
        P.verify(self.logits, self.vocab, self.vocab, n, self.tokens, self.seqs, self.max_rows, self.u,
                 o[5], self.max_rows, o[6], start=self.start, temperature=self.heat, draft=self.draft,
                 draft_stride=self.vocab, logprob=o[7], workspace=self.ws[1],
                 workspace_bytes=self.ws[1].nbytes, stream=stream)

    def got(self):
        return [o.download(np.uint8) for o in self.outs]

    def check(self):
        """Attention, codes read back and tokens against the plain forms."""
        qh, kvh, d = self.heads
        data, scales = self.pool.get()
        table = self.table.download(np.int32).reshape(self.seqs, self.wide)
        length, start = self.length.download(np.int32), self.start.download(np.int32)
        q = self.outs[0].download(np.float16).reshape(self.rows, qh, d)
        layer = (data[0][1], data[1][1], *(None if s is None else s[1] for s in scales))
        mine = np.zeros(self.rows, bool)
        mine[:start[-1]] = True
        ref = R.attention(np.where(mine[:, None, None], q, 0), layer, table, length, start, self.max_rows,
                          float(np.float32(d ** -0.5)))
        check_attn(self.outs[1].download(np.float16).reshape(self.rows, qh, d),
                   self.outs[2].download(np.float32).reshape(self.rows, qh), ref)
        want, accepted, _, margin = R.verify(
            self.logits.download(np.float16).reshape(self.rows, -1), self.tokens.download(np.int32), start,
            self.seqs, self.max_rows, self.u.download(np.float32), self.heat.download(np.float32),
            self.draft.download(np.float32).reshape(self.rows, -1))
        assert margin > 2.0 ** -40
        assert np.array_equal(self.outs[5].download(np.int32).reshape(self.seqs, -1), want)
        assert np.array_equal(self.outs[6].download(np.int32), accepted)


@pytest.mark.parametrize("bits", [16, 8])
def test_captured_and_replayed(gpu, P, bits):
    """One graph of the operators together, replayed as tables, lengths, starts and inputs
    change, with eager runs and synchronizations between: the eager run's bits each time."""
    r = Round(gpu, P, 1, bits)
    stream = gpu.Stream()
    r.run(stream)
    stream.synchronize()
    graph = gpu.Graph(stream, lambda: r.run(stream))
    for seed in range(2, 7):
        r.put(seed)
        r.run(stream)
        stream.synchronize()
        eager = r.got()
        r.check()
        for _ in range(2):
            for o in r.outs:
                o.fill(0xA5)
            graph.launch(stream)
            stream.synchronize()
            for a, b in zip(eager, r.got()):
                assert np.array_equal(a, b)
    graph.destroy()


def test_two_streams_at_once(gpu, P):
    """Rounds with pools and workspaces of their own, in flight together."""
    rounds = [Round(gpu, P, 11, 16), Round(gpu, P, 12, 8), Round(gpu, P, 13, 8, (4, 1, 64), 48, 20011)]
    alone = []
    for r in rounds:
        r.run()
        gpu.synchronize()
        alone.append(r.got())
    streams = [gpu.Stream() for _ in rounds]
    for _ in range(5):
        for r, s in zip(rounds, streams):
            r.run(s)
    for r, s, want in zip(rounds, streams, alone):
        s.synchronize()
        for a, b in zip(want, r.got()):
            assert np.array_equal(a, b)


def test_one_workspace_for_all_calls(gpu, P):
    """A workspace of the largest calls serves other heads, lengths, rows and types in turn,
    also when what lies behind its counters is left over from them."""
    rng = np.random.default_rng(14)
    cases = [((16, 8, 128), 16, 32, [900, 40], [3, 1]), ((14, 2, 64), 8, 16, [5000], [40]),
             ((16, 1, 128), 16, 64, [3000, 0, 17], None), ((64, 2, 64), 8, 256, [700, 2000], [1, 20]),
             ((1, 1, 128), 16, 16, [12000], [1]), ((16, 8, 128), 8, 32, [200] * 30, None)]
    calls, most = [], 0
    for heads, bits, page, lengths, counts in cases:
        need = sum((n + page - 1) // page for n in lengths) + 1
        pool = Pool(gpu, P, rng, 1, need, page, heads[1], heads[2], bits)
        batch = Batch(gpu, P, rng, pool, lengths, counts)
        q = normal(rng, (batch.rows, heads[0], heads[2]))
        calls.append((pool, batch, q, run_attn(gpu, P, pool, batch, q, 0.1)))
        most = max(most, P.attn_workspace_bytes(pool.c, batch.c, heads[0]))
    ws = Guarded(gpu, most, 0)
    for i in rng.integers(0, len(calls), 40):
        pool, batch, q, want = calls[i]
        for a, b in zip(want, run_attn(gpu, P, pool, batch, q, 0.1, ws=ws)):
            assert np.array_equal(a.view(np.uint8), b.view(np.uint8))
    shapes = [([3, 1, 5], 40000), ([1] * 9, 151936), ([5] * 20, 1000), (None, 9000)]
    most = max(P.verify_workspace_bytes(100, 40, v) for _, v in shapes)
    ws = Guarded(gpu, most, 0)
    for i in (0, 1, 2, 3, 2, 1, 0, 3, 1):
        verify_case(gpu, P, 20 + i, shapes[i][1], shapes[i][0], rows=40 if i == 3 else None, ws=ws)


@pytest.mark.parametrize("bits", [16, 8])
def test_offsets_past_32_bits(gpu, P, bits):
    """The pages of a second layer behind 2^32 values: written, attended to, read back."""
    rng = np.random.default_rng(15)
    qh, kvh, d = 16, 8, 128
    page, pages, lengths = 4096, 600, [300, 5000, 20]
    n = 2 * pages * kvh * page
    size = n * d * bits // 8
    kb, vb = gpu.DeviceBuffer(size), gpu.DeviceBuffer(size)
    sb = [gpu.DeviceBuffer(4 * n) if bits == 8 else None for _ in range(2)]
    for b in (kb, vb, *sb):
        if b is not None:
            b.fill(0x7F if bits == 16 else 0)  # f16 NaN
    c = P.Pages(kb, vb, pages, page, 2, kvh, d, *sb)
    table = np.array([[599, 0], [598, 300], [2, 1]], np.int32)
    tb, lb = gpu.DeviceBuffer.from_array(table), gpu.DeviceBuffer.from_array(np.array(lengths, np.int32))
    start = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    stb = gpu.DeviceBuffer.from_array(start)
    every = P.Batch(tb, lb, 3, 2, int(start[-1]), 5000, start=stb)
    x = normal(rng, (int(start[-1]), 2, kvh * d))
    xb = gpu.DeviceBuffer.from_array(x)
    print(f"offsets bits={bits}", flush=True)
    P.append(c, 1, every, xb, 2 * kvh * d, xb.ptr + 2 * kvh * d, 2 * kvh * d)
    outs = [gpu.DeviceBuffer(x.nbytes // 2) for _ in range(2)]
    P.read(c, 1, 1, every, outs[0], outs[1], kvh * d)
    last = P.Batch(tb, lb, 3, 2, 3)
    q = normal(rng, (3, qh, d))
    qb, out, lse = gpu.DeviceBuffer.from_array(q), gpu.DeviceBuffer(q.nbytes), gpu.DeviceBuffer(4 * 3 * qh)
    ws = gpu.DeviceBuffer(P.attn_workspace_bytes(c, last, qh))
    ws.fill(0)
    P.attn(c, 1, last, qb, qh * d, qh, 0.09, out, qh * d, lse, ws, ws.nbytes)
    gpu.synchronize()
    # a small pool with the same rows, under the same tables
    held = sorted({0, 1, 2, 300, 598, 599})
    small_table = np.searchsorted(held, table).astype(np.int32)
    data = [np.zeros((len(held), kvh, page, d), np.float16 if bits == 16 else np.int8) for _ in range(2)]
    scale = [np.zeros(a.shape[:3], np.float32) if bits == 8 else None for a in data]
    for i in range(2):
        got = outs[i].download(np.float16).reshape(-1, kvh, d)
        want = x[:, i].reshape(-1, kvh, d)
        if bits == 16:
            assert np.array_equal(got, want)
        code, sc = quantised(want)
        if bits == 8:  # half a step and f16's rounding
            g, y, step = got.astype(np.float64), want.astype(np.float64), sc[..., None].astype(np.float64)
            assert (np.abs(g - y) <= step * (0.5 + 2.0 ** -16) + 2.0 ** -11 * np.abs(g) + 2.0 ** -25).all()
            code = np.rint(g / np.where(step > 0, step, 1))
        for s in range(3):
            for p in range(lengths[s]):
                at = small_table[s, p // page], slice(None), p % page
                data[i][at] = want[start[s] + p] if bits == 16 else code[start[s] + p]
                if bits == 8:
                    scale[i][at] = sc[start[s] + p]
    ref = R.attention(q, (data[0], data[1], *scale), small_table, np.array(lengths, np.int32), None, 1,
                      float(np.float32(0.09)))
    check_attn(out.download(np.float16).reshape(q.shape), lse.download(np.float32).reshape(3, qh), ref)
    for b in (kb, vb, *sb):
        if b is not None:
            b.free()


@pytest.mark.parametrize("bits", [16, 8])
def test_same_inputs_same_bits(gpu, P, bits):
    """Sequences cut among many workgroups, which arrive in any order."""
    rng = np.random.default_rng(16)
    pool = Pool(gpu, P, rng, 1, 700, 32, 8, 128, bits)
    batch = Batch(gpu, P, rng, pool, [20000, 37, 1500], [2, 1, 5])
    q = normal(rng, (batch.rows, 16, 128), 1.5)
    ws = workspace(gpu, P, pool, batch, 16)
    first = run_attn(gpu, P, pool, batch, q, 0.09, ws=ws)
    for _ in range(6):
        for a, b in zip(first, run_attn(gpu, P, pool, batch, q, 0.09, ws=ws)):
            assert np.array_equal(a.view(np.uint8), b.view(np.uint8))
