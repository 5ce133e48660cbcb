"""Several sequences through the whole model (qwen3_pages_step, serving.PagedSession) on
the GPU: against the prompt path, against a flat cache that the pages were read into,
with drafted tokens, captured and on two streams.

Tolerances.  Two routes through the 28 layers round the same 8 f16 tensors a layer but sum in
other orders, so roundings may fall to the other side: each has an rms of 2^-11 / sqrt(3)
of the value, 28 * 8 of them unrelated 2^-11 * sqrt(28 * 8 / 3) = 4.2e-3; relative L2 is held
to 5e-3.  8-bit pages are compared with the values they stand for, read into a flat cache
(which rounds them to f16, one of those tensors).  Where the same launches run on the
same values, equality is exact."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

import pages_ref as R

pytestmark = pytest.mark.gpu

VOCAB = 151936


@pytest.fixture(scope="module")
def D(gpu):
    from qwen3_iree_amd import decode

    return decode


@pytest.fixture(scope="module")
def S(gpu):
    from qwen3_iree_amd import serving

    return serving


@pytest.fixture(scope="module")
def model(D, model_host):
    m = D.DeviceWeights(model_host)
    yield m
    m.free()


def rel(a, b):
    a, b = a.astype(np.float32), b.astype(np.float32)
    return float(np.linalg.norm(a - b) / np.linalg.norm(b))


def prompt_logits(D, model, tokens):
    s = D.DecodeSession(model, len(tokens) + 1)
    s.prefill_batched(tokens, logits=True)
    out = s.read_logits()
    s.free()
    return out


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("counts", [[1], [5, 9, 2], [20, 30, 1, 13], [100, 28]])
def test_sequences_are_their_prompts(D, S, model, counts, f16):
    """Ragged rows of several sequences behind prompts of other lengths: the last row of each
    is what its whole sequence gives."""
    rng = np.random.default_rng(sum(counts))
    model.use_prefill_matrices(f16)
    try:
        sess = S.PagedSession(model, pages=80, max_seqs=4, max_len=400, page_size=16)
        texts = [rng.integers(0, VOCAB, 7 + 31 * i + m) for i, m in enumerate(counts)]
        seqs = [sess.add() for _ in counts]
        for s, t, m in zip(seqs, texts, counts):
            if t.size > m:
                sess.prompt(s, t[:-m])
        print(f"counts {counts} f16={f16}", flush=True)
        nxt = sess.step({s: t[-m:] for s, t, m in zip(seqs, texts, counts)}, logits=True)
        got = sess.read_logits(sum(counts))
        at = 0
        for s, t, m in zip(seqs, texts, counts):
            assert np.array_equal(nxt[s], got[at:at + m].argmax(1))
            assert rel(got[at + m - 1], prompt_logits(D, model, t)) < 5e-3
            at += m
        sess.free()
    finally:
        model.use_prefill_matrices(True)


@pytest.mark.parametrize("bits,page_size", [(16, 64), (8, 64), (8, 16), (8, 48)])
def test_pages_read_into_a_flat_cache(D, S, model, bits, page_size):
    rng = np.random.default_rng(bits)
    tokens = rng.integers(0, VOCAB, 200)
    sess = S.PagedSession(model, pages=30, max_seqs=2, max_len=300, page_size=page_size, bits=bits)
    other, s = sess.add(), sess.add()
    sess.prompt(other, tokens[:50])
    sess.prompt(s, tokens[:150])
    flat = D.DecodeSession(model, 300)
    sess.to_session(s, flat)
    assert flat.get_state()[1] == 150
    sess.step({other: [3, 4], s: tokens[150:152]}, logits=True)
    got = sess.read_logits(4)[3]
    for t in tokens[150:152]:
        flat.set_state(int(t), flat.get_state()[1])
        flat.step()
        flat.check_status()
    print(f"bits {bits} rel {rel(got, flat.read_logits()):.2e}", flush=True)
    # two of the 152 slots are f16 in the flat cache but codes in the pages: off by half a
    # step of 127 at most, in sums that they have a share of about 2 / 152 in
    assert rel(got, flat.read_logits()) < 5e-3 + (0.5 / 127 * 2 / 152 if bits == 8 else 0)
    flat.free()
    sess.free()


@pytest.mark.parametrize("bits", [16, 8])
def test_greedy_drafts(S, model, bits):
    """Temperature 0: drafts that the model would choose stand, a wrong one ends them, and the
    sequences go on as if no draft had been made."""
    rng = np.random.default_rng(4)
    sess = S.PagedSession(model, pages=60, max_seqs=3, max_len=256, page_size=32, bits=bits)
    texts = [rng.integers(0, VOCAB, n) for n in (30, 5, 61)]
    plain = []
    for t in texts:  # one token a step, one sequence at a time
        s = sess.add()
        out = [sess.prompt(s, t)]
        for _ in range(9):
            out.append(int(sess.step({s: [out[-1]]})[s][0]))
        plain.append(out)
        sess.remove(s)
    seqs = [sess.add() for _ in texts]
    got = [[sess.prompt(s, t)] for s, t in zip(seqs, texts)]
    wrong = 0
    for turn in range(20):
        live = [i for i in range(3) if len(got[i]) < 10]
        if not live:
            break
        rows = {}
        for i in live:
            n = len(got[i])
            ahead = plain[i][n:n + 1 + (turn + i) % 4]
            if (turn + i) % 3 == 0 and ahead:
                ahead[-1] = (ahead[-1] + 1) % VOCAB
                wrong += 1
            rows[seqs[i]] = [got[i][-1], *ahead]
        before = {s: sess.length[s] for s in rows}
        total = sum(len(r) for r in rows.values())
        out = sess.sample(rows, rng.random(total), temperature=np.zeros(len(rows)))
        logits, at = sess.read_logits(total).astype(np.float32), 0
        for i in live:
            tokens, logprob = out[seqs[i]]
            best = logits[at:at + len(rows[seqs[i]])].argmax(1)
            # what stands is what the logits of this very step say
            assert np.array_equal(tokens, best[:tokens.size])
            assert np.array_equal(tokens[:-1], rows[seqs[i]][1:tokens.size])
            assert (logprob == 0).all()
            assert sess.length[seqs[i]] == before[seqs[i]] + tokens.size
            got[i] += tokens.tolist()
            at += len(rows[seqs[i]])
    same = [int(np.argmin([a == b for a, b in zip(g, p)] + [False])) for g, p in zip(got, plain)]
    print(f"bits {bits}: {same} tokens alike, {wrong} wrong drafts", flush=True)
    # the first tokens at least, where two routes' sums do not differ by more than the gap
    assert min(same) >= 1 and wrong > 0
    sess.free()


def test_sampled_drafts_are_what_the_logits_say(S, model):
    rng = np.random.default_rng(6)
    sess = S.PagedSession(model, pages=40, max_seqs=4, max_len=200, page_size=16, bits=8)
    seqs = [sess.add() for _ in range(4)]
    for s in seqs:
        sess.prompt(s, rng.integers(0, VOCAB, 10 + s))
    rows = {s: rng.integers(0, VOCAB, 1 + s) for s in seqs}
    total = sum(len(r) for r in rows.values())
    start = np.concatenate([[0], np.cumsum([len(r) for r in rows.values()])])
    tokens = np.concatenate(list(rows.values()))
    u = rng.random(total, dtype=np.float32)
    heat = np.array([0.7, 1.0, 0.0, 1.3], np.float32)
    for draft in (None, np.full((total, VOCAB), 1.0 / VOCAB, np.float32)):
        before = dict(sess.length)
        out = sess.sample(rows, u, temperature=heat, draft=draft)
        want, accepted, logprob, margin = R.verify(sess.read_logits(total), tokens, start, 4, 4, u, heat, draft)
        assert margin > 2.0 ** -40
        for i, s in enumerate(seqs):
            assert out[s][0].tolist() == want[i, :accepted[i] + 1].tolist()
            assert np.allclose(out[s][1], logprob[i, :accepted[i] + 1], rtol=2.0 ** -23, atol=2.0 ** -40)
            assert sess.length[s] == before[s] + 1 + accepted[i]
            sess.cut(s, before[s])
    sess.free()


@pytest.mark.parametrize("bits", [16, 8])
def test_a_captured_step_follows_its_sequences(S, D, model, gpu, bits):
    """A step captured once, replayed as lengths, pages and tokens change on the device, with
    eager steps between the replays: the eager step's bits every time."""
    from qwen3_iree_amd import pages as P

    rng = np.random.default_rng(9)
    stream = gpu.Stream()
    sess = S.PagedSession(model, pages=40, max_seqs=3, max_len=160, page_size=16, bits=bits, stream=stream)
    seqs = [sess.add() for _ in range(3)]
    for s in seqs:
        sess.prompt(s, rng.integers(0, VOCAB, 30 * s + 14))
    tok, nxt = gpu.DeviceBuffer(12), gpu.DeviceBuffer(12)
    logits = gpu.DeviceBuffer(3 * VOCAB * 2)
    ws = gpu.DeviceBuffer(int(gpu.load_library().qwen3_pages_workspace_bytes(3, 1)))
    ws.fill(0)
    table, length = gpu.DeviceBuffer(4 * 3 * sess.max_pages), gpu.DeviceBuffer(12)
    batch = P.Batch(table, length, 3, sess.max_pages, 3)

    def step():
        gpu._call("qwen3_pages_step", model.ref(), ctypes.byref(sess.pages), ctypes.byref(batch),
                  tok.ptr, nxt.ptr, logits.ptr, ws.ptr, ws.nbytes, stream.handle)

    graph = None
    for trial in range(5):
        tokens = {s: rng.integers(0, VOCAB, 1) for s in seqs}
        eager_next = sess.step(tokens, logits=True)  # takes the pages and moves the lengths
        t = np.zeros((3, sess.max_pages), np.int32)
        for s in seqs:
            t[s, :len(sess._held[s])] = sess._held[s]
        table.upload(t)
        length.upload(np.array([sess.length[s] for s in seqs], np.int32))
        tok.upload(np.concatenate([tokens[s] for s in seqs]).astype(np.int32))
        step()
        stream.synchronize()
        eager = logits.download(np.uint16)
        assert np.array_equal(nxt.download(np.int32), [eager_next[s][0] for s in seqs])
        if graph is None:
            graph = gpu.Graph(stream, step)
        for _ in range(2):
            logits.fill(0)
            nxt.fill(0)
            graph.launch(stream)
            stream.synchronize()
            assert np.array_equal(logits.download(np.uint16), eager)
            assert np.array_equal(nxt.download(np.int32), [eager_next[s][0] for s in seqs])
    graph.destroy()
    sess.free()


def test_two_sessions_on_two_streams(S, model, gpu):
    from qwen3_iree_amd import pages as P

    rng = np.random.default_rng(10)
    sess = [S.PagedSession(model, pages=40, max_seqs=3, max_len=160, page_size=16, bits=b,
                           stream=gpu.Stream()) for b in (16, 8)]
    alone, again = [], []
    for x in sess:
        seqs = [x.add() for _ in range(3)]
        for s in seqs:
            x.prompt(s, rng.integers(0, VOCAB, 20 * s + 40))
        x.step({s: rng.integers(0, VOCAB, 2 + s) for s in seqs}, logits=True)
        alone.append(x.read_logits(9).copy())
        batch = x._batch(seqs, [2, 3, 4], [x.length[s] for s in seqs])
        again.append(batch)
    for x, b in zip(sess, again):  # the same rows once more, both in flight
        at = x._words.ptr + x._tokens
        gpu._call("qwen3_pages_step", x.model.ref(), ctypes.byref(x.pages), ctypes.byref(b), at,
                  at + 512, x._logits.ptr, x._ws.ptr, x._ws.nbytes, x.stream.handle)
    for x, want in zip(sess, alone):
        assert np.array_equal(x.read_logits(9), want)
        x.free()


@pytest.mark.parametrize("bits", [16, 8])
def test_padding_rows_and_used_workspaces(S, model, gpu, bits):
    """A step of 12 rows of which the sequences have 7: tokens outside the vocabulary in the
    rows behind them, NaN left behind the workspace's counters, and no other row, page or
    scale changes."""
    from qwen3_iree_amd import pages as P

    rng = np.random.default_rng(21)
    x = S.PagedSession(model, pages=20, max_seqs=3, max_len=96, page_size=16, bits=bits)
    seqs = [x.add() for _ in range(3)]
    for s in seqs:
        x.prompt(s, rng.integers(0, VOCAB, 20 + 11 * s))
    x.step({s: rng.integers(0, VOCAB, 1 + 2 * (s % 2) + s // 2) for s in seqs}, logits=True)
    counts = [1, 3, 2]
    batch = x._batch(seqs, counts, [x.length[s] for s in seqs])
    tokens = np.concatenate([x._words.download(np.int32, 6, x._tokens), [-5, 1 << 30, 7, 0, -1, 9]])
    tb, nb = gpu.DeviceBuffer.from_array(tokens.astype(np.int32)), gpu.DeviceBuffer(4 * 12)
    logits = gpu.DeviceBuffer(12 * VOCAB * 2)
    n = int(gpu.load_library().qwen3_pages_workspace_bytes(12, 12))
    counters = 1 << 16
    ws = gpu.DeviceBuffer(n)

    def pool():
        return [b.download(np.uint8) for b in (*x._pool, *x._scales) if b is not None]

    results, before = [], pool()
    for behind in (0, 0xFF, 0x7E):
        ws.fill(behind)
        ws.upload(np.zeros(counters, np.uint8))
        wide = P.Batch(batch.table, batch.length, 3, x.max_pages, 12, 12, start=batch.start)
        gpu._call("qwen3_pages_step", model.ref(), ctypes.byref(x.pages), ctypes.byref(wide), tb.ptr, nb.ptr,
                  logits.ptr, ws.ptr, n, None)
        gpu.synchronize()
        results.append((logits.download(np.uint16, 6 * VOCAB), nb.download(np.int32, 6)))
        assert (ws.download(np.uint8, counters) == 0).all()
    for r in results[1:]:
        assert np.array_equal(r[0], results[0][0]) and np.array_equal(r[1], results[0][1])
    # the same rows as before were written again, with the same values
    for a, b in zip(before, pool()):
        assert np.array_equal(a, b)
    assert np.array_equal(results[0][0].view(np.float16).reshape(6, VOCAB).view(np.uint16),
                          x.read_logits(6).view(np.uint16))
    x.free()


def test_sessions_of_all_sizes_share_a_workspace(S, model, gpu):
    """One workspace of the largest step for steps of few and many rows, one and many a
    sequence, in turn: what a fresh one gives."""
    rng = np.random.default_rng(22)
    x = S.PagedSession(model, pages=60, max_seqs=8, max_len=256, page_size=32, bits=8)
    fresh = []
    shapes = [[1], [128], [1] * 8, [16] * 8, [40, 1, 60], [7, 9], [65]]
    for turn in range(2):
        for i, counts in enumerate(shapes):
            seqs = [x.add() for _ in counts]
            r = np.random.default_rng(100 + i)
            x.step({s: r.integers(0, VOCAB, m) for s, m in zip(seqs, counts)}, logits=True)
            got = x.read_logits(sum(counts)).view(np.uint16).copy()
            for s in seqs:
                x.remove(s)
            if turn == 0:
                x._ws.fill(0)
                fresh.append(got)
            else:
                assert np.array_equal(got, fresh[i])
    x.free()
