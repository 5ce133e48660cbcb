"""What refused drafts leave behind in a PagedSession: nothing.  The next step's logits are
those of a session that never saw them.

Tolerance: as in test_gpu_serving, two routes of other sums stay within a relative L2 of 5e-3.
With 8-bit pages the two slots that the routes fill in steps of other sizes may also get
codes one step apart, 1 / 127 of their rows' largest values, in sums over 30 slots at least
that they have a share of 2 / 30 in."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_serving import D, S, VOCAB, model, rel  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("page_size", [16, 48])
def test_refused_drafts_leave_nothing(S, model, bits, page_size):
    """Drafts over the end of a page, all of them refused; another sequence takes the pages that
    this gives back, and one more step goes over their places again."""
    rng = np.random.default_rng(30 + bits)
    texts = [rng.integers(0, VOCAB, n) for n in (30, 46, 61)]
    a = S.PagedSession(model, pages=30, max_seqs=4, max_len=128, page_size=page_size, bits=bits)
    b = S.PagedSession(model, pages=30, max_seqs=4, max_len=128, page_size=page_size, bits=bits)
    seqs = [a.add() for _ in texts]
    assert seqs == [b.add() for _ in texts]
    first = {s: a.prompt(s, t) for s, t in zip(seqs, texts)}
    assert first == {s: b.prompt(s, t) for s, t in zip(seqs, texts)}
    plain = b.step({s: [first[s]] for s in seqs})
    # drafts that the model does not choose: the first of each is not what it says
    rows = {s: [first[s], (int(plain[s][0]) + 1 + s) % VOCAB, *rng.integers(0, VOCAB, 15 + s)] for s in seqs}
    total = sum(len(r) for r in rows.values())
    out = a.sample(rows, rng.random(total), temperature=np.zeros(3))
    logits, at = a.read_logits(total).astype(np.float32), 0
    following = {}
    for s in seqs:
        tokens, _ = out[s]
        top = np.sort(logits[at])[-2:]
        print(f"sequence {s}: {tokens.tolist()}, plain {plain[s].tolist()}, gap {top[1] - top[0]:.3f}", flush=True)
        at += len(rows[s])
        assert tokens.size == 1  # nothing stood
        assert a.length[s] == b.length[s]
        following[s] = [int(tokens[0])]
    other = a.add()
    a.prompt(other, rng.integers(0, VOCAB, 70))
    a.step(following, logits=True)
    got = a.read_logits(3)
    b.step(following, logits=True)
    want = b.read_logits(3)
    for i, s in enumerate(seqs):
        print(f"bits {bits} sequence {s}: rel {rel(got[i], want[i]):.2e}", flush=True)
        assert rel(got[i], want[i]) < 5e-3 + (1 / 127 * 2 / 30 if bits == 8 else 0)
    a.free()
    b.free()
