"""What a PagedSession remembers between its calls, what it refuses, and the refusals of
qwen3_pages_step, on the CPU: the library's calls are recorded in place of being made."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

A = 0x10000


@pytest.fixture(scope="module")
def D(Q):
    from qwen3_iree_amd import decode

    return decode


@pytest.fixture(scope="module")
def P(Q):
    from qwen3_iree_amd import pages

    return pages


class Words:
    """Stands for a DeviceBuffer; keeps what is uploaded, downloads it."""

    def __init__(self, nbytes):
        self.data = np.zeros(min(nbytes, 1 << 16), np.uint8)
        self.ptr, self.nbytes = A, nbytes

    def __int__(self):
        return self.ptr

    def fill(self, value=0):
        pass

    def free(self):
        pass

    def upload(self, array, offset=0):
        raw = np.ascontiguousarray(array).view(np.uint8).ravel()
        self.data[offset:offset + raw.size] = raw

    def download(self, dtype, count=None, offset=0):
        n = np.dtype(dtype).itemsize * count
        return self.data[offset:offset + n].copy().view(dtype)


@pytest.fixture
def make(Q, monkeypatch):
    from qwen3_iree_amd import serving

    calls = []
    monkeypatch.setattr(Q, "DeviceBuffer", Words)
    monkeypatch.setattr(Q, "_call", lambda name, *a: calls.append(name))
    monkeypatch.setattr(Q, "synchronize", lambda: None)
    model = type("Model", (), {"ref": staticmethod(lambda: None)})()

    def build(**kw):
        s = serving.PagedSession(model, **{**dict(pages=6, max_seqs=3, max_len=64, page_size=16), **kw})
        s.calls = calls
        return s

    return build


def held(s):
    pages = [p for h in s._held.values() for p in h] + s._free
    assert sorted(pages) == list(range(6))
    return {q: len(h) for q, h in s._held.items()}


def test_pages_come_and_go(make):
    s = make()
    a, b = s.add(), s.add()
    s.step({a: np.zeros(17), b: [1]})
    assert held(s) == {a: 2, b: 1} and s.length == {a: 17, b: 1}
    s.step({a: [1]})
    assert held(s)[a] == 2 and s.length[a] == 18
    s.cut(a, 16)
    assert held(s)[a] == 1
    s.cut(a, 0)
    assert held(s)[a] == 0
    s.remove(b)
    assert held(s) == {a: 0} and s.add() == b
    assert s.calls.count("qwen3_pages_step") == 2


def test_the_uploaded_batch(make, Q):
    s = make()
    a, b = s.add(), s.add()
    s.step({b: np.arange(20), a: [7, 8]})
    words = s._words.download(np.int32, 2 * 4 + 2 + 3)
    assert words[:2].tolist() == s._held[b] and words[4] == s._held[a][0]
    assert words[8:].tolist() == [20, 2, 0, 20, 22]
    assert s._words.download(np.int32, 22, s._tokens).tolist() == [*range(20), 7, 8]


def test_refused_steps_change_nothing(make):
    s = make()
    a, b = s.add(), s.add()
    s.step({a: np.zeros(40), b: np.zeros(16)})
    before, lengths = held(s), dict(s.length)
    for bad in ({}, {a: []}, {a: np.zeros(129)}, {a: np.zeros(25)}, {b: np.zeros(48), a: np.zeros(10)}):
        with pytest.raises(ValueError):
            s.step(bad)
        assert held(s) == before and s.length == lengths
    for n in (0, 25, 200):  # a prompt that does not fit is not begun
        with pytest.raises(ValueError):
            s.prompt(a, np.zeros(n))
        assert held(s) == before and s.length == lengths
    with pytest.raises(KeyError):
        s.step({9: [1]})
    assert s.add() == 2
    with pytest.raises(ValueError, match="in use"):
        s.add()
    for n in (-1, 41):
        with pytest.raises(ValueError):
            s.cut(a, n)


def test_a_failed_step_gives_its_pages_back(make, Q, monkeypatch):
    s = make()
    a = s.add()
    s.step({a: np.zeros(10)})

    def fail(name, *args):
        raise Q.Q8GemvError(8, "no")

    monkeypatch.setattr(Q, "_call", fail)
    with pytest.raises(Q.Q8GemvError):
        s.step({a: np.zeros(30)})
    assert held(s) == {a: 1} and s.length[a] == 10


def test_sample_refuses_what_does_not_fit(make):
    s = make()
    a = s.add()
    for kw in (dict(uniform=[0.5]), dict(uniform=[0.5] * 2, temperature=[1.0, 1.0]),
               dict(uniform=[0.5] * 2, draft=np.zeros((2, 10)))):
        with pytest.raises(ValueError):
            s.sample({a: [1, 2]}, **kw)
        assert s.length[a] == 0


def test_a_failed_verification_drops_the_rows(make, Q, monkeypatch):
    s = make()
    a = s.add()
    s.step({a: np.zeros(5)})

    def fail(name, *args):
        if name == "kv_verify":
            raise Q.Q8GemvError(8, "no")

    monkeypatch.setattr(Q, "_call", fail)
    with pytest.raises(Q.Q8GemvError):
        s.sample({a: [1, 2, 3]}, [0.1, 0.2, 0.3])
    assert s.length[a] == 5


def test_sample_keeps_the_accepted_slots(make):
    s = make()
    a = s.add()
    s.step({a: np.zeros(14)})
    out = s.sample({a: [1, 2, 3, 4]}, [0.1] * 4)  # the stand-in says 0 accepted
    assert s.length[a] == 15 and held(s)[a] == 1
    assert out[a][0].size == 1


@pytest.mark.parametrize("kw", [dict(max_seqs=0), dict(max_seqs=1025), dict(bits=4), dict(page_size=24),
                                dict(page_size=0), dict(pages=0), dict(max_len=0)])
def test_bad_sessions(make, kw):
    with pytest.raises(ValueError):
        make(**kw)


# ---------------------------------------------------- qwen3_pages_step ----

PAGES = dict(k=A, v=A, pages=10, page_size=16, layers=28, kv_heads=8, head_dim=128)
BATCH = dict(table=A, length=A, seqs=3, max_pages=4, rows=3, max_rows=1)
STEP = dict(tokens=A, nxt=A, logits=A, ws=A, nbytes=1 << 40)


def call(Q, D, P, pages={}, batch={}, weights=True, **kw):
    w = D.WeightsC(*([A] * len(D.WEIGHT_FIELDS)), None)
    a = {**STEP, **kw}
    return Q.load_library().qwen3_pages_step(
        ctypes.byref(w) if weights else None,
        None if pages is None else ctypes.byref(P.Pages(**{**PAGES, **pages})),
        None if batch is None else ctypes.byref(P.Batch(**{**BATCH, **batch})),
        a["tokens"], a["nxt"], a["logits"], a["ws"], a["nbytes"], None)


@pytest.mark.parametrize("kw,code", [
    ({"weights": False}, 3), ({"pages": None}, 3), ({"batch": None}, 3), ({"tokens": None}, 3),
    ({"nxt": None}, 3), ({"ws": None}, 3), ({"tokens": A + 2}, 5), ({"nxt": A + 1}, 5),
    ({"logits": A + 1}, 5), ({"ws": A + 128}, 5), ({"nbytes": 1000}, 6),
    ({"pages": {"layers": 27}}, 6), ({"pages": {"kv_heads": 16}}, 6), ({"pages": {"head_dim": 64}}, 6),
    ({"pages": {"page_size": 8}}, 6), ({"pages": {"k": None}}, 3), ({"pages": {"k_scale": A}}, 3),
    ({"batch": {"rows": 129, "start": A}}, 6), ({"batch": {"max_rows": 4, "start": A}}, 6),
    ({"batch": {"seqs": 0}}, 6), ({"batch": {"table": None}}, 3), ({"batch": {"rows": 5}}, 6)])
def test_step_refusals(Q, D, P, kw, code):
    assert call(Q, D, P, **kw) == code
    assert Q.last_error()


def test_step_workspace_bytes(Q):
    f = Q.load_library().qwen3_pages_workspace_bytes
    assert [f(0, 1), f(129, 1), f(5, 0), f(5, 6), f(-1, -1)] == [0] * 5
    for rows in (1, 16, 17, 64, 65, 128):
        sizes = [f(rows, m) for m in range(1, rows + 1)]
        assert sizes[0] > 0 and sizes == sorted(sizes)
    for m in (1, 8, 9, 16, 17, 32):
        sizes = [f(rows, m) for rows in range(m, 129)]
        assert sizes == sorted(sizes)
