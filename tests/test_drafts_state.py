"""What a DraftSession remembers between its calls, and the calls it refuses, on the CPU:
the library's calls are recorded in place of being made."""
from __future__ import annotations

import numpy as np
import pytest


class Words:
    """Stands for a DeviceBuffer; downloads zeros."""

    ptr, nbytes = 0x10000, 1 << 20

    def __int__(self):
        return self.ptr

    def upload(self, array, offset=0):
        pass

    def download(self, dtype, count, offset=0):
        return np.zeros(count, dtype)


@pytest.fixture
def session(Q, monkeypatch):
    from qwen3_iree_amd import decode, drafts

    s = object.__new__(drafts.DraftSession)
    s.model = type("Model", (), {"ref": staticmethod(lambda: None)})()
    s.max_seq, s.max_nodes, s.length, s.position, s.stream = 100, 8, 20, 20, None
    s.k_cache = s.v_cache = s.state = s._ws = s._nodes = s.tree_logits = Words()
    s._q = s._lse = s._weights = s._tree = None
    s.calls = []
    monkeypatch.setattr(Q, "_call", lambda name, *a: s.calls.append(name))
    monkeypatch.setattr(Q, "synchronize", lambda: None)
    monkeypatch.setattr(decode.DecodeSession, "prefill_batched", lambda self, t: None)
    return s


def test_a_prompt_drops_the_verified_tree(session):
    s = session
    s.verify([1, 2, 3], [-1, 0, 0])
    s.prompt([5, 6, 7, 8])
    assert s.length == s.position == 24
    s.calls.clear()
    with pytest.raises(ValueError, match="no tree"):
        s.accept([0, 1])
    assert not s.calls and s.length == 24
    s.verify([1], [-1])
    s.accept([0])
    assert s.calls[-1] == "f16_cache_compact" and s.length == 25


def test_a_refused_prompt_keeps_the_tree(session):
    s = session
    s.verify([1, 2, 3], [-1, 0, 0])
    for bad in ([], np.zeros(81)):
        with pytest.raises(ValueError):
            s.prompt(bad)
    s.accept([0, 2])
    assert s.length == 22


def test_every_call_by_the_device_words_is_refused(session):
    """The parts of a decode step read or write the token or position word too."""
    for name, args in (("layer", (0, Words(), Words())), ("embed", (Words(),)), ("head", (Words(),))):
        with pytest.raises(TypeError):
            getattr(session, name)(*args)
    assert not session.calls


def test_a_draft_may_keep_and_change_its_context(session, monkeypatch):
    """The tokens so far are the draft's own copy."""
    s = session
    monkeypatch.setattr(type(s), "verify", lambda self, t, p: np.arange(100, 100 + len(t)))
    monkeypatch.setattr(type(s), "accept", lambda self, path: None)
    seen = []

    def draft(context):
        seen.append(context)
        context += [7, 7]
        return [], []

    out = s.generate_drafted(3, 4, -1, draft)
    assert out.tolist() == [100] * 4
    assert seen == [[3, 7, 7], [3, 100, 7, 7], [3, 100, 100, 7, 7], [3, 100, 100, 100, 7, 7]]


def test_a_refused_eviction_changes_nothing(Q, session, monkeypatch):
    """The verified tree can still be accepted behind it."""
    from qwen3_iree_amd import cache as C

    s = session
    s._weights, s.cache = Words(), None

    class Buffer(Words):
        def __init__(self, nbytes):
            pass

        def __enter__(self):
            return self

        def __exit__(self, *exc):
            pass

        def download(self, dtype, count=28 * 8 * 10, offset=0):
            return np.zeros(count, dtype)

    def select(cache, length, budget, *args):
        if not 1 <= budget <= length:
            raise Q.Q8GemvError(6, "budget")

    monkeypatch.setattr(Q, "DeviceBuffer", Buffer)
    monkeypatch.setattr(C, "cache_select", select)
    monkeypatch.setattr(C, "cache_compact", lambda *a: None)
    monkeypatch.setattr(C, "attn_weights_add", lambda *a: None)
    s.verify([1, 2], [-1, 0])
    for budget in (0, 21, 10 ** 12):
        with pytest.raises(Q.Q8GemvError):
            s.evict(budget)
    assert s.length == 20
    s.accept([0])
    assert s.length == s.position == 21
    s.verify([1, 2], [-1, 0])
    assert s.evict(10).shape == (28, 8, 10) and s.length == 10 and s.position == 21
    with pytest.raises(ValueError, match="no tree"):
        s.accept([0])


def test_weights_that_are_not_kept_are_refused(session):
    with pytest.raises(ValueError, match="no attention weights"):
        session.slot_weights()
    with pytest.raises(ValueError, match="no attention weights"):
        session.evict(5)
