"""Sequences handed over to flat sessions, and steps that fail before their launch, on the CPU: the
library's calls are recorded in place of being made."""
from __future__ import annotations

import numpy as np
import pytest

from test_serving import make  # noqa: F401  (a fixture)


class Flat:
    """The parts of a DecodeSession that a hand-over uses."""
    max_seq, stream, k_cache, v_cache = 40, None, 0x10000, 0x10000

    def __init__(self):
        self.state = (11, 3)

    def synchronize(self):
        pass

    def get_state(self):
        return self.state

    def set_state(self, token, pos):
        self.state = (token, pos)


def test_a_flat_session_takes_the_sequence(make):
    s = make()
    a = s.add()
    s.step({a: np.zeros(20)})
    flat = Flat()
    s.to_session(a, flat)
    assert flat.state == (11, 20) and s.calls[-1] == "kv_pages_read"


def test_a_session_of_drafted_trees_is_refused(make):
    """It goes by slots and positions of its own, which a hand-over would leave as they were."""
    from qwen3_iree_amd import drafts

    class Trees(Flat, drafts.DraftSession):
        pass

    s = make()
    a = s.add()
    s.step({a: np.zeros(20)})
    calls, flat = len(s.calls), Trees()
    flat.length = flat.position = 7
    with pytest.raises(TypeError, match="drafted trees"):
        s.to_session(a, flat)
    assert len(s.calls) == calls and flat.state == (11, 3) and flat.length == flat.position == 7


def test_a_step_without_room_for_its_logits_takes_no_pages(make, Q, monkeypatch):
    """Pages that a refused step kept would be counted as room for others' rows."""
    s = make()
    a, b = s.add(), s.add()
    s.step({a: np.zeros(10)})

    def full(nbytes):
        raise Q.Q8GemvError(8, "out of memory")

    monkeypatch.setattr(Q, "DeviceBuffer", full)
    with pytest.raises(Q.Q8GemvError):
        s.step({a: np.zeros(50)}, logits=True)
    assert len(s._held[a]) == 1 and len(s._free) == 5 and s.length[a] == 10
    s.step({a: [1], b: np.zeros(64)})
    assert len(s._held[a]) == 1 and len(s._held[b]) == 4
