"""Which sessions PagedSession.to_session hands a sequence over to, on the CPU: the library's
calls are recorded in place of being made."""
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
