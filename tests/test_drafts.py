"""CPU-side checks of the drafted-tree calls: refusals before the device is touched,
workspace sizes, and the choice of the accepted path."""
from __future__ import annotations

import ctypes

import pytest

A = 0x10000


@pytest.fixture(scope="module")
def D(Q):
    from qwen3_iree_amd import decode

    return decode


def weights(D):
    return D.WeightsC(*([A] * len(D.WEIGHT_FIELDS)), None)


GOOD = dict(k=A, v=A, max_seq=100, tokens=A, parents=A, n=4, len=10, position=10, nxt=A, logits=A,
            q=A, lse=A, ws=A, nbytes=1 << 40)


def call(Q, D, **kw):
    a = {**GOOD, **kw}
    w = weights(D)
    return Q.load_library().qwen3_tree_step(
        ctypes.byref(w), a["k"], a["v"], a["max_seq"], a["tokens"], a["parents"], a["n"], a["len"],
        a["position"], a["nxt"], a["logits"], a["q"], a["lse"], a["ws"], a["nbytes"], None)


@pytest.mark.parametrize("kw,code", [
    ({"k": None}, 3), ({"v": None}, 3), ({"tokens": None}, 3), ({"parents": None}, 3),
    ({"nxt": None}, 3), ({"ws": None}, 3), ({"q": None}, 3), ({"lse": None}, 3), ({"k": A + 8}, 5),
    ({"tokens": A + 2}, 5), ({"parents": A + 1}, 5), ({"nxt": A + 2}, 5), ({"logits": A + 1}, 5),
    ({"q": A + 8}, 5), ({"lse": A + 2}, 5), ({"ws": A + 128}, 5), ({"n": 0}, 6), ({"n": 257}, 6),
    ({"len": -1}, 6), ({"len": 97}, 6), ({"len": 2 ** 31 - 1}, 6), ({"max_seq": 0}, 6),
    ({"position": -1}, 6), ({"position": (1 << 24) + 1}, 6), ({"nbytes": 1000}, 6)])
def test_refusals(Q, D, kw, code):
    assert call(Q, D, **kw) == code
    assert Q.last_error()


def test_null_weights(Q):
    assert Q.load_library().qwen3_tree_step(None, A, A, 100, A, A, 4, 10, 10, A, A, A, A, A,
                                            1 << 40, None) == 3


def test_workspace_bytes(Q):
    f = Q.load_library().qwen3_tree_workspace_bytes
    assert [f(0, 100), f(257, 1000), f(5, 4), f(1, (1 << 24) + 1)] == [0, 0, 0, 0]
    for n in (1, 12, 64, 65, 256):
        sizes = [f(n, s) for s in (n, n + 1, 1000, 5000, 1 << 20)]
        assert sizes[0] > 0 and sizes == sorted(sizes)
        assert sizes[0] > Q.load_library().qwen3_prefill_workspace_bytes(n)


def test_greedy_path(Q):
    from qwen3_iree_amd import drafts

    tokens, parents = [5, 7, 8, 9, 7, 3], [-1, 0, 0, 2, 2, 3]
    assert drafts.greedy_path(tokens, parents, [8, 0, 9, 3, 0, 0]) == [0, 2, 3, 5]
    assert drafts.greedy_path(tokens, parents, [7, 9, 9, 3, 0, 0]) == [0, 1]
    assert drafts.greedy_path(tokens, parents, [1, 0, 0, 0, 0, 0]) == [0]
    assert drafts.greedy_path([5], [-1], [5]) == [0]


def test_session_refuses_bad_sizes(Q, D):
    from qwen3_iree_amd import drafts

    for max_seq, nodes in ((100, 0), (100, 257), (10, 11)):
        with pytest.raises(ValueError):
            drafts.DraftSession(None, max_seq, nodes)


def test_session_refuses_the_calls_by_device_words(Q, D):
    from qwen3_iree_amd import drafts

    s = object.__new__(drafts.DraftSession)
    for name, args in (("step", ()), ("step_checked", ()), ("capture", ()), ("replay", ()),
                       ("prefill", ([1],)), ("prefill_batched", ([1],)), ("generate", (4, 0))):
        assert hasattr(D.DecodeSession, name)
        with pytest.raises(TypeError):
            getattr(s, name)(*args)
