"""Workspace sizes of tree attention and of the model's tree step: one sized for the
largest tree of a session serves every smaller one, over any part of the cache."""
from __future__ import annotations

import pytest

A = 0x10000


@pytest.fixture(scope="module")
def C(Q):
    from qwen3_iree_amd import cache

    return cache


@pytest.mark.parametrize("max_seq", [256, 300, 511, 1000, 2048, 4999, 8192, 16384, 70000, 1 << 20])
@pytest.mark.parametrize("qh,kvh,d", [(16, 8, 128), (14, 2, 64), (9, 3, 64), (64, 2, 64), (32, 1, 64),
                                      (256, 64, 128), (1, 1, 128), (28, 4, 128)])
def test_the_largest_tree_serves_all(Q, C, qh, kvh, d, max_seq):
    c = C.Cache(A, A, max_seq, 1, kvh, d)
    sizes = [C.attn_tree_workspace_bytes(c, max_seq - n, n, qh) for n in range(1, 257)]
    assert sizes == sorted(sizes)
    for n in (1, 2, 16, 17, 31, 32, 33, 63, 64, 65, 100, 128, 129, 200, 255, 256):
        for length in {0, 1, 31, 200, max_seq // 3, max_seq // 2 - n, max_seq - n - 1, max_seq - n}:
            if 0 <= length <= max_seq - n:
                need = C.attn_tree_workspace_bytes(c, length, n, qh)
                assert all(need <= s for s in sizes[n - 1:])


@pytest.mark.parametrize("length", [0, 33, 700, 5000, 16384])
def test_more_rows_need_no_less(Q, C, length):
    c = C.Cache(A, A, 1 << 16, 1, 8, 128)
    sizes = [C.attn_tree_workspace_bytes(c, length, n, 16) for n in range(1, 257)]
    assert sizes == sorted(sizes)


@pytest.mark.parametrize("max_seq", [256, 1000, 4096, 8192, 16384, 1 << 20])
def test_the_step_of_the_largest_tree_serves_all(Q, max_seq):
    sizes = [Q.load_library().qwen3_tree_workspace_bytes(n, max_seq) for n in range(1, 257)]
    assert sizes[0] > 0 and sizes == sorted(sizes)
