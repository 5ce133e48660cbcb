"""CPU-side checks of include/f16_cache.h: declared, exported and bound, and every
argument outside its contract refused with a status before the device is touched."""
from __future__ import annotations

import ctypes
import math
import re
from pathlib import Path

import numpy as np
import pytest

REPO = Path(__file__).resolve().parent.parent
A = 0x10000  # fake, aligned "device" addresses: never dereferenced here


@pytest.fixture(scope="module")
def C(Q):
    from qwen3_iree_amd import cache

    return cache


def test_declared_exported_and_bound(Q):
    text = re.sub(r"/\*.*?\*/", "", (REPO / "include" / "f16_cache.h").read_text(), flags=re.S)
    names = re.findall(r"^(?:int|int64_t|void|size_t)\s+(\w+)\s*\(", text, flags=re.M)
    assert set(names) == set(Q._CACHE_SIGNATURES)
    lib = Q.load_library()
    assert all(hasattr(lib, n) for n in names)


def test_struct_layout(C):
    assert ctypes.sizeof(C.Cache) == 48
    assert [getattr(C.Cache, f).offset for f, _ in C.Cache._fields_] == [0, 8, 16, 24, 32, 36, 40]


def test_code_object(Q):
    data = (REPO / "qwen3-iree_amd" / "lib" / "cache_gfx950.hsaco").read_bytes()
    assert data[:4] == b"\x7fELF" and b"amdgcn-amd-amdhsa--gfx950" in data


def refused(Q, code, fn, *args, **kw):
    with pytest.raises(Q.Q8GemvError) as e:
        fn(*args, **kw)
    assert e.value.code == code, e.value
    assert e.value.message


CACHE = dict(k=A, v=A, max_seq=100, layers=2, kv_heads=2, head_dim=64, weights=A)


def cache(C, **kw):
    return C.Cache(**{**CACHE, **kw})


BAD_CACHES = [({"max_seq": 0}, 6), ({"max_seq": (1 << 24) + 1}, 6), ({"layers": 0}, 6),
              ({"layers": 1025}, 6), ({"kv_heads": 0}, 6), ({"kv_heads": 257}, 6),
              ({"head_dim": 96}, 6), ({"head_dim": 256}, 6), ({"k": A + 8}, 5), ({"v": A + 2}, 5),
              ({"weights": A + 2}, 5)]


@pytest.mark.parametrize("kw,code", BAD_CACHES)
def test_bad_caches(Q, C, kw, code):
    bad, good = cache(C, **kw), cache(C)
    refused(Q, code, C.attn_tree, bad, 0, 5, A, 256, 4, A, 2, 0.125, A, 256, A, A, 1 << 30)
    refused(Q, code, C.attn_weights_add, bad, 5, A, 0, 256, 4, A, 0, 2, None, 2, 0.125)
    refused(Q, code, C.cache_select, bad, 10, 5, 0, 0, A)
    refused(Q, code, C.cache_compact, bad, good, A, True, 0, 5)
    refused(Q, code, C.cache_compact, good, bad, A, True, 0, 5)


def test_null_caches(Q):
    lib = Q.load_library()
    assert lib.f16_attn_tree(None, 0, 5, A, 256, 4, A, 2, 0.125, A, 256, A, A, 1 << 30, None) == 3
    assert lib.f16_attn_weights_add(None, 5, A, 0, 256, 4, A, 0, 2, None, 2, 0.125, None) == 3
    assert lib.f16_cache_select(None, 10, 5, 0, 0, A, None) == 3
    assert lib.f16_cache_compact(None, None, A, 1, 0, 5, None) == 3


TREE = dict(layer=0, length=5, q=A, q_stride=256, q_heads=4, mask=A, n=2, scale=0.125, out=A,
            out_stride=256, lse=A, workspace=A, workspace_bytes=1 << 30)


@pytest.mark.parametrize("kw,code", [
    ({"layer": -1}, 4), ({"layer": 2}, 4), ({"q": None}, 3), ({"out": None}, 3),
    ({"q": A + 8}, 5), ({"out": A + 8}, 5), ({"mask": A + 1}, 5), ({"lse": A + 2}, 5),
    ({"q_heads": 0}, 6), ({"q_heads": 3}, 6), ({"q_heads": 66}, 6), ({"q_heads": 258}, 6),
    ({"n": 0}, 6), ({"n": 257}, 6), ({"n": -1}, 6), ({"length": -1}, 6), ({"length": 99}, 6),
    ({"length": 2 ** 31 - 1}, 6), ({"q_stride": 248}, 6), ({"q_stride": 260}, 6),
    ({"q_stride": -256}, 6), ({"out_stride": 255}, 6), ({"out_stride": 128}, 6),
    ({"scale": 0.0}, 9), ({"scale": -1.0}, 9), ({"scale": math.inf}, 9), ({"scale": math.nan}, 9)])
def test_tree_refusals(Q, C, kw, code):
    refused(Q, code, C.attn_tree, cache(C), **{**TREE, **kw})


def test_tree_refuses_a_cache_without_k_or_v(Q, C):
    refused(Q, 3, C.attn_tree, cache(C, k=None), **TREE)
    refused(Q, 3, C.attn_tree, cache(C, v=None), **TREE)


@pytest.mark.parametrize("args,code", [
    ((None, 4, A, A), 3), ((A, 4, None, A), 3), ((A + 2, 4, A, A), 5), ((A, 4, A + 1, A), 5),
    ((A, 4, A, A + 2), 5), ((A, 0, A, A), 6), ((A, 257, A, A), 6), ((A, -3, A, None), 6)])
def test_mask_refusals(Q, C, args, code):
    refused(Q, code, C.tree_mask, *args)


WEIGHTS = dict(length=5, q=A, q_layer_stride=512, q_stride=256, q_heads=4, lse=A,
               lse_layer_stride=8, rows=2, path=A, n=2, scale=0.125)


@pytest.mark.parametrize("kw,code", [
    ({"q": None}, 3), ({"lse": None}, 3), ({"q": A + 8}, 5), ({"lse": A + 1}, 5),
    ({"path": A + 2}, 5), ({"q_heads": 5}, 6), ({"n": 0}, 6), ({"n": 257}, 6),
    ({"length": 99}, 6), ({"length": -1}, 6), ({"rows": 0}, 6), ({"rows": (1 << 20) + 1}, 6),
    ({"path": None, "n": 3}, 6), ({"q_stride": 200}, 6), ({"q_layer_stride": 4}, 6),
    ({"q_layer_stride": -512}, 6), ({"lse_layer_stride": -1}, 6), ({"scale": math.nan}, 9)])
def test_weights_refusals(Q, C, kw, code):
    refused(Q, code, C.attn_weights_add, cache(C), **{**WEIGHTS, **kw})
    refused(Q, 3, C.attn_weights_add, cache(C, weights=None), **WEIGHTS)
    refused(Q, 3, C.attn_weights_add, cache(C, k=None), **WEIGHTS)


@pytest.mark.parametrize("args,code", [
    ((10, 5, 0, 0, None), 3), ((10, 5, 0, 0, A + 2), 5), ((101, 5, 0, 0, A), 6),
    ((10, 0, 0, 0, A), 6), ((10, 11, 0, 0, A), 6), ((0, 0, 0, 0, A), 6), ((-1, 1, 0, 0, A), 6),
    ((10, 5, -1, 0, A), 6), ((10, 5, 0, -1, A), 6), ((10, 5, 3, 3, A), 6),
    ((10, 5, 2 ** 31 - 1, 2 ** 31 - 1, A), 6)])
def test_select_refusals(Q, C, args, code):
    refused(Q, code, C.cache_select, cache(C), *args)
    refused(Q, 3, C.cache_select, cache(C, weights=None), 10, 5, 0, 0, A)


def test_compact_refusals(Q, C):
    good, other = cache(C), cache(C, k=2 * A, v=2 * A, weights=2 * A, max_seq=50)
    refused(Q, 3, C.cache_compact, cache(C, k=None), other, A, True, 0, 5)
    refused(Q, 3, C.cache_compact, good, cache(C, v=None), A, True, 0, 5)
    refused(Q, 3, C.cache_compact, good, other, None, True, 0, 5)
    refused(Q, 5, C.cache_compact, good, other, A + 1, True, 0, 5)
    for kw in ({"layers": 1}, {"kv_heads": 1}, {"head_dim": 128}):
        refused(Q, 6, C.cache_compact, good, cache(C, k=2 * A, v=2 * A, weights=2 * A, **kw), A,
                True, 0, 5)
    for base, count in ((-1, 5), (0, -1), (0, 51), (46, 5), (2 ** 31 - 1, 2 ** 31 - 1)):
        refused(Q, 6, C.cache_compact, good, other, A, True, base, count)
    # caches that share only part of their buffers
    refused(Q, 9, C.cache_compact, good, cache(C, v=2 * A), A, True, 0, 5)
    refused(Q, 9, C.cache_compact, good, cache(C, max_seq=99), A, True, 0, 5)
    refused(Q, 9, C.cache_compact, good, cache(C, weights=2 * A), A, True, 0, 5)


@pytest.mark.parametrize("args,code", [
    ((None, 10, A, 2, A, A, A), 3), ((A, 10, None, 2, A, A, A), 3), ((A, 10, A, 2, A, None, A), 3),
    ((A, 10, A, 2, A, A, None), 3), ((A, 0, A, 2, A, A, A), 6), ((A, 1 << 31, A, 2, A, A, A), 6),
    ((A, 10, A, 0, A, A, A), 6), ((A, 10, A, 257, A, A, A), 6), ((A + 8, 10, A, 2, A, A, A), 5),
    ((A, 10, A + 4, 2, A, A, A), 5), ((A, 10, A, 2, A + 1, A, A), 5),
    ((A, 10, A, 2, A, A + 2, A), 5), ((A, 10, A, 2, A, A, A + 8), 5)])
def test_vocab_refusals(Q, args, code):
    refused(Q, code, Q.f16_gemm_argmax, *args)


def test_workspace_sizes(Q, C):
    assert [Q.gemm_argmax_workspace_bytes(n) > 0 for n in (0, 1, 256, 257)] == [False, True, True, False]
    c = C.Cache(A, A, 1 << 20, 1, 8, 128)
    for n in (1, 5, 64, 256):
        sizes = [C.attn_tree_workspace_bytes(c, length, n, 16)
                 for length in (0, 1, 31, 300, 1000, 4096, 16384, 100000, (1 << 20) - n)]
        assert sizes == sorted(sizes)
    # arguments that f16_attn_tree refuses have no workspace
    for length, n, qh in ((-1, 1, 16), (0, 0, 16), (0, 257, 16), (0, 1, 12), (1 << 20, 1, 16)):
        assert C.attn_tree_workspace_bytes(c, length, n, qh) == 0


def test_calls_before_init_report_it(Q, C):
    import subprocess
    import sys

    code = f"""
import sys; sys.path.insert(0, {str(REPO / 'tests')!r})
import conftest
from qwen3_iree_amd import q8gemv as Q, cache as C
c = C.Cache({A}, {A}, 100, 2, 2, 64, {A})
for f, a in ((C.tree_mask, ({A}, 3, {A})), (C.cache_select, (c, 10, 5, 0, 0, {A})),
             (C.cache_compact, (c, c, {A}, True, 0, 5)),
             (Q.f16_gemm_argmax, ({A}, 10, {A}, 2, None, {A}, {A}))):
    try:
        f(*a)
    except Q.Q8GemvError as e:
        assert e.code == 1, e
    else:
        raise SystemExit('no error')
"""
    subprocess.run([sys.executable, "-c", code], check=True, timeout=120)


def test_reference_forms_agree_with_a_second_writing():
    """The plain forms used on the GPU tests, against direct sums."""
    import cache_ref as R

    rng = np.random.default_rng(0)
    n, length, qh, kvh, d = 5, 9, 4, 2, 8
    q, k, v = (rng.standard_normal(s) for s in ((n, qh, d), (length + n, kvh, d), (length + n, kvh, d)))
    parents = [-1, 0, 0, 2, 7]
    see = R.tree_see(parents)
    assert see.sum(1).tolist() == [1, 2, 2, 3, 0]
    out, lse, _, _ = R.attention(q, k, v, see, length, 0.5)
    for i in range(n):
        for h in range(qh):
            js = list(range(length)) + [length + j for j in range(n) if see[i, j]]
            if not see[i].any():
                assert (out[i, h] == 0).all() and lse[i, h] == -np.inf
                continue
            e = np.array([np.exp(0.5 * sum(q[i, h, t] * k[j, h // 2, t] for t in range(d))) for j in js])
            assert np.isclose(lse[i, h], np.log(e.sum()))
            assert np.allclose(out[i, h], (e / e.sum()) @ v[js, h // 2])
    assert R.pack_mask(see).tolist() == [[1], [3], [5], [13], [0]]
    w = np.array([[5, 1, 3, 3, 2, 3, 0]], np.float32)
    assert R.select(w, 7, 4, 1, 1).tolist() == [[0, 2, 3, 6]]


@pytest.mark.parametrize("qh,kvh,d", [(16, 8, 128), (64, 2, 64), (256, 64, 128), (32, 1, 64), (1, 1, 128)])
def test_workspace_does_not_shrink_over_every_rule(Q, C, qh, kvh, d):
    lengths = sorted({*range(0, 700, 13), *(2 ** i + j for i in range(9, 24) for j in (-257, 0, 31, 999))})
    for n in (1, 2, 7, 9, 17, 31, 33, 61, 64, 65, 100, 129, 200, 256):
        c = C.Cache(0x10000, 0x10000, 1 << 24, 1, kvh, d)
        sizes = [C.attn_tree_workspace_bytes(c, length, n, qh) for length in lengths]
        assert sizes == sorted(sizes), n
