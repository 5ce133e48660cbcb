"""CPU-side checks of include/kv_pages.h: declared, exported and bound, struct layouts, and
every argument outside its contract refused with a status before the device is touched."""
from __future__ import annotations

import ctypes
import math
import re
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest

REPO = Path(__file__).resolve().parent.parent
A = 0x10000  # fake, aligned "device" addresses: never dereferenced here


@pytest.fixture(scope="module")
def P(Q):
    from qwen3_iree_amd import pages

    return pages


def test_declared_exported_and_bound(Q):
    text = re.sub(r"/\*.*?\*/", "", (REPO / "include" / "kv_pages.h").read_text(), flags=re.S)
    names = re.findall(r"^(?:int|int64_t|void|size_t)\s+(\w+)\s*\(", text, flags=re.M)
    assert set(names) == set(Q._PAGES_SIGNATURES)
    lib = Q.load_library()
    assert all(hasattr(lib, n) for n in names)


def test_struct_layouts(P, tmp_path):
    """The ctypes structs against what a C compiler makes of the header."""
    structs = {"kv_pages": P.Pages, "kv_batch": P.Batch, "kv_rows": P.Rows, "kv_drafts": P.Drafts}
    lines = [f'printf("{s}.{f} %zu\\n", offsetof({s}, {f}));' for s, c in structs.items()
             for f, _ in c._fields_] + [f'printf("{s} %zu\\n", sizeof({s}));' for s in structs]
    src = tmp_path / "layout.c"
    src.write_text('#include "kv_pages.h"\n#include <stdio.h>\nint main(void) {\n'
                   + "\n".join(lines) + "\nreturn 0;\n}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", f"-I{REPO / 'include'}", str(src), "-o", str(exe)], check=True)
    out = dict(l.split() for l in subprocess.run([str(exe)], check=True, capture_output=True,
                                                 text=True).stdout.splitlines())
    for s, c in structs.items():
        assert int(out[s]) == ctypes.sizeof(c)
        for f, _ in c._fields_:
            assert int(out[f"{s}.{f}"]) == getattr(c, f).offset, (s, f)


def test_packed_structs(P):
    """The packed forms that append and verify pass, against the structures."""
    for packed, struct in ((P._ROWS, P.Rows), (P._DRAFTS, P.Drafts)):
        values = [0.5 * i if t is ctypes.c_double else i + 1 for i, (_, t) in enumerate(struct._fields_)]
        assert packed.size == ctypes.sizeof(struct)
        got = struct.from_buffer_copy(packed.pack(*values))
        assert [getattr(got, f) for f, _ in struct._fields_] == values


def test_code_object(Q):
    data = (REPO / "qwen3-iree_amd" / "lib" / "pages_gfx950.hsaco").read_bytes()
    assert data[:4] == b"\x7fELF" and b"amdgcn-amd-amdhsa--gfx950" in data


def refused(Q, code, fn, *args, **kw):
    with pytest.raises(Q.Q8GemvError) as e:
        fn(*args, **kw)
    assert e.value.code == code, e.value
    assert e.value.message


PAGES = dict(k=A, v=A, pages=10, page_size=16, layers=2, kv_heads=2, head_dim=64)
BATCH = dict(table=A, length=A, seqs=3, max_pages=4, rows=3, max_rows=1)
APPEND = dict(k=A, k_stride=128, v=A, v_stride=128, k_norm=A, q=A, q_stride=256, q_heads=4,
              q_norm=A, q_out=A * 16, q_out_stride=256, theta=1e6)
ATTN = dict(q=A, q_stride=256, q_heads=4, scale=0.125, out=2 * A, out_stride=256, lse=A, workspace=A,
            workspace_bytes=1 << 40)
READ = dict(layer=0, layers=2, k_out=A, v_out=A, row_stride=128, layer_stride=1024)


def pages(P, **kw):
    return P.Pages(**{**PAGES, **kw})


def batch(P, **kw):
    return P.Batch(**{**BATCH, **kw})


def every(Q, P, code, pool, b):
    refused(Q, code, P.append, pool, 0, b, **APPEND)
    refused(Q, code, P.attn, pool, 0, b, **ATTN)
    refused(Q, code, P.read, pool, batch=b, **READ)


Q8 = dict(k_scale=A, v_scale=A)


@pytest.mark.parametrize("kw,code", [
    ({"pages": 0}, 6), ({"pages": (1 << 24) + 1}, 6), ({"layers": 0}, 6), ({"layers": 1025}, 6),
    ({"kv_heads": 0}, 6), ({"kv_heads": 257}, 6), ({"head_dim": 96}, 6), ({"head_dim": 256}, 6),
    ({"page_size": 0}, 6), ({"page_size": 8}, 6), ({"page_size": 24}, 6), ({"page_size": 4112}, 6),
    ({"page_size": -16}, 6), ({"k": None}, 3), ({"v": None}, 3), ({"k": A + 8}, 5), ({"v": A + 2}, 5),
    ({"k_scale": A}, 3), ({"v_scale": A}, 3), ({**Q8, "k_scale": A + 4}, 5), ({**Q8, "v_scale": A + 8}, 5)])
def test_bad_pages(Q, P, kw, code):
    every(Q, P, code, pages(P, **kw), batch(P))


def test_bad_type_and_nulls(Q, P):
    pool = pages(P)
    pool.type = 2
    every(Q, P, 2, pool, batch(P))
    lib = Q.load_library()
    good, b, x = pages(P), batch(P), P.Rows()
    ref = ctypes.byref
    assert lib.kv_pages_append(None, 0, ref(b), ref(x), None) == 3
    assert lib.kv_pages_append(ref(good), 0, None, ref(x), None) == 3
    assert lib.kv_pages_append(ref(good), 0, ref(b), None, None) == 3
    assert lib.kv_pages_attn(None, 0, ref(b), A, 256, 4, 0.1, A, 256, A, A, 1 << 30, None) == 3
    assert lib.kv_pages_attn(ref(good), 0, None, A, 256, 4, 0.1, A, 256, A, A, 1 << 30, None) == 3
    assert lib.kv_pages_read(None, 0, 1, ref(b), A, A, 128, 0, None) == 3
    assert lib.kv_pages_read(ref(good), 0, 1, None, A, A, 128, 0, None) == 3
    assert lib.kv_verify(None, A, 1 << 30, None) == 3


@pytest.mark.parametrize("kw,code", [
    ({"table": None}, 3), ({"length": None}, 3), ({"table": A + 2}, 5), ({"length": A + 1}, 5),
    ({"start": A + 2}, 5), ({"seqs": 0}, 6), ({"seqs": 1025, "rows": 1025}, 6), ({"rows": 0}, 6),
    ({"rows": (1 << 23) + 1, "start": A}, 6), ({"rows": 2}, 6), ({"rows": 4}, 6),
    ({"max_rows": 0}, 6), ({"max_rows": -1}, 6), ({"max_rows": (1 << 23) + 1}, 6),
    ({"max_pages": 0}, 6), ({"max_pages": (1 << 20) + 1}, 6), ({"max_pages": 2 ** 31 - 1}, 6),
    ({"table_stride": 3}, 6)])
def test_bad_batches(Q, P, kw, code):
    every(Q, P, code, pages(P), batch(P, **kw))


@pytest.mark.parametrize("layer", [-1, 2, 2 ** 31 - 1])
def test_layers(Q, P, layer):
    refused(Q, 4, P.append, pages(P), layer, batch(P), **APPEND)
    refused(Q, 4, P.attn, pages(P), layer, batch(P), **ATTN)
    refused(Q, 4, P.read, pages(P), batch=batch(P), **{**READ, "layer": layer, "layers": 1})


@pytest.mark.parametrize("kw,code", [
    ({"k": None}, 3), ({"v": None}, 3), ({"q_out": None}, 3), ({"q": None}, 3), ({"k": A + 8}, 5),
    ({"v": A + 2}, 5), ({"q": A + 8}, 5), ({"q_out": A + 4}, 5), ({"k_norm": A + 1}, 5),
    ({"q_norm": A + 1}, 5), ({"positions": A + 2}, 5), ({"k_stride": 120}, 6), ({"v_stride": 132}, 6),
    ({"k_stride": -128}, 6), ({"q_stride": 248}, 6), ({"q_out_stride": 128}, 6), ({"q_heads": 0}, 6),
    ({"q_heads": 3}, 6), ({"q_heads": 66}, 6), ({"q_out": A, "q_out_stride": 512}, 9),
    ({"eps": -1.0}, 9), ({"eps": math.nan}, 9), ({"eps": math.inf}, 9), ({"theta": -1.0}, 9),
    ({"theta": math.nan}, 9), ({"theta": math.inf}, 9)])
def test_append_refusals(Q, P, kw, code):
    refused(Q, code, P.append, pages(P), 0, batch(P), **{**APPEND, **kw})


@pytest.mark.parametrize("kw,code", [
    ({"q": None}, 3), ({"out": None}, 3), ({"q": A + 8}, 5), ({"out": A + 8}, 5), ({"lse": A + 2}, 5),
    ({"q_heads": 0}, 6), ({"q_heads": 3}, 6), ({"q_heads": 66}, 6), ({"q_heads": 258}, 6),
    ({"q_stride": 248}, 6), ({"q_stride": 260}, 6), ({"out_stride": 255}, 6), ({"out_stride": 128}, 6),
    ({"scale": 0.0}, 9), ({"scale": -1.0}, 9), ({"scale": math.inf}, 9), ({"scale": math.nan}, 9),
    ({"scale": 2.0 ** 127.8}, 9), ({"out": A}, 9), ({"workspace": A + 16}, 5)])
def test_attn_refusals(Q, P, kw, code):
    refused(Q, code, P.attn, pages(P), 0, batch(P), **{**ATTN, **kw})


def test_attn_rows_of_a_sequence(Q, P):
    refused(Q, 6, P.attn, pages(P), 0, batch(P, max_rows=257, start=A), **ATTN)


@pytest.mark.parametrize("kw,code", [
    ({"layers": 0}, 4), ({"layers": 3}, 4), ({"layer": 1}, 4), ({"k_out": A + 8}, 5), ({"v_out": A + 2}, 5),
    ({"row_stride": 120}, 6), ({"row_stride": 132}, 6), ({"row_stride": -128}, 6),
    ({"layer_stride": 4}, 6), ({"layer_stride": -1024}, 6), ({"layer_stride": 0}, 6)])
def test_read_refusals(Q, P, kw, code):
    refused(Q, code, P.read, pages(P), batch=batch(P), **{**READ, **kw})


VERIFY = dict(logits=A, logits_stride=100, vocab=100, rows=6, tokens=A, seqs=2, max_rows=4, uniform=A,
              out=A, out_stride=4, accepted=A, start=A, temperature=A, draft=A, draft_stride=100,
              logprob=A, workspace=A, workspace_bytes=1 << 30)


@pytest.mark.parametrize("kw,code", [
    ({"logits": None}, 3), ({"tokens": None}, 3), ({"uniform": None}, 3), ({"out": None}, 3),
    ({"accepted": None}, 3), ({"workspace": None}, 3), ({"logits": A + 1}, 5), ({"tokens": A + 2}, 5),
    ({"uniform": A + 2}, 5), ({"out": A + 2}, 5), ({"accepted": A + 2}, 5), ({"start": A + 2}, 5),
    ({"temperature": A + 2}, 5), ({"draft": A + 2}, 5), ({"logprob": A + 2}, 5), ({"workspace": A + 16}, 5),
    ({"rows": 0}, 6), ({"rows": 65536}, 6), ({"seqs": 0}, 6), ({"seqs": 1025}, 6), ({"max_rows": 0}, 6),
    ({"max_rows": 257, "out_stride": 300}, 6), ({"vocab": 0}, 6), ({"vocab": (1 << 24) + 1}, 6),
    ({"logits_stride": 99}, 6), ({"draft_stride": 99}, 6), ({"out_stride": 3}, 6), ({"start": None}, 6),
    ({"workspace_bytes": 100}, 6)])
def test_verify_refusals(Q, P, kw, code):
    refused(Q, code, P.verify, **{**VERIFY, **kw})


def test_workspace_sizes(Q, P):
    assert P.verify_workspace_bytes(6, 2, 100) > 0
    for rows, seqs, vocab in ((0, 1, 10), (65536, 1, 10), (1, 0, 10), (1, 1025, 10), (1, 1, 0),
                              (1, 1, (1 << 24) + 1)):
        assert P.verify_workspace_bytes(rows, seqs, vocab) == 0
    # arguments that kv_pages_attn refuses have no workspace
    for qh in (0, 3, 66, 258):
        assert P.attn_workspace_bytes(pages(P), batch(P), qh) == 0
    assert P.attn_workspace_bytes(pages(P, head_dim=96), batch(P), 4) == 0
    assert P.attn_workspace_bytes(pages(P), batch(P, seqs=0), 4) == 0


def test_attn_workspace_of_the_largest_call_serves_all(Q, P):
    for qh, kvh, d in ((16, 8, 128), (64, 2, 64), (256, 64, 128), (32, 1, 64), (1, 1, 128), (256, 256, 64)):
        pool = pages(P, kv_heads=kvh, head_dim=d)
        sizes = [P.attn_workspace_bytes(pool, batch(P, start=A, rows=300, max_rows=m), qh)
                 for m in (1, 2, 3, 5, 8, 9, 16, 17, 31, 32, 33, 64, 65, 100, 128, 200, 256)]
        assert sizes == sorted(sizes)
        # whatever the sequences and their pages are
        for kw in (dict(seqs=1, rows=1), dict(seqs=1024, rows=1024), dict(max_pages=1 << 20),
                   dict(rows=5000)):
            assert P.attn_workspace_bytes(pool, batch(P, **{"start": A, **kw}), qh) == sizes[0]


def test_calls_before_init_report_it(Q):
    code = f"""
import sys; sys.path.insert(0, {str(REPO / 'tests')!r})
import test_pages_abi as T
from qwen3_iree_amd import q8gemv as Q, pages as P
b, p = T.batch(P), T.pages(P)
for f, a in ((P.append, (p, 0, b)), (P.attn, (p, 0, b)), (P.read, (p,)), (P.verify, ())):
    kw = {{P.append: T.APPEND, P.attn: T.ATTN, P.read: dict(T.READ, batch=b), P.verify: T.VERIFY}}[f]
    try:
        f(*a, **kw)
    except Q.Q8GemvError as e:
        assert e.code == 1, e
    else:
        raise SystemExit('no error')
"""
    subprocess.run([sys.executable, "-c", "import sys; sys.path.insert(0, %r); import conftest\n%s"
                    % (str(REPO / "tests"), code)], check=True, timeout=120)


def test_reference_forms_agree_with_a_second_writing():
    """The plain forms used on the GPU tests, against direct sums."""
    import pages_ref as R

    rng = np.random.default_rng(0)
    k, v = (rng.standard_normal((6, 2, 16, 4)).astype(np.float16) for _ in range(2))
    table = np.array([[3, 1], [5, -1]], np.int32)
    q = rng.standard_normal((3, 4, 4)).astype(np.float16)
    out, lse, _, _, mine = R.attention(q, (k, v, None, None), table, [20, 18], [0, 2, 3], 2, 0.5)
    assert mine.all()
    for r, s, n in ((0, 0, 19), (1, 0, 20), (2, 1, 16)):
        for h in range(4):
            ks = [k[table[s, j // 16], h // 2, j % 16].astype(float) for j in range(n)]
            vs = [v[table[s, j // 16], h // 2, j % 16].astype(float) for j in range(n)]
            e = np.array([math.exp(0.5 * sum(a * b for a, b in zip(q[r, h].astype(float), x))) for x in ks])
            assert np.isclose(lse[r, h], math.log(e.sum()))
            assert np.allclose(out[r, h], (e / e.sum()) @ np.array(vs))
    y = R.turned(np.array([[1.0, 2.0, 3.0, 4.0]], np.float16), None, 0.0, 100.0, 3)
    for i, a in enumerate((3.0, 0.3)):
        assert np.allclose([y[0, i], y[0, i + 2]], [(i + 1) * math.cos(a) - (i + 3) * math.sin(a),
                                                    (i + 3) * math.cos(a) + (i + 1) * math.sin(a)])
    # one drafted token of two, by hand: p = (1/4, 3/4) twice
    logits = np.log(np.array([[1.0, 3.0], [1.0, 3.0]])).astype(np.float16)
    q = np.array([[0.5, 0.5], [0, 0]], np.float32)
    for u, want, n in ((0.49, [0, 1], 1), (0.51, [1, -1], 0)):
        out, acc, _, _ = R.verify(logits, np.array([9, 0]), [0, 2], 1, 2, np.array([u, 0.5], np.float32), draft=q)
        assert out[0].tolist() == want and acc[0] == n


def test_mfma_sources_have_arrived(Q):
    from qwen3_iree_amd import build
    from test_mfma_wait_states import too_close

    lines = subprocess.run([str(build.ROCM / "llvm" / "bin" / "llvm-objdump"), "-d", str(build.PAGES_OBJECT)],
                           check=True, capture_output=True, text=True, timeout=120).stdout.splitlines()
    assert any("v_mfma" in line for line in lines)
    assert not any("v_pk_" in line and "_f32" in line for line in lines)
    assert not too_close(lines)
