"""Serving several sequences from one paged KV cache (include/kv_pages.h): rows
appended with their heads' norm and rotation, attention over the pages, pages read
back, and drafted tokens verified against the model's probabilities.

The calls take device addresses (DeviceBuffer objects or integers) and only
enqueue; a refused argument raises Q8GemvError.  No counterpart in the reference,
which runs one sequence over a flat cache (model/qwen3_full.mlir:1431-1526).
"""
from __future__ import annotations

import ctypes
import struct

from . import q8gemv as Q

F16, Q8 = 0, 1
MAX_SEQS = 1024
MAX_ROWS = 256  # of a sequence, in attn and verify

_P, _I32, _I64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64


class Pages(ctypes.Structure):
    """struct kv_pages: k, v [layers, pages, kv_heads, page_size, head_dim], f16 or
    (with scales f32 [layers, pages, kv_heads, page_size]) int8 codes."""
    _fields_ = [("k", _P), ("v", _P), ("k_scale", _P), ("v_scale", _P), ("pages", _I64),
                ("layers", _I32), ("page_size", _I32), ("kv_heads", _I32), ("head_dim", _I32),
                ("type", _I32)]

    def __init__(self, k, v, pages: int, page_size: int, layers: int, kv_heads: int,
                 head_dim: int, k_scale=None, v_scale=None):
        super().__init__(Q._ptr(k), Q._ptr(v), Q._ptr(k_scale), Q._ptr(v_scale), int(pages),
                         int(layers), int(page_size), int(kv_heads), int(head_dim),
                         F16 if k_scale is None and v_scale is None else Q8)


class Batch(ctypes.Structure):
    """struct kv_batch: the page table int32 [seqs, max_pages], the lengths int32 [seqs]
    (new rows among them) and the first rows int32 [seqs + 1] (None: one row each) of
    the sequences of a call."""
    _fields_ = [("table", _P), ("length", _P), ("start", _P), ("table_stride", _I64),
                ("seqs", _I32), ("max_pages", _I32), ("rows", _I32), ("max_rows", _I32)]

    def __init__(self, table, length, seqs: int, max_pages: int, rows: int, max_rows: int = 1,
                 start=None, table_stride: int | None = None):
        super().__init__(Q._ptr(table), Q._ptr(length), Q._ptr(start),
                         int(max_pages if table_stride is None else table_stride), int(seqs),
                         int(max_pages), int(rows), int(max_rows))


class Rows(ctypes.Structure):
    """struct kv_rows"""
    _fields_ = [("q", _P), ("k", _P), ("v", _P), ("q_out", _P), ("q_norm", _P), ("k_norm", _P),
                ("positions", _P), ("q_stride", _I64), ("k_stride", _I64), ("v_stride", _I64),
                ("q_out_stride", _I64), ("eps", ctypes.c_double), ("theta", ctypes.c_double),
                ("q_heads", _I32)]


_ROWS = struct.Struct("=7Q4q2di4x")


class Drafts(ctypes.Structure):
    """struct kv_drafts"""
    _fields_ = [("logits", _P), ("tokens", _P), ("start", _P), ("temperature", _P), ("draft", _P),
                ("uniform", _P), ("out", _P), ("accepted", _P), ("logprob", _P),
                ("logits_stride", _I64), ("draft_stride", _I64), ("out_stride", _I64),
                ("vocab", _I32), ("rows", _I32), ("seqs", _I32), ("max_rows", _I32)]


_DRAFTS = struct.Struct("=9Q3q4i")


def append(pages: Pages, layer: int, batch: Batch, k, k_stride: int, v, v_stride: int,
           k_norm=None, q=None, q_stride: int = 0, q_heads: int = 0, q_norm=None, q_out=None,
           q_out_stride: int = 0, eps: float = 1e-6, theta: float = 0.0, positions=None,
           stream=None) -> None:
    """Writes new rows of a layer into the pages, k after its heads' norm (k_norm f16
    [head_dim], None: none) and rotation (theta, 0: none) by its position (None: its
    slot); the queries, treated alike, go to q_out."""
    p = Q._ptr
    # (struct kv_rows; filling a ctypes structure takes twice as long)
    rows = _ROWS.pack(p(q) or 0, p(k) or 0, p(v) or 0, p(q_out) or 0, p(q_norm) or 0,
                      p(k_norm) or 0, p(positions) or 0, q_stride, k_stride, v_stride,
                      q_out_stride, eps, theta, q_heads)
    Q._call("kv_pages_append", ctypes.byref(pages), int(layer), ctypes.byref(batch), rows,
            Q._stream(stream))


def attn_workspace_bytes(pages: Pages, batch: Batch, q_heads: int) -> int:
    return int(Q.load_library().kv_pages_attn_workspace_bytes(
        ctypes.byref(pages), ctypes.byref(batch), int(q_heads)))


def attn(pages: Pages, layer: int, batch: Batch, q, q_stride: int, q_heads: int, scale: float,
         out, out_stride: int, lse=None, workspace=None, workspace_bytes: int = 0,
         stream=None) -> None:
    """Attention of the batch's rows, each over its sequence's slots up to its own; out
    f16 [rows, q_heads x head_dim], lse f32 [rows, q_heads]."""
    Q._call("kv_pages_attn", ctypes.byref(pages), int(layer), ctypes.byref(batch), Q._ptr(q),
            int(q_stride), int(q_heads), float(scale), Q._ptr(out), int(out_stride), Q._ptr(lse),
            Q._ptr(workspace), int(workspace_bytes), Q._stream(stream))


def read(pages: Pages, layer: int, layers: int, batch: Batch, k_out, v_out, row_stride: int,
         layer_stride: int = 0, stream=None) -> None:
    """The batch's rows of some layers read back as f16 [rows, kv_heads, head_dim] with
    the given strides."""
    Q._call("kv_pages_read", ctypes.byref(pages), int(layer), int(layers), ctypes.byref(batch),
            Q._ptr(k_out), Q._ptr(v_out), int(row_stride), int(layer_stride), Q._stream(stream))


def verify_workspace_bytes(rows: int, seqs: int, vocab: int) -> int:
    return int(Q.load_library().kv_verify_workspace_bytes(int(rows), int(seqs), int(vocab)))


def verify(logits, logits_stride: int, vocab: int, rows: int, tokens, seqs: int, max_rows: int,
           uniform, out, out_stride: int, accepted, start=None, temperature=None, draft=None,
           draft_stride: int = 0, logprob=None, workspace=None, workspace_bytes: int = 0,
           stream=None) -> None:
    """How many drafted tokens of each sequence stand (accepted int32 [seqs]), those and
    one more sampled token (out int32 [seqs, out_stride], -1 behind), and their log
    probabilities."""
    p = Q._ptr
    drafts = _DRAFTS.pack(p(logits) or 0, p(tokens) or 0, p(start) or 0, p(temperature) or 0,
                          p(draft) or 0, p(uniform) or 0, p(out) or 0, p(accepted) or 0,
                          p(logprob) or 0, logits_stride, draft_stride, out_stride, vocab, rows,
                          seqs, max_rows)
    Q._call("kv_verify", drafts, Q._ptr(workspace), int(workspace_bytes), Q._stream(stream))
