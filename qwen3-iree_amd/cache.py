"""Operators over an f16 KV cache (include/f16_cache.h): attention of a tree of
drafted tokens, the attention weights cached positions got, and eviction by them.

The calls take device addresses (DeviceBuffer objects or integers) and only
enqueue; a refused argument raises Q8GemvError.  No counterpart in the reference,
whose cache holds one growing sequence (model/qwen3_full.mlir:1431-1526).
"""
from __future__ import annotations

import ctypes

from . import q8gemv as Q

TREE_MAX_NODES = 256


class Cache(ctypes.Structure):
    """struct f16_cache: k, v f16 [layers * max_seq, kv_heads, head_dim] and
    (optional) weights f32 [layers, kv_heads, max_seq]."""
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("weights", ctypes.c_void_p),
                ("max_seq", ctypes.c_int64), ("layers", ctypes.c_int32),
                ("kv_heads", ctypes.c_int32), ("head_dim", ctypes.c_int32)]

    def __init__(self, k, v, max_seq: int, layers: int, kv_heads: int, head_dim: int,
                 weights=None):
        super().__init__(Q._ptr(k), Q._ptr(v), Q._ptr(weights), int(max_seq), int(layers),
                         int(kv_heads), int(head_dim))


def tree_mask(parents, n: int, mask, depth=None, stream=None) -> None:
    """The ancestor masks u32 [n, ceil(n / 32)] and depths int32 [n] of a tree
    given by its parents int32 [n] (-1: right behind the cache)."""
    Q._call("f16_tree_mask", Q._ptr(parents), int(n), Q._ptr(mask), Q._ptr(depth),
            Q._stream(stream))


def attn_tree_workspace_bytes(cache: Cache, length: int, n: int, q_heads: int) -> int:
    return int(Q.load_library().f16_attn_tree_workspace_bytes(
        ctypes.byref(cache), int(length), int(n), int(q_heads)))


def attn_tree(cache: Cache, layer: int, length: int, q, q_stride: int, q_heads: int, mask, n: int,
              scale: float, out, out_stride: int, lse=None, workspace=None,
              workspace_bytes: int = 0, stream=None) -> None:
    """Attention of n rows (their k and v in slots length .. length + n - 1)
    over the cached positions and the rows their mask names (None: the rows
    before them); out f16 [n, q_heads x head_dim], lse f32 [n, q_heads]."""
    Q._call("f16_attn_tree", ctypes.byref(cache), int(layer), int(length), Q._ptr(q),
            int(q_stride), int(q_heads), Q._ptr(mask), int(n), float(scale), Q._ptr(out),
            int(out_stride), Q._ptr(lse), Q._ptr(workspace), int(workspace_bytes),
            Q._stream(stream))


def attn_weights_add(cache: Cache, length: int, q, q_layer_stride: int, q_stride: int,
                     q_heads: int, lse, lse_layer_stride: int, rows: int, path, n: int,
                     scale: float, stream=None) -> None:
    """Adds the attention of n tokens at slots length .. length + n - 1 (rows
    path[i] of q and lse, None: row i) to cache.weights, in every layer."""
    Q._call("f16_attn_weights_add", ctypes.byref(cache), int(length), Q._ptr(q),
            int(q_layer_stride), int(q_stride), int(q_heads), Q._ptr(lse), int(lse_layer_stride),
            int(rows), Q._ptr(path), int(n), float(scale), Q._stream(stream))


def cache_select(cache: Cache, length: int, budget: int, sinks: int, recent: int, keep,
                 stream=None) -> None:
    """keep int32 [layers, kv_heads, budget]: the first `sinks`, the last
    `recent` and the most attended of the slots between, ascending."""
    Q._call("f16_cache_select", ctypes.byref(cache), int(length), int(budget), int(sinks),
            int(recent), Q._ptr(keep), Q._stream(stream))


def cache_compact(src: Cache, dst: Cache, keep, per_head: bool, base: int, count: int,
                  stream=None) -> None:
    """Slot base + j of dst becomes slot base + keep[j] of src (dst may be src
    where keep ascends); keep [layers, kv_heads, count] or one [count] for all."""
    Q._call("f16_cache_compact", ctypes.byref(src), ctypes.byref(dst), Q._ptr(keep),
            int(bool(per_head)), int(base), int(count), Q._stream(stream))
