"""Drafted trees and eviction over a session's KV cache.

DraftSession runs trees of drafted tokens through the model at once
(qwen3_tree_step), keeps the path the model agrees with, adds up the attention
every cached slot gets, and evicts the least attended slots when the cache is
full.  After an eviction the cache holds fewer slots than the sequence has
positions, so the session keeps the two apart: `length` slots, next RoPE position
`position`.  No counterpart in the reference, whose loop takes one token a step
over a cache that only grows (model/qwen3_full.mlir:1431-1526).
"""
from __future__ import annotations

import numpy as np

from . import cache as C
from . import decode as D
from . import q8gemv as Q

SCALE = 128 ** -0.5


def greedy_path(tokens, parents, following) -> list[int]:
    """The nodes from node 0 down whose tokens the model itself would have chosen:
    following[i] is the model's token after node i."""
    path = [0]
    while True:
        nxt = [i for i in range(path[-1] + 1, len(tokens))
               if parents[i] == path[-1] and tokens[i] == following[path[-1]]]
        if not nxt:
            return path
        path.append(nxt[0])


class DraftSession(D.DecodeSession):
    """A session whose tokens come in trees of up to max_nodes nodes.

    weights: keep the attention weights eviction goes by; then a prompt is read in
    trees too (chunks of max_nodes tokens), else in one piece.  The calls of a
    DecodeSession that go by the token or position on the device, whole steps and
    their parts, are refused: they know nothing of `length`."""

    def __init__(self, model: D.DeviceWeights, max_seq: int, max_nodes: int = 64,
                 weights: bool = True, stream: Q.Stream | None = None):
        if not 1 <= max_nodes <= C.TREE_MAX_NODES or max_nodes > max_seq:
            raise ValueError(f"max_nodes {max_nodes} outside [1, {C.TREE_MAX_NODES}] or the cache")
        super().__init__(model, max_seq, stream)
        self.max_nodes = int(max_nodes)
        self.length = self.position = 0
        n = self.max_nodes
        lib = Q.load_library()
        self._ws = Q.DeviceBuffer(int(lib.qwen3_tree_workspace_bytes(n, self.max_seq)))
        self._nodes = Q.DeviceBuffer(4 * 4 * n)  # tokens, parents, next tokens, path
        self.tree_logits: Q.DeviceBuffer | None = None
        self._q = self._lse = self._weights = None
        if weights:
            self._q = Q.DeviceBuffer(D.LAYERS * n * D.Q_DIM * 2)
            self._lse = Q.DeviceBuffer(D.LAYERS * n * D.Q_HEADS * 4)
            self._weights = Q.DeviceBuffer(D.LAYERS * D.KV_HEADS * self.max_seq * 4)
            self._weights.fill(0)
        self.cache = C.Cache(self.k_cache, self.v_cache, self.max_seq, D.LAYERS, D.KV_HEADS,
                             D.HEAD_DIM, self._weights)
        self._tree: tuple[np.ndarray, np.ndarray] | None = None  # of the last verify

    def _refused(self, *args, **kwargs):
        raise TypeError("a session of drafted trees moves by prompt, verify and accept")

    step = step_checked = capture = replay = prefill = prefill_batched = generate = _refused
    embed = layer = head = _refused

    def _slot(self, i: int) -> int:
        return self._nodes.ptr + 4 * self.max_nodes * i

    def verify(self, tokens, parents, logits: bool = False) -> np.ndarray:
        """Runs a tree (parents[i] < i, -1: right behind the cache) and returns the
        model's next token after every node.  logits: also leave them in
        tree_logits (f16 [n, vocab])."""
        tokens = np.ascontiguousarray(tokens, np.int32).reshape(-1)
        parents = np.ascontiguousarray(parents, np.int32).reshape(-1)
        n = tokens.size
        if not 1 <= n <= self.max_nodes or parents.size != n:
            raise ValueError(f"a tree of 1 to {self.max_nodes} nodes and as many parents")
        if (parents < -1).any() or (parents >= np.arange(n)).any():
            raise ValueError("a node's parent comes before it")
        if logits and self.tree_logits is None:
            self.tree_logits = Q.DeviceBuffer(self.max_nodes * D.VOCAB * 2)
        self._nodes.upload(tokens, 0)
        self._nodes.upload(parents, 4 * self.max_nodes)
        self._tree = None
        Q._call("qwen3_tree_step", self.model.ref(), self.k_cache.ptr, self.v_cache.ptr,
                self.max_seq, self._slot(0), self._slot(1), n, self.length, self.position,
                self._slot(2), self.tree_logits.ptr if logits else None, Q._ptr(self._q),
                Q._ptr(self._lse), self._ws.ptr, self._ws.nbytes, Q._stream(self.stream))
        self.synchronize()
        self._tree = (tokens, parents)
        return self._nodes.download(np.int32, n, 8 * self.max_nodes)

    def accept(self, path) -> None:
        """Keeps the nodes `path` (a chain from a node behind the cache down) of the
        tree last verified; the others are dropped.  Synchronizes."""
        if self._tree is None:
            raise ValueError("no tree has been verified")
        tokens, parents = self._tree
        path = np.ascontiguousarray(path, np.int32).reshape(-1)
        chain = [-1, *path.tolist()]
        if path.size == 0 or (path < 0).any() or (path >= tokens.size).any() or any(
                parents[b] != a for a, b in zip(chain, chain[1:])):
            raise ValueError("not a chain of the verified tree")
        m, n = int(path.size), int(tokens.size)
        self._nodes.upload(path, 12 * self.max_nodes)
        C.cache_compact(self._kv(), self._kv(), self._slot(3), False, self.length, m, self.stream)
        if self._weights is not None:
            C.attn_weights_add(self.cache, self.length, self._q, n * D.Q_DIM, D.Q_DIM, D.Q_HEADS,
                               self._lse, n * D.Q_HEADS, n, self._slot(3), m, SCALE, self.stream)
        self.synchronize()
        self._tree = None
        self.length += m
        self.position += m

    def _kv(self) -> C.Cache:
        """The cache without its weights."""
        return C.Cache(self.k_cache, self.v_cache, self.max_seq, D.LAYERS, D.KV_HEADS, D.HEAD_DIM)

    def prompt(self, tokens) -> int:
        """Reads tokens behind what the session holds; the model's next token."""
        tokens = np.ascontiguousarray(tokens, np.int32).reshape(-1)
        if tokens.size == 0 or self.length + tokens.size > self.max_seq:
            raise ValueError(f"{tokens.size} tokens behind {self.length} of {self.max_seq} slots")
        self._tree = None  # the tokens go where its nodes are
        if self._weights is None and self.length == self.position:
            self.set_state(0, self.length)
            super().prefill_batched(tokens)
            self.length += int(tokens.size)
            self.position = self.length
            return self.get_state()[0]
        for i in range(0, tokens.size, self.max_nodes):
            part = tokens[i:i + self.max_nodes]
            following = self.verify(part, np.arange(-1, part.size - 1))
            self.accept(np.arange(part.size))
        return int(following[-1])

    def generate_drafted(self, token: int, max_new: int, eos_id: int, draft) -> np.ndarray:
        """Greedy tokens behind `token` (not yet in the cache).  draft(context) is
        called with the tokens so far (`token` first) and returns (tokens,
        parents) of a tree that continues them (parents -1: behind the last one;
        may be empty).  Stops behind eos_id, at max_new tokens or a full cache."""
        out = [int(token)]
        while len(out) - 1 < max_new and self.length < self.max_seq:
            room = min(self.max_nodes, self.max_seq - self.length) - 1
            d_tokens, d_parents = draft(list(out))
            d_tokens, d_parents = list(d_tokens)[:room], list(d_parents)[:room]
            tokens = [out[-1], *d_tokens]
            parents = [-1, *(p + 1 for p in d_parents)]
            following = self.verify(tokens, parents)
            path = greedy_path(tokens, parents, following)[:max_new - (len(out) - 1)]
            new = [int(following[i]) for i in path]
            if eos_id in new:
                path = path[:new.index(eos_id) + 1]
                new = new[:len(path)]
            self.accept(path)
            out += new
            if new[-1] == eos_id:
                break
        return np.array(out[1:], np.int32)

    def evict(self, budget: int, sinks: int = 4, recent: int = 64) -> np.ndarray:
        """Keeps `budget` of the slots in every layer and kv head: the first
        `sinks`, the last `recent` and the most attended between, moved to the
        front in order.  Returns the kept slots int32 [28, 8, budget]."""
        if self._weights is None:
            raise ValueError("the session keeps no attention weights")
        with Q.DeviceBuffer(4 * D.LAYERS * D.KV_HEADS * max(int(budget), 1)) as keep:
            C.cache_select(self.cache, self.length, budget, sinks, recent, keep, self.stream)
            self._tree = None  # the slots move under it
            C.cache_compact(self.cache, self.cache, keep, True, 0, budget, self.stream)
            self.synchronize()
            self.length = int(budget)
            return keep.download(np.int32).reshape(D.LAYERS, D.KV_HEADS, -1)

    def slot_weights(self) -> np.ndarray:
        """The attention every slot got, f32 [28, 8, length]."""
        if self._weights is None:
            raise ValueError("the session keeps no attention weights")
        self.synchronize()
        w = self._weights.download(np.float32).reshape(D.LAYERS, D.KV_HEADS, self.max_seq)
        return w[:, :, :self.length]

    def free(self) -> None:
        super().free()
        for b in (self._ws, self._nodes, self.tree_logits, self._q, self._lse, self._weights):
            if b is not None:
                b.free()
