"""Several sequences through the model at once, over one paged KV cache.

PagedSession keeps the k and v of up to max_seqs sequences in pages of a shared pool (f16,
or 8 bits with a scale for each token and head), runs new rows of any of them in one
step (qwen3_pages_step), takes tokens by drafts and random numbers (kv_verify), and hands
a sequence over to a DecodeSession's flat cache (kv_pages_read).  No counterpart in the
reference, whose loop runs one sequence (model/qwen3_full.mlir:1431-1526).
"""
from __future__ import annotations

import ctypes

import numpy as np

from . import decode as D
from . import drafts
from . import pages as P
from . import q8gemv as Q

MAX_ROWS = 128  # of a step


class PagedSession:
    """pages of page_size slots, shared by the sequences; bits 16 or 8.  A sequence has at
    most max_len slots.  The methods synchronize."""

    def __init__(self, model: D.DeviceWeights, pages: int, max_seqs: int, max_len: int,
                 page_size: int = 64, bits: int = 16, stream: Q.Stream | None = None):
        if not 1 <= max_seqs <= P.MAX_SEQS or bits not in (8, 16) or page_size % 16 or page_size < 16:
            raise ValueError(f"{max_seqs} sequences, {bits} bits, pages of {page_size}")
        if pages < 1 or max_len < 1:
            raise ValueError(f"{pages} pages, {max_len} slots of a sequence")
        self.model, self.stream = model, stream
        self.page_size, self.max_seqs, self.bits = int(page_size), int(max_seqs), int(bits)
        self.max_pages = (int(max_len) + self.page_size - 1) // self.page_size
        rows = D.LAYERS * int(pages) * D.KV_HEADS * self.page_size
        size = rows * D.HEAD_DIM * self.bits // 8
        self._pool = [Q.DeviceBuffer(size), Q.DeviceBuffer(size)]
        self._scales = [Q.DeviceBuffer(4 * rows), Q.DeviceBuffer(4 * rows)] if bits == 8 else [None, None]
        self.pages = P.Pages(*self._pool, pages, self.page_size, D.LAYERS, D.KV_HEADS, D.HEAD_DIM,
                             *self._scales)
        self._free = list(range(int(pages)))[::-1]
        self._held: dict[int, list[int]] = {}   # a sequence's pages
        self.length: dict[int, int] = {}        # and its slots in use
        # of a step: page table, lengths, first rows, tokens, next tokens
        words = (self.max_seqs * (self.max_pages + 2) + 1) + 2 * MAX_ROWS
        self._words = Q.DeviceBuffer(4 * words)
        self._ws = Q.DeviceBuffer(int(Q.load_library().qwen3_pages_workspace_bytes(MAX_ROWS, MAX_ROWS)))
        self._ws.fill(0)
        self._logits: Q.DeviceBuffer | None = None
        self._verify: tuple[Q.DeviceBuffer, ...] | None = None

    # sequences
    def add(self) -> int:
        """A new, empty sequence."""
        for s in range(self.max_seqs):
            if s not in self._held:
                self._held[s], self.length[s] = [], 0
                return s
        raise ValueError(f"all {self.max_seqs} sequences are in use")

    def remove(self, seq: int) -> None:
        """Ends a sequence; its pages serve others."""
        self._free += self._held.pop(seq)[::-1]
        del self.length[seq]

    def cut(self, seq: int, length: int) -> None:
        """Drops the slots from `length` on."""
        if not 0 <= length <= self.length[seq]:
            raise ValueError(f"{length} of {self.length[seq]} slots")
        self.length[seq] = int(length)
        self._trim(seq)

    def _trim(self, seq: int) -> None:
        keep = (self.length[seq] + self.page_size - 1) // self.page_size
        held = self._held[seq]
        self._free += held[keep:][::-1]
        del held[keep:]

    def _batch(self, seqs: list[int], counts: list[int], lengths: list[int]) -> P.Batch:
        """Uploads the page table, lengths and first rows of some sequences."""
        n = len(seqs)
        table = np.zeros((n, self.max_pages), np.int32)
        for i, s in enumerate(seqs):
            table[i, :len(self._held[s])] = self._held[s]
        start = np.concatenate([[0], np.cumsum(counts)])
        self._words.upload(np.concatenate([table.ravel(), lengths, start]).astype(np.int32))
        at = self._words.ptr
        return P.Batch(at, at + 4 * table.size, n, self.max_pages, int(start[-1]), max(counts),
                       start=at + 4 * (table.size + n))

    @property
    def _tokens(self) -> int:
        """Offset of the step's tokens (then the next tokens)."""
        return 4 * (self.max_seqs * (self.max_pages + 2) + 1)

    def _pages_for(self, seqs: list[int], counts: list[int]) -> dict[int, int]:
        """The pages each sequence needs for more rows; refused where there are none."""
        need = {}
        for s, m in zip(seqs, counts):
            if self.length[s] + m > self.max_pages * self.page_size:
                raise ValueError(f"sequence {s}: {self.length[s]} + {m} slots")
            need[s] = (self.length[s] + m + self.page_size - 1) // self.page_size - len(self._held[s])
        if sum(need.values()) > len(self._free):
            raise ValueError(f"{sum(need.values())} pages needed, {len(self._free)} free")
        return need

    def step(self, rows: dict[int, object], logits: bool = False) -> dict[int, np.ndarray]:
        """Runs each sequence's new tokens (behind the slots in use; at most 128 in all) and
        keeps their k and v; the model's next token after each.  logits: also leave
        them on the device, f16 [rows, vocab] in the order of `rows`."""
        seqs = list(rows)
        new = [np.ascontiguousarray(rows[s], np.int32).reshape(-1) for s in seqs]
        counts = [int(t.size) for t in new]
        if not seqs or not 0 < sum(counts) <= MAX_ROWS or min(counts) < 1:
            raise ValueError(f"{counts} rows: each sequence at least one, {MAX_ROWS} at most in all")
        need = self._pages_for(seqs, counts)
        if logits and self._logits is None:
            self._logits = Q.DeviceBuffer(MAX_ROWS * D.VOCAB * 2)
        for s in seqs:
            self._held[s] += [self._free.pop() for _ in range(need[s])]
        total = sum(counts)
        try:
            batch = self._batch(seqs, counts, [self.length[s] + m for s, m in zip(seqs, counts)])
            self._words.upload(np.concatenate(new), self._tokens)
            at = self._words.ptr + self._tokens
            Q._call("qwen3_pages_step", self.model.ref(), ctypes.byref(self.pages),
                    ctypes.byref(batch), at, at + 4 * MAX_ROWS,
                    self._logits.ptr if logits else None, self._ws.ptr, self._ws.nbytes,
                    Q._stream(self.stream))
            self.synchronize()
        except Exception:
            for s in seqs:
                self._trim(s)
            raise
        for s, m in zip(seqs, counts):
            self.length[s] += m
        out = self._words.download(np.int32, total, self._tokens + 4 * MAX_ROWS)
        return dict(zip(seqs, np.split(out, np.cumsum(counts)[:-1])))

    def prompt(self, seq: int, tokens) -> int:
        """Reads tokens behind what a sequence holds; the model's next token."""
        tokens = np.ascontiguousarray(tokens, np.int32).reshape(-1)
        if tokens.size == 0:
            raise ValueError("empty prompt")
        self._pages_for([seq], [int(tokens.size)])
        for i in range(0, tokens.size, MAX_ROWS):
            following = self.step({seq: tokens[i:i + MAX_ROWS]})[seq]
        return int(following[-1])

    def sample(self, rows: dict[int, object], uniform, temperature=None, draft=None):
        """step(rows) of each sequence's last token and the drafted ones behind it, then what
        stands of them: {sequence: tokens} (the accepted drafts and one more) and their log
        probabilities; the slots of refused drafts are dropped.  uniform: a number in
        [0, 1) for every row; temperature: one for each sequence (None: 1, 0: the
        likeliest); draft f32 [rows, vocab]: the probabilities each drafted token was
        taken with, in the row before it (None: drafts are taken as they are)."""
        seqs = list(rows)
        new = [np.ascontiguousarray(rows[s], np.int32).reshape(-1) for s in seqs]
        counts = [int(t.size) for t in new]
        total, n = sum(counts), len(seqs)
        uniform = np.ascontiguousarray(uniform, np.float32).reshape(-1)
        if uniform.size != total:
            raise ValueError(f"{uniform.size} random numbers for {total} rows")
        if temperature is not None:
            temperature = np.ascontiguousarray(temperature, np.float32).reshape(-1)
            if temperature.size != n:
                raise ValueError(f"{temperature.size} temperatures of {n} sequences")
        if draft is not None:
            draft = np.ascontiguousarray(draft, np.float32)
            if draft.shape != (total, D.VOCAB):
                raise ValueError(f"draft {draft.shape} is not {(total, D.VOCAB)}")
        before = {s: self.length[s] for s in seqs}
        self.step(rows, logits=True)
        try:
            if self._verify is None:
                # random numbers, temperatures, accepted, first rows; tokens, log
                # probabilities; workspace
                ws = Q.DeviceBuffer(P.verify_workspace_bytes(MAX_ROWS, self.max_seqs, D.VOCAB))
                ws.fill(0)
                self._verify = (Q.DeviceBuffer(4 * (MAX_ROWS + 3 * self.max_seqs + 1)),
                                Q.DeviceBuffer(8 * MAX_ROWS * self.max_seqs), ws)
            small, out, ws = self._verify
            most = max(counts)
            start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
            small.upload(np.concatenate([uniform.view(np.int32), start]))
            heat = small.ptr + 4 * (total + n + 1)
            if temperature is not None:
                small.upload(temperature, heat - small.ptr)
            accepted = heat + 4 * n
            draft_dev = None if draft is None else Q.DeviceBuffer.from_array(draft)
            try:
                P.verify(self._logits, D.VOCAB, D.VOCAB, total, self._words.ptr + self._tokens, n,
                         most, small, out, most, accepted, start=small.ptr + 4 * total,
                         temperature=None if temperature is None else heat, draft=draft_dev,
                         draft_stride=D.VOCAB, logprob=out.ptr + 4 * n * most, workspace=ws,
                         workspace_bytes=ws.nbytes, stream=self.stream)
                self.synchronize()
            finally:
                if draft_dev is not None:
                    draft_dev.free()
            kept = small.download(np.int32, n, accepted - small.ptr)
            tokens = out.download(np.int32, n * most).reshape(n, most)
            logprob = out.download(np.float32, n * most, 4 * n * most).reshape(n, most)
        except Exception:
            for s in seqs:
                self.cut(s, before[s])
            raise
        result = {}
        for i, s in enumerate(seqs):
            self.cut(s, before[s] + 1 + int(kept[i]))
            result[s] = (tokens[i, :kept[i] + 1].copy(), logprob[i, :kept[i] + 1].copy())
        return result

    def to_session(self, seq: int, session: D.DecodeSession) -> None:
        """Reads a sequence's slots into a DecodeSession's cache and puts its position behind
        them (its token word stays).  A session of drafted trees, which counts its own slots, is
        refused."""
        if isinstance(session, drafts.DraftSession):
            raise TypeError("a session of drafted trees takes no sequence over")
        n = self.length[seq]
        if not 1 <= n < session.max_seq:
            raise ValueError(f"{n} slots into a cache of {session.max_seq}")
        self.synchronize()
        batch = self._batch([seq], [n], [n])
        P.read(self.pages, 0, D.LAYERS, batch, session.k_cache, session.v_cache, D.KV_DIM,
               session.max_seq * D.KV_DIM, session.stream)
        session.synchronize()
        session.set_state(session.get_state()[0], n)

    def read_logits(self, rows: int) -> np.ndarray:
        """The logits f16 [rows, vocab] the last step left."""
        if self._logits is None:
            raise ValueError("no step has left logits")
        self.synchronize()
        return self._logits.download(np.float16, rows * D.VOCAB).reshape(rows, D.VOCAB)

    def synchronize(self) -> None:
        if self.stream is not None:
            self.stream.synchronize()
        else:
            Q.synchronize()

    def free(self) -> None:
        for b in (*self._pool, *self._scales, self._words, self._ws, self._logits,
                  *(self._verify or ())):
            if b is not None:
                b.free()
