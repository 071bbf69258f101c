"""Decoding with a cache that stays small, over a batch engine's rows.

:class:`BoundedDecoder` takes over the rows of a prefilled
:class:`~pagelora_b200.batch_engine.BatchDecodeEngine` like
:class:`~pagelora_b200.tree_decode.TreeDecoder` (page bookkeeping on the device,
rows fork and end) and decodes one token per row and step with one of

* a sliding window with sinks (``window``): every layer's attention is
  paged_window_decode, and :meth:`BoundedDecoder.trim` gives back what no later
  token sees;
* eviction by accumulated attention weight (``evict``): the steps'
  paged_decode_weights note what every cached token receives, over heads and
  layers, and :meth:`BoundedDecoder.evict` cuts the rows that outgrew their
  budget (evict_select, then cache_compact in every layer);
* a cache in 4 bits (``kv4``, with or without a window): the engine's pages are
  quantised once, new tokens as they come (kv4_append), and the attention runs
  over the records (paged_kv4_decode).

The prompt is the engine's, with full attention over bf16, and notes no weights:
:attr:`BoundedDecoder.weight` [rows, positions] starts at 0, so an eviction goes
by the steps so far and, among positions without weight, keeps the lower ones.  A
caller with the prompt's queries and log sums adds its weights there
(paged_prefill_weights, layer by layer).  A step that notes weights takes a
workspace by the rows' capacity, not their length: 4 bytes a position and query
head of every row.

Keys keep the rotation of the position where they were computed, so a new
token's position counts all tokens that the row has had, evicted ones too.  No
step waits for the device, except the first after rows ended or began.  No
reference counterpart: the reference decodes over the whole bf16 context
(model/flashinfer/generation.py:188-247).
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from pagelora_b200 import kernels as K
from pagelora_b200.batch_engine import BatchDecodeEngine
from pagelora_b200.tree_decode import TreeDecoder, TreeStep


@dataclass(frozen=True)
class Window:
    """A token sees the last ``size`` positions and the first ``sinks``."""

    size: int
    sinks: int = 4


@dataclass(frozen=True)
class EvictBudget:
    """Tokens that a row keeps: its first ``sinks``, its last ``recent`` and
    those of the highest accumulated weight, ``tokens`` in all."""

    tokens: int
    sinks: int = 4
    recent: int = 64


class BoundedDecoder(TreeDecoder):
    """``engine.step_*`` must not be used any more; with ``kv4`` neither its bf16
    pages, which stay as they were, beside the records.  The decoder does not
    read them again: ``engine.kv = None`` gives their memory back."""

    def __init__(self, engine: BatchDecodeEngine, *, window: Window | None = None, evict: EvictBudget | None = None,
                 kv4: bool = False) -> None:
        if evict is not None and (window is not None or kv4):
            raise ValueError("eviction by weight needs the whole bf16 context: no window, no 4-bit cache")
        if window is None and evict is None and not kv4:
            raise ValueError("a bounded decoder needs a window, an eviction budget or a 4-bit cache")
        if window is not None:
            K._need_window(window.size, window.sinks)
        if evict is not None and (evict.tokens < 1 or evict.sinks < 0 or evict.recent < 0 or
                                  evict.sinks + evict.recent > evict.tokens):
            raise ValueError("a budget needs tokens >= 1, sinks >= 0, recent >= 0 and sinks + recent <= tokens")
        if engine.spec.num_qo_heads > 16 * engine.spec.num_kv_heads:
            raise ValueError("at most 16 query heads per kv head")
        super().__init__(engine)
        self.window, self.budget = window, evict
        self.pos = self.lens.clone()  # tokens that every row has had
        spec, dev = engine.spec, engine.device
        if evict is not None:
            width = self.cap * engine.page_size
            self.weight = torch.zeros(self.rows, width, device=dev)
            self._weight_next = torch.zeros_like(self.weight)
            self._keep = torch.empty(self.rows, max(1, evict.tokens - evict.sinks), dtype=torch.int32, device=dev)
            self._keep_from, self._keep_count = torch.empty_like(self.lens), torch.empty_like(self.lens)
        self.kv4 = None
        if kv4:
            layers, pages, _, ps, hkv, d = engine.kv.shape
            self.kv4 = torch.zeros(layers, pages, 2, ps, hkv, K.kv4_record_bytes(d), dtype=torch.uint8, device=dev)
            some = max(1, (1 << 24) // (ps * hkv * d))  # pages a call: its K and V are copied, 32 MB each
            slot = torch.arange(min(some, pages) * ps, dtype=torch.int32, device=dev)
            for li in range(layers):
                for p0 in range(0, pages, some):
                    x = engine.kv[li, p0:p0 + some]
                    n = x.shape[0] * ps
                    k, v = (x[:, i].reshape(n, hkv, d) for i in (0, 1))
                    K.kv4_append(k, v, self.kv4[li], slot[:n] // ps + p0, slot[:n] % ps, self.status)
            # the step's new K/V, one page a row, on their way into the records
            self._staged = torch.zeros(self.rows, 2, 1, hkv, d, dtype=torch.bfloat16, device=dev)
            self._staged_page = torch.arange(self.rows, dtype=torch.int32, device=dev)
            self._staged_off = torch.zeros_like(self._staged_page)

    def verify(self, *args, **kwargs) -> TreeStep:
        raise ValueError("a bounded decoder decodes one token per row; TreeDecoder verifies drafted trees")

    @torch.no_grad()
    def step(self, tokens: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """One token per row (int64 [rows]); returns (next tokens [rows], logits
        [rows, vocab]).  Rows without a context take no part: their next token
        is -1 and their logits are 0.  A step that was refused (a row or the
        pool without room) returns -1 for every row and changes none."""

        self._need_tokens(tokens, self.rows)
        rows, tok_indptr = self._live_rows()
        n, some = rows.numel(), rows.numel() < self.rows
        if n == 0:
            logits = torch.zeros(self.rows, self.e.lm_head.shape[0], dtype=torch.bfloat16, device=rows.device)
            return torch.full_like(tokens, -1), logits
        before = self.weight.clone() if self.budget is not None else None
        slot_page, slot_off, _ = self._reserve(tok_indptr, n)
        indptr, last, positions, weight = self.indptr, self.last, self.pos, None
        if self.budget is not None:
            weight = self.weight
        if some:  # (rows without a context have no pages between those of the others)
            tokens, last, positions = tokens[rows], last[rows], positions[rows]
            indptr = torch.cat([indptr[rows], indptr[-1:]])
            weight = None if weight is None else weight[rows]
        table = (indptr, self.indices, last)
        win = self.window

        def attend(li, q):
            if self.kv4 is not None:
                k, v = self._staged[:n, 0, 0], self._staged[:n, 1, 0]
                K.kv4_append(k, v, self.kv4[li], slot_page, slot_off, self.status)
                return K.paged_kv4_decode(q, self.kv4[li], *table, window=None if win is None else win.size,
                                          sinks=0 if win is None else win.sinks, status=self.status)
            if win is not None:
                return K.paged_window_decode(q, self.e.kv[li], *table, window=win.size, sinks=win.sinks,
                                             status=self.status)
            return K.paged_decode_weights(q, self.e.kv[li], *table, weight, status=self.status)

        logits = self._forward(tokens, positions, rows, slot_page, slot_off, attend)
        nxt = K.argmax(logits, torch.empty_like(tokens))
        lens = self._row_lens()
        refused = (lens == self.lens).all()  # the reservation is for all rows or for none
        nxt.masked_fill_(refused, -1)
        if weight is not None:
            if some:
                self.weight.index_copy_(0, rows, weight)
            self.weight = torch.where(refused, before, self.weight)
        self.pos.add_(lens - self.lens)
        self.lens.copy_(lens)
        if some:
            nxt = nxt.new_full((self.rows,), -1).index_copy_(0, rows, nxt)
            logits = logits.new_zeros(self.rows, logits.shape[1]).index_copy_(0, rows, logits)
        return nxt, logits

    def _kv_target(self, li, slot_page, slot_off):
        if self.kv4 is None:
            return super()._kv_target(li, slot_page, slot_off)
        n = slot_page.numel()
        return self._staged, self._staged_page[:n], self._staged_off[:n]

    @torch.no_grad()
    def evict(self) -> None:
        """Rows longer than the budget keep the budget's tokens.  A call that is
        refused (no free pages to move what stays) changes no row."""

        if self.budget is None:
            raise ValueError("the decoder was built without an eviction budget (evict)")
        b = self.budget
        K.evict_select(self.weight, self.lens, b.tokens, sinks=b.sinks, recent=b.recent, keep_from=self._keep_from,
                       keep=self._keep, keep_count=self._keep_count, out_weight=self._weight_next, status=self.status)
        K.cache_compact(self.e.kv, self.refcount, self.table, self.num, self.last, self._keep_from, self._keep,
                        self._keep_count, status=self.status)
        lens = self._row_lens()
        done = (lens == self._keep_from + self._keep_count).all()
        self.weight, self._weight_next = torch.where(done, self._weight_next, self.weight), self.weight
        self.lens.copy_(lens)

    @torch.no_grad()
    def trim(self) -> None:
        """Rows give back what no later token sees: a row longer than ``sinks`` +
        ``size`` of the window keeps its first ``sinks`` and last ``size`` tokens.
        What stays moves to new pages in every layer, so a call is for when rows
        have grown by many tokens, not for every step.  One that is refused (no
        free pages to move what stays) changes no row."""

        if self.window is None:
            raise ValueError("the decoder was built without a window (window)")
        size, sinks = self.window.size, self.window.sinks
        if sinks + size >= self.cap * self.e.page_size:
            return  # no row is longer
        cut = self.lens > sinks + size
        keep_from, count = torch.where(cut, sinks, self.lens), cut.to(torch.int32) * size
        keep = (self.lens - size)[:, None] + torch.arange(size, dtype=torch.int32, device=self.lens.device)
        K.cache_compact(self.e.kv if self.kv4 is None else self.kv4, self.refcount, self.table, self.num, self.last,
                        keep_from, keep, count, status=self.status)
        self.lens.copy_(self._row_lens())

    def fork(self, src: list[int], dst: list[int]) -> None:
        """As TreeDecoder's; positions, weights and records go with the row."""

        empty = self.num == 0
        if self.kv4 is not None:
            s, d = self._row_ids(src), self._row_ids(dst)
            if len(src) != len(dst):
                raise ValueError("src and dst differ in length")
            if any(self.e.row_adapter[a] != self.e.row_adapter[b] for a, b in zip(src, dst)):
                raise ValueError("a row forks into a row with the same adapter")
            self._live = None
            K.page_fork(self.kv4, self.refcount, self.table, self.num, self.last, s, d, status=self.status)
            self.lens.copy_(self._row_lens())
        else:
            super().fork(src, dst)
        # The rows that the call began.  A refused one began none, whatever its dst held; a dst listed twice is refused.
        s, d = self._row_ids(src).long(), self._row_ids(dst).long()
        began = empty[d] & (self.num[d] > 0)
        self.pos[d] = torch.where(began, self.pos[s], self.pos[d])
        if self.budget is not None:
            self.weight[d] = torch.where(began[:, None], self.weight[s], self.weight[d])

    def release(self, rows: list[int]) -> None:
        super().release(rows)
        r = self._row_ids(rows).long()
        self.pos[r] = 0
        if self.budget is not None:
            self.weight[r] = 0.0
