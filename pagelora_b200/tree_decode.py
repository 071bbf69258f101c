"""Speculative, branching and sparse decode over a batch engine's cache.

:class:`TreeDecoder` takes over the rows of a prefilled
:class:`~pagelora_b200.batch_engine.BatchDecodeEngine` and keeps their page
bookkeeping on the device.  One verification step of drafted trees is

    page_reserve (slots of all drafted tokens, page table) -> tree_mask
    per layer:  (rmsnorm + LoRA shrink ->) q/k/v projection -> q/k norm + RoPE
                + KV append -> paged_tree_attention -> o projection -> MLP
    lm_head -> argmax -> tree_accept -> cache_compact (the accepted path's K/V
    move together, the rest of the drafts' pages go back to the pool)

with no host synchronisation; rows fork and end with :meth:`fork` and
:meth:`release`.  What the device refuses (a row or the pool without room)
changes no row and accepts no token; :meth:`check` says why.  With ``sparse``
the decoder also keeps the int8 key bounds of every page, and
:meth:`step_sparse` decodes one token per row over the pages that their score
selects.  No reference counterpart: the reference decodes one token per row and
step (model/flashinfer/generation.py:188-247).
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from pagelora_b200 import kernels as K
from pagelora_b200._capi import PL_PROLOGUE_RMSNORM, PL_PROLOGUE_SILU_MUL
from pagelora_b200.batch_engine import BatchDecodeEngine


@dataclass(frozen=True)
class SparsePages:
    """Page budget of a sparse step: the first ``sink`` and last ``recent``
    pages of a row and the highest scores, ``select`` in all."""

    select: int
    sink: int = 1
    recent: int = 2


@dataclass
class TreeStep:
    """Result of :meth:`TreeDecoder.verify` (device tensors).  A step that was
    refused keeps nothing: keep -1, keep_count 0, next_token -1, and targets and
    logits without meaning."""

    targets: torch.Tensor     # int64 [tokens]: the model's choice after each drafted token
    keep: torch.Tensor        # int32 [rows, max]: positions of the accepted path, then -1
    keep_count: torch.Tensor  # int32 [rows]
    next_token: torch.Tensor  # int64 [rows]: the choice after the accepted path
    logits: torch.Tensor      # bf16 [tokens, vocab]


class TreeDecoder:
    """Takes over ``engine``'s rows (``engine.step_*`` must not be used any
    more).  Drafted trees of all rows are given flat, row after row; token 0
    of a row's tree is its last sampled token, whose K/V are not cached yet."""

    def __init__(self, engine: BatchDecodeEngine, *, sparse: SparsePages | None = None) -> None:
        if engine.world != 1 or engine.cascade is not None:
            raise ValueError("the engine's rows must hold their whole context (no split-KV, no shared prefix)")
        spec = engine.spec
        if engine.lora_rank and max(spec.hidden, spec.q_dim) > K.SHRINK_ROWS_MAX_K:
            raise ValueError(f"LoRA rows need hidden and query features <= {K.SHRINK_ROWS_MAX_K}")
        if sparse is not None:
            if sparse.sink < 0 or sparse.recent < 1 or sparse.sink + sparse.recent > sparse.select:
                raise ValueError("a page budget needs sink >= 0, recent >= 1 and sink + recent <= select")
            if engine.page_size not in (16, 32) or spec.num_qo_heads > 16 * spec.num_kv_heads:
                raise ValueError("sparse decode needs pages of 16 or 32 tokens and at most 16 query heads per kv head")
        self.e = engine
        dev = engine.device
        self.table, self.num, self.last = engine.row_pages, engine.row_num_pages, engine.last_page_len
        self.rows, self.cap = self.table.shape
        self.status = engine.status
        held = torch.tensor([p for pages in engine.host_pages for p in pages], dtype=torch.int64)
        self.refcount = torch.bincount(held, minlength=engine.num_pages).to(device=dev, dtype=torch.int32)
        self.lens = torch.tensor(engine.context_len, dtype=torch.int32, device=dev)
        self.indptr = torch.zeros(self.rows + 1, dtype=torch.int32, device=dev)
        self.indices = torch.zeros(self.rows * self.cap, dtype=torch.int32, device=dev)
        self._none = torch.zeros(self.rows, dtype=torch.int32, device=dev)
        # the rows that step_sparse advances: (row ids, their slots' indptr); None: not known
        self._live = None
        self._ended = 0 in engine.context_len  # some row may be without a context
        self._gemm_ws: dict[int, torch.Tensor] = {}
        self.sparse = sparse
        if sparse is not None:
            layers, pages, _, _, hkv, d = engine.kv.shape
            self.bounds = torch.zeros(layers, pages, hkv, 2, d, dtype=torch.int8, device=dev)
            self.bound_scale = torch.zeros(layers, pages, hkv, device=dev)
            self._refresh_bounds(torch.zeros_like(self.num), self.cap)

    # ------------------------------------------------------------- forward
    def _linear(self, x, w, *, prologue=0, norm_weight=None, gemm=False, **kw):
        """One projection of any number of tokens: the fused GEMV for few, the
        tcgen05 GEMM in blocks of 128 for more."""

        s, tokens = self.e.spec, x.shape[0]
        if not gemm and K.gemv_fits(tokens, w.shape[1]):
            return K.linear_lora_fused(x, w, prologue=prologue, norm_weight=norm_weight, norm_eps=s.rms_eps,
                                       weights_static=True, status=self.status, **kw)
        if prologue == PL_PROLOGUE_RMSNORM:
            x = K.rmsnorm(x, norm_weight, s.rms_eps)
        elif prologue == PL_PROLOGUE_SILU_MUL:
            x = K.silu_mul(x)
        wide = w.shape[0] // (2 if kw.get("silu_pairs") else 1)
        out = kw.pop("out", None)
        if out is None:
            out = torch.empty(tokens, wide, dtype=torch.bfloat16, device=x.device)
        per_token = ("lora_down", "tok_adapter", "residual")
        for t0 in range(0, tokens, K.GEMM_MAX_ROWS):
            part = slice(t0, min(tokens, t0 + K.GEMM_MAX_ROWS))
            n = part.stop - t0
            need = int(K.gemm_plan(n, w.shape[1], w.shape[0]).workspace_bytes)
            ws = self._gemm_ws.get(n)
            if ws is None or ws.numel() < need:
                ws = self._gemm_ws[n] = torch.zeros(need, dtype=torch.uint8, device=x.device)
            cut = {k: (v[part] if k in per_token and v is not None else v) for k, v in kw.items()}
            K.linear_lora_gemm(x[part], w, out=out[part], workspace=ws, weights_static=True, status=self.status, **cut)
        return out

    def _forward(self, tokens, positions, tok_row, slot_page, slot_off, attend) -> torch.Tensor:
        """Logits of ``tokens`` whose K/V go to the given slots; ``attend(layer,
        q)`` is the attention of one layer over the cache."""

        e, s = self.e, self.e.spec
        n = tokens.numel()
        x = torch.empty(n, s.hidden, dtype=torch.bfloat16, device=tokens.device)
        K.embed(tokens, e.embed, x, self.status)
        lora = e.lora_rank > 0
        adapter = e.tok_adapter[tok_row] if lora else None
        q = torch.empty(n, s.num_qo_heads, s.head_dim, dtype=torch.bfloat16, device=x.device)
        for li, L in enumerate(e.layers):
            down = None
            if lora:
                xn = torch.empty_like(x)
                down = K.lora_shrink_rows(x, L["a_qkv"], tok_adapter=adapter, norm_weight=L["input_norm"],
                                          norm_eps=s.rms_eps, xn_out=xn)
                qkv = self._linear(xn, L["w_qkv"])
            else:
                qkv = self._linear(x, L["w_qkv"], prologue=PL_PROLOGUE_RMSNORM, norm_weight=L["input_norm"])
            kv, kv_page, kv_off = self._kv_target(li, slot_page, slot_off)
            K.qkv_rope_append(qkv, num_qo_heads=s.num_qo_heads, num_kv_heads=s.num_kv_heads, head_dim=s.head_dim,
                              positions=positions, rope_theta=s.rope_theta, kv_cache=kv, page_id=kv_page,
                              page_offset=kv_off, q_out=q, lora_down=down, lora_b=L["b_qkv"] if lora else None,
                              lora_scale=e.qkv_lora_scale, tok_adapter=adapter, q_norm_weight=L["q_norm"],
                              k_norm_weight=L["k_norm"], norm_eps=s.rms_eps, status=self.status)
            attn = attend(li, q).view(n, s.q_dim)
            down_o = K.lora_shrink_rows(attn, L["a_o"], tok_adapter=adapter) if lora else None
            x = self._linear(attn, L["w_o"], lora_down=down_o, lora_b=L["b_o"] if lora else None,
                             lora_scale=e.lora_scale, tok_adapter=adapter, residual=x)
            if e.silu_pairs:
                act = self._linear(K.rmsnorm(x, L["post_norm"], s.rms_eps), L["w_gate_up"], gemm=True, silu_pairs=True)
                x = self._linear(act, L["w_down"], gemm=True, residual=x)
            else:
                gate_up = self._linear(x, L["w_gate_up"], prologue=PL_PROLOGUE_RMSNORM, norm_weight=L["post_norm"])
                x = self._linear(gate_up, L["w_down"], prologue=PL_PROLOGUE_SILU_MUL, residual=x)
        return self._linear(x, e.lm_head, prologue=PL_PROLOGUE_RMSNORM, norm_weight=e.final_norm)

    def _kv_target(self, li, slot_page, slot_off):
        """(pool, pages, offsets) that a layer's new K/V are written to."""

        return self.e.kv[li], slot_page, slot_off

    def _reserve(self, tok_indptr, total):
        slot_page = torch.empty(total, dtype=torch.int32, device=self.lens.device)
        slot_off, positions = torch.empty_like(slot_page), torch.empty_like(slot_page)
        K.page_reserve(self.refcount, self.table, self.num, self.last, tok_indptr, self.e.page_size,
                       slot_page=slot_page, slot_offset=slot_off, positions=positions, out_indptr=self.indptr,
                       out_indices=self.indices, status=self.status)
        return slot_page, slot_off, positions

    def _row_lens(self) -> torch.Tensor:
        """Cached tokens of every row, from its pages."""

        ps = self.e.page_size
        return torch.add(self.last, self.num, alpha=ps).sub_(ps).clamp_(min=0)

    @staticmethod
    def _need_tokens(tokens: torch.Tensor, n: int) -> None:
        K._vecs(torch.int64, "tokens", (tokens,), (n,))
        if tokens.dim() != 1 or tokens.numel() != n:
            raise ValueError(f"tokens must be [{n}]")

    def _row_ids(self, rows: list[int]) -> torch.Tensor:
        if any(not 0 <= r < self.rows for r in rows):
            raise ValueError(f"rows are 0 .. {self.rows - 1}")
        return torch.tensor(rows, dtype=torch.int32, device=self.lens.device)

    # --------------------------------------------------------------- steps
    @torch.no_grad()
    def verify(self, tokens: torch.Tensor, parents: torch.Tensor, qo_indptr: torch.Tensor, max_tokens: int) -> TreeStep:
        """One verification step.  ``tokens`` int64 [total] and ``parents``
        int32 [total] (index in the row's tree, -1 for its token 0) hold row
        r's tree at qo_indptr[r]:qo_indptr[r+1], at most ``max_tokens`` each;
        a row without tokens stays as it is."""

        total = tokens.numel()
        self._need_tokens(tokens, total)
        K._vecs(torch.int32, "parents qo_indptr", (parents, qo_indptr), (total, self.rows + 1))
        if parents.numel() != total or qo_indptr.numel() != self.rows + 1 or max_tokens < 1:
            raise ValueError("parents needs an entry per token, qo_indptr one per row and one more, max_tokens >= 1")
        if total == 0:
            logits = torch.empty(0, self.e.lm_head.shape[0], dtype=torch.bfloat16, device=tokens.device)
            return TreeStep(tokens.clone(), self._none.new_full((self.rows, max_tokens), -1), self._none.clone(),
                            tokens.new_full((self.rows,), -1), logits)
        if self._ended:  # a draft may begin an empty row
            self._live = None
        tok_row = torch.searchsorted(qo_indptr[1:], torch.arange(total, device=tokens.device, dtype=torch.int32),
                                     right=True)
        slot_page, slot_off, _ = self._reserve(qo_indptr, total)
        positions = torch.empty(total, dtype=torch.int32, device=tokens.device)
        mask, _ = K.tree_mask(parents, qo_indptr, (max_tokens + 31) // 32, base_positions=self.lens,
                              positions=positions, status=self.status)

        def attend(li, q):
            return K.paged_tree_attention(q, self.e.kv[li], qo_indptr, self.indptr, self.indices, self.last, mask,
                                          status=self.status)

        logits = self._forward(tokens, positions, tok_row, slot_page, slot_off, attend)
        targets = K.argmax(logits, torch.empty_like(tokens))
        keep = torch.empty(self.rows, max_tokens, dtype=torch.int32, device=tokens.device)
        count = torch.empty(self.rows, dtype=torch.int32, device=tokens.device)
        nxt = torch.empty(self.rows, dtype=torch.int64, device=tokens.device)
        K.tree_accept(parents, tokens, targets, qo_indptr, self.lens, keep=keep, keep_count=count, next_token=nxt,
                      status=self.status)
        tables = (self.e.kv, self.refcount, self.table, self.num, self.last)
        K.cache_compact(*tables, self.lens, keep, count, status=self.status)
        # A refused reservation or compaction left the rows as they were before
        # it: the step keeps nothing, and the drafts' pages are given back.
        # (Cutting rows to the length that they have changes nothing.)
        undone = (self._row_lens() != self.lens + count).any()
        for t, nothing in ((count, 0), (keep, -1), (nxt, -1)):
            t.masked_fill_(undone, nothing)
        first = self.lens // self.e.page_size if self.sparse is not None else None
        self.lens.add_(count)
        K.cache_compact(*tables, self.lens, keep, self._none, status=self.status)
        if first is not None:
            self._refresh_bounds(first, (max_tokens - 1) // self.e.page_size + 2)
        return TreeStep(targets, keep, count, nxt, logits)

    def _live_rows(self) -> tuple[torch.Tensor, torch.Tensor]:
        """The rows that hold a context, ascending, and the indptr of one token
        each.  Waits for the device when rows may have ended or begun since."""

        if self._live is None:
            dev = self.lens.device
            live = torch.ones(self.rows, dtype=torch.int32)
            if self._ended:
                live = (self.num > 0).to("cpu", torch.int32)
                self._ended = not live.all()
            indptr = torch.cat([live.new_zeros(1), live.cumsum(0, dtype=torch.int32)])
            self._live = live.nonzero().flatten().to(dev), indptr.to(dev)
        return self._live

    @torch.no_grad()
    def step_sparse(self, tokens: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """One token per row (int64 [rows]) over the selected pages; returns
        (next tokens [rows], logits [rows, vocab]).  Rows without a context take
        no part: their next token is -1 and their logits are 0.  A step that was
        refused returns -1 for every row."""

        if self.sparse is None:
            raise ValueError("the decoder was built without a page budget (sparse)")
        self._need_tokens(tokens, self.rows)
        rows, tok_indptr = self._live_rows()
        n, some = rows.numel(), rows.numel() < self.rows
        if n == 0:
            logits = torch.zeros(self.rows, self.e.lm_head.shape[0], dtype=torch.bfloat16, device=rows.device)
            return torch.full_like(tokens, -1), logits
        slot_page, slot_off, positions = self._reserve(tok_indptr, n)
        indptr, last = self.indptr, self.last
        if some:  # (rows without a context have no pages between those of the others)
            tokens, last = tokens[rows], last[rows]
            indptr = torch.cat([indptr[rows], indptr[-1:]])
        sp = self.sparse

        def attend(li, q):
            kv, bounds, scale = self.e.kv[li], self.bounds[li], self.bound_scale[li]
            # the page that takes the token is among the recent ones, whose
            # bounds are not read; they are kept current for when it is not
            K.page_bounds(kv, slot_page, bounds, scale, page_len=slot_off + 1, status=self.status)
            return K.paged_sparse_decode(q, kv, indptr, self.indices, last, bounds, scale, num_select=sp.select,
                                         sink_pages=sp.sink, recent_pages=sp.recent, max_pages=self.cap,
                                         status=self.status)

        logits = self._forward(tokens, positions, rows, slot_page, slot_off, attend)
        nxt = K.argmax(logits, torch.empty_like(tokens))
        lens = self._row_lens()
        nxt.masked_fill_((lens == self.lens).all(), -1)  # the reservation is for all rows or for none
        self.lens.copy_(lens)
        if some:
            nxt = nxt.new_full((self.rows,), -1).index_copy_(0, rows, nxt)
            logits = logits.new_zeros(self.rows, logits.shape[1]).index_copy_(0, rows, logits)
        return nxt, logits

    # ---------------------------------------------------------------- rows
    def fork(self, src: list[int], dst: list[int]) -> None:
        """Empty rows ``dst`` continue as copies of ``src`` (same adapters)."""

        s, d = self._row_ids(src), self._row_ids(dst)
        if len(src) != len(dst):
            raise ValueError("src and dst differ in length")
        if any(self.e.row_adapter[a] != self.e.row_adapter[b] for a, b in zip(src, dst)):
            raise ValueError("a row forks into a row with the same adapter")
        self._live = None
        K.page_fork(self.e.kv, self.refcount, self.table, self.num, self.last, s, d, status=self.status)
        self.lens.copy_(self._row_lens())
        if self.sparse is not None:  # the copied last pages
            self._refresh_bounds((self.num - 1).clamp(min=0), 1)

    def release(self, rows: list[int]) -> None:
        """The rows end: their pages go back to the pool, and they stay empty
        until a fork or a draft begins them anew."""

        r = self._row_ids(rows)
        self._live, self._ended = None, True
        K.page_release(self.refcount, self.table, self.num, self.last, r, status=self.status)
        self.lens.copy_(self._row_lens())

    def check(self) -> None:
        """Raises when a step reported a device status (the first one since the
        last call, which this one clears)."""

        try:
            self.e._check_status()
        finally:
            self.status.zero_()

    def _refresh_bounds(self, first: torch.Tensor, most: int) -> None:
        """Bounds of the pages first[r] .. of every row (at most ``most``)."""

        at = first[:, None] + torch.arange(most, device=first.device, dtype=torch.int32)
        at = torch.minimum(at, (self.num - 1).clamp(min=0)[:, None])
        ids = torch.gather(self.table, 1, at.long())
        length = torch.where(at == self.num[:, None] - 1, self.last[:, None], self.e.page_size)
        live = (self.num > 0)[:, None]  # rows without pages: entries that page_bounds leaves out
        ids, length = torch.where(live, ids, -1), torch.where(live, length, 0)
        for li in range(self.e.kv.shape[0]):
            K.page_bounds(self.e.kv[li], ids, self.bounds[li], self.bound_scale[li], page_len=length,
                          status=self.status)
