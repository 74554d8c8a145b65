"""Paged int8 KV cache for a batch of sequences of different lengths (int8t64 format).

The reference serves one sequence at a time (src/nova/kvattn.py:326-327) and pads lengths to
power-of-two buckets with an additive -inf mask (src/nova/decode.py:39-48, 200-205). Here a batch
of ragged sequences shares one page pool per layer:

- a page is one 64-token group of one KV head: K codes (64 x 128 B), V codes, then the four fp16
  rulers ``kst | kmn | vst | vmn`` (128 each) = 17408 bytes, 128-byte aligned;
  ``pages[layer]`` is uint8 ``[num_pages, H_kv, 17408]``;
- ``page_table`` int32 ``[max_seqs, max_pages_per_seq]`` maps a sequence's group ``g`` to a page
  (the same page id in every layer's pool); -1 marks a slot without a page (never reserved, or
  released), and the kernels neither read nor write through it;
- each sequence keeps its own fp16 ring of the newest tokens (``rings[layer]`` fp16
  ``[max_seqs, H_kv, 2, 64, 128]``, K then V) and its write position ``pos[b]``.

A decode step appends one token per sequence (ring write + requantization of the ring into the
sequence's current page) and attends each sequence over exactly its own tokens ``[0, pos_b]``:
the bucket-padded positions the reference masks to -inf are not read, so whatever they hold
cannot change an output. Every computation is a HIP launch (``nkv_paged_decode_step_t64``);
lengths are device scalars, so one captured graph serves every step while pages stay reserved.

``PagedKVInt8TokCache`` holds the per-token symmetric format (one fp16 scale per token and KV
head) in the same page pool scheme: a page is 64 tokens of one KV head, K codes | V codes | K
scales (64 fp16) | V scales = 16640 bytes, 128-byte aligned. It keeps no ring; a decode step is
one launch (``nkv_paged_decode_step_tok``) that stores each sequence's new token into its page and
attends over ``[0, pos_b]``.

Several tokens per sequence in one step, packed (``nova_amd.chunks``): the per-token format's
``append_chunks`` (head norms, rotary embedding and quantized store) and ``attend_chunks`` (causal
attention over the pages); ``read`` brings cached tokens of either format back.

Host bookkeeping (``PagePool``: free pages, reservations, lengths; ``plan_parts``: the prefix
work plan) is plain Python so that its guards are testable without a GPU.
"""

from __future__ import annotations

import torch

from . import _lib
from . import chunks as C
from .chunks import ChunkPlan, SpanPlan
from .kvquant import _DT

D = 128
GT = 64
PAGE_BYTES = 2 * GT * D + 4 * D * 2
PAGE_BYTES_TOK = 2 * GT * D + 2 * GT * 2
CODE_BYTES = GT * D
MAX_PARTS_PER_SEQ = 256  # partials the tail's merge holds for one sequence
CUS = 256  # compute units of an MI355X: one workgroup each at a time


class PagePool:
    """Which pages each sequence owns, and how far each has written.

    ``reserve`` hands out pages for a sequence's first ``n`` tokens (always from group 0 up, the
    kernels rely on it); ``release`` returns them; ``advance`` records decode steps and refuses one
    that would write past the reserved pages. Table rows to write are returned to the caller."""

    def __init__(self, num_pages: int, max_seqs: int, max_pages_per_seq: int) -> None:
        self.num_pages, self.max_seqs, self.max_pages_per_seq = int(num_pages), int(max_seqs), int(max_pages_per_seq)
        self.free = list(range(self.num_pages - 1, -1, -1))
        self.owned: list[list[int]] = [[] for _ in range(self.max_seqs)]
        self.length = [0] * self.max_seqs

    def _seq(self, b: int) -> int:
        b = int(b)
        if not 0 <= b < self.max_seqs:
            raise ValueError(f"sequence {b} outside [0, {self.max_seqs})")
        return b

    def reserve(self, b: int, n_tokens: int) -> list[tuple[int, int]]:
        """Pages for every group of sequence ``b``'s first ``n_tokens`` tokens; returns the new
        ``(group, page)`` entries of its table row."""
        b = self._seq(b)
        need = -(-int(n_tokens) // GT)
        if need > self.max_pages_per_seq:
            raise ValueError(f"{n_tokens} tokens need {need} pages > max_pages_per_seq {self.max_pages_per_seq}")
        own = self.owned[b]
        if need - len(own) > len(self.free):
            raise RuntimeError(f"page pool exhausted: sequence {b} needs {need - len(own)} more pages, "
                               f"{len(self.free)} are free")
        new = []
        while len(own) < need:
            own.append(self.free.pop())
            new.append((len(own) - 1, own[-1]))
        return new

    def release(self, b: int) -> None:
        b = self._seq(b)
        self.free.extend(reversed(self.owned[b]))
        self.owned[b] = []
        self.length[b] = 0

    def set_length(self, b: int, n: int) -> None:
        b = self._seq(b)
        if n > 0 and (n - 1) // GT >= len(self.owned[b]):
            raise RuntimeError(f"sequence {b}: {n} tokens but only {len(self.owned[b])} pages reserved")
        self.length[b] = int(n)

    def advance(self, seqs: int, steps: int) -> None:
        """``steps`` decode steps of sequences ``0 .. seqs - 1``: each writes tokens at its length;
        the last one written must lie in a reserved page."""
        for b in range(seqs):
            last = self.length[b] + steps - 1
            if last // GT >= len(self.owned[b]):
                raise RuntimeError(f"sequence {b}: {steps} more steps write token {last}, beyond its "
                                   f"{len(self.owned[b])} reserved pages; reserve() more first")
        for b in range(seqs):
            self.length[b] += steps


def plan_parts(lengths: list[int], target_parts: int) -> tuple[list[int], list[int]]:
    """The prefix kernel's work plan: about ``target_parts`` units per KV head split over the
    sequences in proportion to their groups, each sequence at least one and at most
    ``MAX_PARTS_PER_SEQ``. Returns ``(wg_map, seq_parts)``: unit w serves sequence
    ``wg_map[w] >> 16``, part ``wg_map[w] & 0xffff``; ``seq_parts[2b]`` counts the parts
    of the sequences before b and ``seq_parts[2b + 1]`` those of b; the units themselves may be put in any
    order."""
    if not lengths:
        raise ValueError("no sequences to plan")
    groups = [max(1, int(n) // GT) for n in lengths]
    tot = sum(groups)
    parts = [max(1, min(MAX_PARTS_PER_SEQ, round(target_parts * gr / tot))) for gr in groups]
    wg_map, seq_parts = [], []
    for b, p in enumerate(parts):
        seq_parts += [len(wg_map), p]
        wg_map += [(b << 16) | i for i in range(p)]
    return wg_map, seq_parts


class PagedKVInt8Cache:
    page_bytes = PAGE_BYTES  # bytes of one page of one KV head
    has_rings = True

    def __init__(self, num_layers: int, num_kv_heads: int, head_dim: int, num_q_heads: int, max_seqs: int,
                 num_pages: int, max_pages_per_seq: int, device: str | torch.device = "cuda",
                 target_parts: int | None = None) -> None:
        if head_dim != D:
            raise NotImplementedError(f"head_dim {head_dim}: the HIP kernels are built for {D}")
        if num_q_heads % num_kv_heads or num_q_heads // num_kv_heads > 16:
            raise ValueError(f"Q heads {num_q_heads} / KV heads {num_kv_heads}")
        _lib.load()
        self.num_layers, self.num_kv_heads, self.head_dim = int(num_layers), int(num_kv_heads), int(head_dim)
        self.num_q_heads, self.max_seqs, self.num_pages = int(num_q_heads), int(max_seqs), int(num_pages)
        self.max_pages_per_seq, self.device = int(max_pages_per_seq), device
        self.pool = PagePool(self.num_pages, self.max_seqs, self.max_pages_per_seq)
        self.pages = [torch.zeros((self.num_pages, self.num_kv_heads, self.page_bytes), dtype=torch.uint8,
                                  device=device) for _ in range(self.num_layers)]
        self.rings = ([torch.zeros((self.max_seqs, self.num_kv_heads, 2, GT, D), dtype=torch.float16, device=device)
                       for _ in range(self.num_layers)] if self.has_rings else None)
        self.page_table = torch.full((self.max_seqs, self.max_pages_per_seq), -1, dtype=torch.int32, device=device)
        self.pos = torch.zeros(self.max_seqs, dtype=torch.long, device=device)
        self.merged = torch.zeros((self.max_seqs, self.num_q_heads, 1, D), dtype=torch.float16, device=device)
        self.lse = torch.zeros((self.max_seqs, self.num_q_heads), dtype=torch.float32, device=device)
        self.target_parts = int(target_parts or max(1, CUS // self.num_kv_heads))
        self.wg_map = self.seq_parts = self.ws = None
        self.total_parts = 0
        self.nseq = 0

    # the pool's lists, as attributes (tests hand out pages in a scrambled order through _free)
    @property
    def _free(self) -> list[int]:
        return self.pool.free

    @_free.setter
    def _free(self, ids: list[int]) -> None:
        self.pool.free = list(ids)

    @property
    def _owned(self) -> list[list[int]]:
        return self.pool.owned

    @property
    def _len(self) -> list[int]:
        return self.pool.length

    # ---- pages

    def reserve(self, b: int, n_tokens: int) -> None:
        """Give sequence ``b`` pages for every group of its first ``n_tokens`` tokens."""
        new = self.pool.reserve(b, n_tokens)
        if new:
            g0 = new[0][0]
            ids = torch.tensor([p for _, p in new], dtype=torch.int32)
            self.page_table[b, g0:g0 + len(new)] = ids.to(self.page_table.device)

    def release(self, b: int) -> None:
        """Return sequence ``b``'s pages to the pool; its table row goes back to -1, so a plan that
        still names it appends nothing and attends nothing for it."""
        self.pool.release(b)
        self.page_table[b].fill_(-1)
        self.pos[b] = 0

    # ---- prefill of one sequence

    def _check_prompt(self, key: torch.Tensor, value: torch.Tensor) -> int:
        h = self.num_kv_heads
        for name, x in (("key", key), ("value", value)):
            if x.dim() != 4 or x.shape[0] != 1 or x.shape[1] != h or x.shape[3] != D or x.dtype not in _DT:
                raise ValueError(f"{name} must be [1, {h}, n, {D}] fp16 / bf16 / fp32, got {tuple(x.shape)} {x.dtype}")
        if key.shape != value.shape:
            raise ValueError(f"key {tuple(key.shape)} and value {tuple(value.shape)} differ")
        return key.shape[2]

    def prefill(self, b: int, layer: int, key: torch.Tensor, value: torch.Tensor) -> None:
        """Store a prompt of n tokens (``[1, H_kv, n, 128]``) for sequence ``b``: whole groups
        quantized by the HIP quantizer straight into their pages (``nkv_paged_quantize_t64``, the
        int8t64 arithmetic bit for bit), the newest <= 64 tokens into its ring (slot = position
        mod 64)."""
        n = self._check_prompt(key, value)
        h = self.num_kv_heads
        self.reserve(b, n + 1)
        q = n // GT * GT
        if q:
            row = self.page_table[b]
            for which, x in enumerate((key, value)):
                xc = x if x.stride(3) == 1 and x.stride(2) == D and x.data_ptr() % 16 == 0 else x.contiguous()
                _lib.call("nkv_paged_quantize_t64", xc.data_ptr(), _DT[x.dtype], xc.stride(1), h, q, which,
                          self.pages[layer].data_ptr(), row.data_ptr(), 0, self.num_pages, _lib.stream_ptr(row.device))
        take = min(n, GT)
        if take:
            slots = torch.remainder(torch.arange(n - take, n, device=key.device), GT)
            self.rings[layer][b, :, 0].index_copy_(1, slots, key[0, :, n - take:n].to(torch.float16))
            self.rings[layer][b, :, 1].index_copy_(1, slots, value[0, :, n - take:n].to(torch.float16))
        self.pool.set_length(b, n)
        self.pos[b] = n

    # ---- cached tokens read back

    def plan_read(self, counts: list[int] | None = None, starts: list[int] | None = None) -> SpanPlan:
        """Which tokens :meth:`read` takes: ``counts[b]`` tokens of sequence ``b`` from ``starts[b]`` (default
        0) for sequences ``0 .. len(counts) - 1``; by default everything the sequences have."""
        if counts is None:
            n = self.max_seqs if starts is None else len(starts)
            counts = [self._len[b] - (0 if starts is None else int(starts[b])) for b in range(min(n, self.max_seqs))]
        counts = C.check_counts(counts, self.max_seqs)
        starts = [0] * len(counts) if starts is None else C.check_counts(starts, self.max_seqs, "starts")
        if len(starts) != len(counts):
            raise ValueError(f"{len(starts)} starts for {len(counts)} counts")
        for b, (s, n) in enumerate(zip(starts, counts)):
            if s + n > self._len[b]:
                raise ValueError(f"sequence {b}: tokens {s} .. {s + n - 1} of {self._len[b]}")
        return C.span_plan(counts, starts, self.pos)

    def read(self, plan: SpanPlan, layer: int, dtype: torch.dtype = torch.float16,
             out: tuple[torch.Tensor, torch.Tensor] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """The keys and values of ``plan``'s tokens as ``dtype`` (fp16 / bf16 / fp32), packed
        ``[tokens, H_kv, 128]``, in one launch: the values that the pages' codes stand for, rounded once (in
        the int8t64 format a sequence's tokens after its last whole group come from its fp16 ring). A token
        without a page is 0. ``out``: two contiguous tensors to write instead of new ones; rows after the
        plan's tokens stay as they are."""
        if dtype not in _DT:
            raise ValueError(f"unsupported dtype {dtype}")
        C.of_cache(plan, self.pos)
        dev, h = self.pos.device, self.num_kv_heads
        if out is None:
            k = torch.empty((plan.total, h, D), dtype=dtype, device=dev)
            out = k, torch.empty_like(k)
        else:
            for x in out:
                if (x.dim() != 3 or x.shape[0] < plan.total or x.shape[1:] != (h, D) or x.dtype != dtype or x.device != dev
                        or not x.is_contiguous() or x.data_ptr() % 16):
                    raise ValueError(f"out must be two contiguous, 16-byte aligned {dtype} tensors [{plan.total}, {h}, {D}] "
                                     f"on {dev}")
            if C.overlap(*out):
                raise ValueError("the two tensors of out overlap")
        self._read(plan, layer, dtype, *out)
        return out

    def _read(self, plan: SpanPlan, layer: int, dtype: torch.dtype, k: torch.Tensor, v: torch.Tensor) -> None:
        C.launch(self.pos.device, "nkv_paged_read_t64", self.pages[layer].data_ptr(), self.page_table.data_ptr(),
                 self.page_table.stride(0), self.num_pages, self.rings[layer].data_ptr(), self.pos.data_ptr(),
                 plan.seq_ptr, *plan.where, plan.total, plan.nseq, self.num_kv_heads, D, k.data_ptr(), v.data_ptr(),
                 _DT[dtype])

    # ---- work plan of the prefix kernel

    def plan(self, lengths: list[int] | None = None) -> None:
        """Split the prefix work of the active sequences into work units (about ``target_parts``
        per KV head, proportional to each sequence's groups, at most 256 per sequence) and size
        the workspace. Lengths default to the current ones; a plan stays valid while the lengths
        grow (each unit covers a fixed fraction of its sequence's groups)."""
        lengths = list(self._len if lengths is None else lengths)
        wg_map, seq_parts = plan_parts(lengths, self.target_parts)
        if len(wg_map) * self.num_kv_heads > CUS:
            # more workgroups than CUs: the longest units (in groups per wave) start first, so that the ones
            # that start last, or share a CU, are short. 48 sequences of 64 .. 2048 tokens: 43.0 -> 37.5 us
            # a layer (per-token format 31.6 -> 26.9), 64 of 100 .. 3000: 66 -> 54 us (45 -> 43)
            groups = [max(1, int(n) // GT) for n in lengths]
            wg_map.sort(key=lambda u: -(-(-groups[u >> 16] // (8 * seq_parts[2 * (u >> 16) + 1]))))
        dev = self.page_table.device
        self.wg_map = torch.tensor(wg_map, dtype=torch.int32, device=dev)
        self.seq_parts = torch.tensor(seq_parts, dtype=torch.int32, device=dev)
        self.total_parts = len(wg_map)
        nbytes = int(_lib.load().nkv_paged_workspace_bytes(self.num_kv_heads, self.num_q_heads, self.total_parts))
        if self.ws is None or self.ws.numel() * 4 < nbytes:
            self.ws = torch.zeros(nbytes // 4, dtype=torch.float32, device=dev)
        self.nseq = len(lengths)

    # ---- decode

    def _step_args(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor):
        n = self.nseq
        if q.shape != (n, self.num_q_heads, 1, D) or k.shape != (n, self.num_kv_heads, 1, D) or k.shape != v.shape:
            raise ValueError("q [B, Hq, 1, 128], k / v [B, Hkv, 1, 128] fp16, B = the planned sequences")
        return q.contiguous(), k.contiguous(), v.contiguous()

    def decode_step(self, key: torch.Tensor, value: torch.Tensor, query: torch.Tensor, layer: int) -> torch.Tensor:
        """Append one token per sequence at ``pos`` and attend each sequence over ``[0, pos_b]``, in
        one launch (``nkv_paged_decode_step_t64``: the tails append). Returns ``merged[:B]``
        ``[B, Hq, 1, 128]``; ``lse`` holds the log-sum-exp."""
        if self.wg_map is None:
            raise RuntimeError("call plan() before decoding")
        q, k, v = self._step_args(query, key, value)
        _lib.call("nkv_paged_decode_step_t64", q.data_ptr(), k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1),
                  self.pages[layer].data_ptr(), self.page_table.data_ptr(), self.page_table.stride(0), self.num_pages,
                  self.rings[layer].data_ptr(), self.pos.data_ptr(), self.nseq, self.num_q_heads, self.num_kv_heads,
                  D, self.wg_map.data_ptr(), self.seq_parts.data_ptr(), self.total_parts, self.merged.data_ptr(),
                  self.lse.data_ptr(), self.ws.data_ptr(), self.ws.numel() * 4, _lib.stream_ptr(self.pos.device))
        return self.merged[:self.nseq]

    def attend(self, query: torch.Tensor, layer: int) -> torch.Tensor:
        """Attention of each planned sequence over ``[0, pos_b]`` with nothing appended (the
        token at ``pos_b`` read from its ring slot), into ``merged[:B]`` / ``lse``: the second
        launch of ``decode_step`` alone (``nkv_paged_attn_decode_t64``)."""
        if self.wg_map is None:
            raise RuntimeError("call plan() before decoding")
        n = self.nseq
        if query.shape != (n, self.num_q_heads, 1, D):
            raise ValueError("q [B, Hq, 1, 128] fp16, B = the planned sequences")
        q = query.contiguous()
        _lib.call("nkv_paged_attn_decode_t64", q.data_ptr(), self.pages[layer].data_ptr(), self.page_table.data_ptr(),
                  self.page_table.stride(0), self.num_pages, self.rings[layer].data_ptr(), self.pos.data_ptr(), n,
                  self.num_q_heads, self.num_kv_heads, D, self.wg_map.data_ptr(), self.seq_parts.data_ptr(),
                  self.total_parts, self.merged.data_ptr(), self.lse.data_ptr(), self.ws.data_ptr(),
                  self.ws.numel() * 4, _lib.stream_ptr(self.pos.device))
        return self.merged[:n]

    def advance(self) -> None:
        """``pos += 1`` for every planned sequence (device op, graph-safe); refuses a step that
        would take a sequence past its reserved pages."""
        self.note_advanced(1)
        self.pos[:self.nseq].add_(1)

    def note_advanced(self, steps: int) -> None:
        """Host bookkeeping of ``steps`` decode steps that advanced every planned sequence on the
        device (``advance()``, or a replayed graph that adds to ``pos``). Raises when a sequence
        would write past the pages reserved for it."""
        self.pool.advance(self.nseq, steps)


class PagedKVInt8TokCache(PagedKVInt8Cache):
    """A batch of ragged sequences in the per-token symmetric format, in pages of 64 tokens of
    one KV head: K codes int8 ``[64, 128]``, V codes, K scales fp16 ``[64]``, V scales
    (16640 bytes). Codes and scales are those of ``nkv_quantize_tok`` bit for bit, token p of
    sequence b at row ``p % 64`` of page ``page_table[b, p // 64]``. Same pool, table, plan and
    graph-safe ``pos`` as ``PagedKVInt8Cache``; no rings."""

    page_bytes = PAGE_BYTES_TOK
    has_rings = False

    def prefill(self, b: int, layer: int, key: torch.Tensor, value: torch.Tensor) -> None:
        """Store a prompt of n tokens (``[1, H_kv, n, 128]``) for sequence ``b``: every token
        quantized by the HIP quantizer straight into its page (``nkv_paged_quantize_tok``)."""
        n = self._check_prompt(key, value)
        h = self.num_kv_heads
        self.reserve(b, n + 1)
        if n:
            row = self.page_table[b]
            for which, x in enumerate((key, value)):
                xc = x if x.stride(3) == 1 and x.stride(2) == D and x.data_ptr() % 16 == 0 else x.contiguous()
                _lib.call("nkv_paged_quantize_tok", xc.data_ptr(), _DT[x.dtype], xc.stride(1), h, n, which,
                          self.pages[layer].data_ptr(), row.data_ptr(), 0, self.num_pages, _lib.stream_ptr(row.device))
        self.pool.set_length(b, n)
        self.pos[b] = n

    def decode_step(self, key: torch.Tensor, value: torch.Tensor, query: torch.Tensor, layer: int) -> torch.Tensor:
        """Store one token per sequence at ``pos`` and attend each sequence over ``[0, pos_b]``, in
        one launch. Returns ``merged[:B]`` ``[B, Hq, 1, 128]``; ``lse`` holds the log-sum-exp."""
        if self.wg_map is None:
            raise RuntimeError("call plan() before decoding")
        q, k, v = self._step_args(query, key, value)
        _lib.call("nkv_paged_decode_step_tok", q.data_ptr(), k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1),
                  self.pages[layer].data_ptr(), self.page_table.data_ptr(), self.page_table.stride(0), self.num_pages,
                  self.pos.data_ptr(), self.nseq, self.num_q_heads, self.num_kv_heads, D, self.wg_map.data_ptr(),
                  self.seq_parts.data_ptr(), self.total_parts, self.merged.data_ptr(), self.lse.data_ptr(),
                  self.ws.data_ptr(), self.ws.numel() * 4, _lib.stream_ptr(self.pos.device))
        return self.merged[:self.nseq]

    # ---- steps of several tokens per sequence

    def plan_chunks(self, counts: list[int]) -> ChunkPlan:
        """Plan a step that brings ``counts[b]`` new tokens (0 or more) for each of the sequences
        ``0 .. len(counts) - 1``, and reserve their pages. The plan stays valid while the sequences grow (the
        cut of the attention follows their lengths on the device), for any number of layers and steps that
        bring the same counts; reserve further pages before further steps.

        Made once a step, for all layers, in 0.16 to 0.25 ms of host time, and 0.02 ms more for each sequence
        that gets new pages; its copies to the device wait for the work queued on the current stream."""
        counts = C.check_counts(counts, self.max_seqs)
        need = [-(-(self._len[b] + n) // GT) - len(self._owned[b]) for b, n in enumerate(counts)]
        if sum(n for n in need if n > 0) > len(self._free):
            raise RuntimeError(f"page pool exhausted: the step needs {sum(n for n in need if n > 0)} more pages, "
                               f"{len(self._free)} are free")
        for b, n in enumerate(counts):
            if self._len[b] + n > self.max_pages_per_seq * GT:
                raise ValueError(f"sequence {b}: {self._len[b]} + {n} tokens exceed max_pages_per_seq "
                                 f"{self.max_pages_per_seq}")
        for b, n in enumerate(counts):
            if n:
                self.reserve(b, self._len[b] + n)
        return C.chunk_plan(counts, self._len[:len(counts)], self.pos, self.num_q_heads // self.num_kv_heads,
                            self.num_kv_heads)

    def append_chunks(self, plan: ChunkPlan, qkv: torch.Tensor, layer: int, q_gamma: torch.Tensor | None = None,
                      k_gamma: torch.Tensor | None = None, eps: float = 1e-6, inv_freq: torch.Tensor | None = None,
                      q_out: torch.Tensor | None = None) -> torch.Tensor:
        """Store the new tokens' keys and values in their pages and return their queries, in one launch.

        ``qkv``: the stacked projections ``[tokens, (H_q + 2 H_kv) * 128]`` (q heads, k heads, v heads; fp16 /
        bf16 / fp32, unit element stride). With ``q_gamma`` / ``k_gamma`` (``[128]``, of qkv's type) each q and
        k head gets its RMSNorm, with ``inv_freq`` (fp32 ``[64]``) the rotary embedding at the token's own
        position (element i with i + 64). All of it in fp32, rounded once: q to fp16, K and V to the codes and
        scales of ``quantize_tok``. A token whose page is missing is not stored. Returns fp16 ``[tokens, H_q,
        128]``, or writes ``q_out``, which may be qkv's own q heads; rows after the plan's tokens are neither
        read nor written."""
        hq, hkv, dev, total = self.num_q_heads, self.num_kv_heads, self.pos.device, plan.total
        C.step_of_cache(plan, self.pos)
        shape, dtype, width = qkv.shape, qkv.dtype, (hq + 2 * hkv) * D
        if len(shape) != 2 or shape[0] < total or shape[1] != width or dtype not in _DT or qkv.device != dev:
            raise ValueError(f"qkv must be fp16 / bf16 / fp32 [{total}, {width}] on {dev} (more tokens may "
                             f"follow), got {tuple(shape)} {dtype} on {qkv.device}")
        if (q_gamma is None) != (k_gamma is None):
            raise ValueError("q_gamma and k_gamma come together")
        if q_gamma is not None:
            for name, t in (("q_gamma", q_gamma), ("k_gamma", k_gamma)):
                if t.dtype != dtype or t.numel() != D or not t.is_contiguous() or t.device != dev or t.data_ptr() % 16:
                    raise ValueError(f"{name} must be a contiguous, 16-byte aligned {dtype} tensor of {D} elements on {dev}")
        if inv_freq is not None and (inv_freq.dtype != torch.float32 or inv_freq.numel() != D // 2
                                     or not inv_freq.is_contiguous() or inv_freq.device != dev):
            raise ValueError(f"inv_freq must be a contiguous fp32 tensor of {D // 2} elements on {dev}")
        given, (row, element) = qkv, qkv.stride()
        if element != 1 or row % 8 or qkv.data_ptr() % 16 or (row < width and shape[0] > 1):
            qkv = qkv.clone(memory_format=torch.contiguous_format)  # (contiguous() keeps rows that start between)
            row = width
        if q_out is None:
            q_out = torch.empty((total, hq, D), dtype=torch.float16, device=dev)
        else:
            C.heads_of(q_out, "q_out", total, hq, dev)
            if q_out.stride(1) != D or not C.rows_in_place(q_out) or not C.distinct_rows(q_out):
                raise ValueError("q_out: a token's heads must be contiguous and its row 16-byte aligned")
            own_rows = (given is qkv and q_out.data_ptr() == qkv.data_ptr() and q_out.dtype == dtype
                        and (q_out.stride(0) == row or total <= 1))
            if not own_rows and C.overlap(q_out, given):
                raise ValueError("q_out must be qkv's q heads themselves or not overlap qkv")
        C.launch(dev, "nkv_paged_append_chunks_tok", qkv.data_ptr(), _DT[dtype], max(row, width), total,
                 self.pages[layer].data_ptr(), self.page_table.data_ptr(), self.page_table.stride(0), self.num_pages,
                 plan.seq_ptr, *plan.where, plan.nseq, hq, hkv, D, _lib.ptr(q_gamma), _lib.ptr(k_gamma), float(eps),
                 _lib.ptr(inv_freq), q_out.data_ptr(), max(q_out.stride(0), hq * D))
        return q_out

    def attend_chunks(self, plan: ChunkPlan, query: torch.Tensor, layer: int, out: torch.Tensor | None = None,
                      lse: torch.Tensor | None = None) -> torch.Tensor:
        """Causal attention of the new tokens over their sequences' pages, the step's own keys and values
        among them (``append_chunks`` runs first): the token at position p attends ``[0, p]``.

        ``query`` fp16 ``[tokens, H_q, 128]`` (any token and head strides; rows that do not start on 16 bytes are
        copied). Returns ``out``, fp16 of the same shape (strides as query's), which must not overlap ``query``;
        ``lse`` (fp32 ``[tokens, H_q]``, contiguous) receives the log-sum-exp of the scaled scores. Groups
        without a page take no part; a token with none gets 0 and -inf. Rows after the plan's tokens are neither
        read nor written. Calls may overlap on streams (each has its own scratch memory). The plan decides the order
        of the sums: the same sequence in another batch, or in a plan made at other lengths, may give other last bits."""
        hq, hkv, dev, total = self.num_q_heads, self.num_kv_heads, self.pos.device, plan.total
        C.step_of_cache(plan, self.pos)
        C.heads_of(query, "query", total, hq, dev)
        if not C.rows_in_place(query):
            query = query.clone(memory_format=torch.contiguous_format)
        if out is None:
            out = torch.empty((total, hq, D), dtype=torch.float16, device=dev)
        else:
            C.heads_of(out, "out", total, hq, dev)
            if not C.rows_in_place(out) or not C.distinct_rows(out):
                raise ValueError("out: rows of 128 elements, apart from each other, must start on 16 bytes")
            if C.overlap(out, query):
                raise ValueError("out must not overlap query")
        if lse is not None and (lse.dtype != torch.float32 or lse.dim() != 2 or lse.shape[0] < total or lse.shape[1] != hq
                                or not lse.is_contiguous() or lse.device != dev):
            raise ValueError(f"lse must be a contiguous fp32 tensor [{total}, {hq}] on {dev}")
        ws = _lib.scratch(dev, plan.ws_bytes) if plan.ws_bytes else None
        C.launch(dev, "nkv_paged_attn_chunks_tok", query.data_ptr(), query.stride(0), query.stride(1), total,
                 self.pages[layer].data_ptr(), self.page_table.data_ptr(), self.page_table.stride(0), self.num_pages,
                 *plan.where, plan.nseq, hq, hkv, D, *plan.work, out.data_ptr(), *out.stride()[:2], _lib.ptr(lse), _lib.ptr(ws),
                 plan.ws_bytes)
        return out

    def advance_chunks(self, plan: ChunkPlan, accepted: list[int] | None = None) -> None:
        """``pos`` moves past the step's tokens, or past the first ``accepted[b]`` of each sequence's (drafted
        tokens that were kept; the others' places are written again). Refuses a step whose pages are not
        reserved."""
        self.note_chunks(plan, 1, accepted)
        if accepted is None:
            self.pos[:plan.nseq].add_(plan.new)
        else:
            self.pos[:plan.nseq].add_(torch.tensor([int(n) for n in accepted], dtype=torch.int64).to(self.pos.device))

    def note_chunks(self, plan: ChunkPlan, steps: int = 1, accepted: list[int] | None = None) -> None:
        """Host bookkeeping of ``steps`` steps that advanced ``pos`` on the device (:meth:`advance_chunks`, or a
        replayed graph that adds ``plan.new`` to ``pos[:plan.nseq]``)."""
        C.step_of_cache(plan, self.pos)
        if steps < 0:
            raise ValueError(f"{steps} steps")
        moved = plan.counts if accepted is None else C.check_counts(accepted, self.max_seqs, "accepted")
        if len(moved) != plan.nseq or any(a > n for a, n in zip(moved, plan.counts)):
            raise ValueError(f"accepted {moved} of a step of {plan.counts}")
        for b, n in enumerate(moved):
            if n and (self._len[b] + n * int(steps) - 1) // GT >= len(self._owned[b]):
                raise RuntimeError(f"sequence {b}: {n * int(steps)} more tokens after {self._len[b]}, but only "
                                   f"{len(self._owned[b])} pages reserved; reserve() more first")
        for b, n in enumerate(moved):
            self.pool.set_length(b, self._len[b] + n * int(steps))

    def _read(self, plan: SpanPlan, layer: int, dtype: torch.dtype, k: torch.Tensor, v: torch.Tensor) -> None:
        C.launch(self.pos.device, "nkv_paged_read_tok", self.pages[layer].data_ptr(), self.page_table.data_ptr(),
                 self.page_table.stride(0), self.num_pages, plan.seq_ptr, *plan.where, plan.total, plan.nseq,
                 self.num_kv_heads, D, k.data_ptr(), v.data_ptr(), _DT[dtype])
