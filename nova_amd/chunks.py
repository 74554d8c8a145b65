"""Plans of the paged caches' calls over several tokens per sequence.

A step of a paged batch may bring any number of tokens for each sequence: a prompt's chunk, a few
drafted tokens, one decode token, none. The tokens are packed one after another, sequence 0's
first, as ``[tokens, heads, 128]``. ``SpanPlan`` says which tokens of which sequences a packed
tensor holds; ``ChunkPlan`` adds how their attention is cut into work units. Plans are read only
(any number of calls, layers and graphs may share one) and hold the counts fixed, while positions
come from the cache's device tensor ``pos``, so a captured step follows the sequences as they grow.

``plan_units`` is plain Python on integers, testable without a GPU. The reference decodes one token
of one sequence (src/nova/kvattn.py:326-327) and has no paged layout.
"""

from __future__ import annotations

from dataclasses import dataclass

import numpy as np
import torch

from . import _lib

D, GT = 128, 64
CUS = 256        # compute units of an MI355X: one attention workgroup each at a time
UNIT_INTS = 8    # int32 words of a work unit and of a merge entry
ROWS16, ROWS32, ROWS256 = 0, 1, 2  # unit kinds
TILE_ROWS = {ROWS16: 16, ROWS32: 32, ROWS256: 256}  # query rows (tokens x q heads per KV head) of a tile, at most
MERGE_ROWS = 8   # rows a merge entry covers
MAX_PARTS = 256
# Rows of a sequence from which its tiles are ROWS256 (32 query and 8 KV heads; all as ROWS256 / as ROWS32): 64 rows over
# 32000 tokens 52 / 32 us, 96 rows 52 / 49, 8 times 128 rows over 4000 tokens 53 / 42, 256 rows 62 / 65. (Set when the
# small units were slower, at 42, 56, 58 and 89 us: up to about 200 rows they are now the faster ones.)
BIG_FROM = 64
# 64-token groups of a small unit's part, at least: 32 rows over 4000 tokens 16.4 us (8: 18.8; 1: 15.7), 4 times one
# token over 2000 12.4 us (8: 13.4; 1: 12.4)
SMALL_PART = 4
# prices of a cut in us: a step of a wide tile, a group of a small one with the card full of them, a unit's start and end,
# the second launch, a partial row written and read. The cut that they choose is within 10% of the best of CUTS for every
# batch of the comment above, prompts of 512 and 4096 tokens, chunks of 256 to 2048 over 8192 to 32000, 1 to 64
# sequences of one token over 2000 to 131000.
STEP_US, GROUP_US, UNIT_US, MERGE_US, PARTIAL_US = 2.4, 0.75, 7.0, 5.0, 0.0002
CUTS = (1, 1.5, 2, 3, 4, 6, 8, 12, 16, 24, 32, 64, 128, 256)


@dataclass
class SpanPlan:
    """Tokens ``starts[b] .. starts[b] + counts[b] - 1`` of sequences ``0 .. nseq - 1``, packed. A captured graph reads
    the plan's tensors: keep the plan as long as the graph."""

    counts: list[int]
    total: int
    pos: torch.Tensor      # the positions of the cache that made the plan
    starts: torch.Tensor   # int64 [nseq] on the device
    cu: torch.Tensor       # int32 [nseq + 1]: where each sequence's tokens begin in the packed tensor
    seq_of: torch.Tensor   # int32 [total]: the sequence of each packed token

    def __post_init__(self):
        self.nseq = len(self.counts)
        self.where = self.cu.data_ptr(), self.starts.data_ptr()  # (the plan's own memory: the addresses stay)
        self.seq_ptr = self.seq_of.data_ptr()


@dataclass
class ChunkPlan(SpanPlan):
    """A step's new tokens: ``starts`` is the cache's ``pos`` itself, ``new`` the counts on the device."""

    new: torch.Tensor = None      # int64 [nseq]
    units: torch.Tensor = None    # int32 [n, 8]
    merges: torch.Tensor = None   # int32 [m, 8]
    ws_bytes: int = 0
    wide: bool = False            # some unit is ROWS256
    kind: int = ROWS16            # the largest kind of a unit

    def __post_init__(self):
        super().__post_init__()
        self.work = self.units.data_ptr(), self.units.shape[0], self.wide, self.merges.data_ptr(), self.merges.shape[0]
        self.work_q4 = *self.work[:2], self.kind, *self.work[3:]


def check_counts(counts, max_seqs: int, what: str = "counts") -> list[int]:
    counts = [int(n) for n in counts]
    if not 0 < len(counts) <= max_seqs:
        raise ValueError(f"{what} for {len(counts)} sequences; the cache has {max_seqs}")
    if min(counts) < 0:
        raise ValueError(f"{what} must not be negative, got {min(counts)}")
    return counts


def plan_units(starts, counts, gq: int, hkv: int, q4: bool = False) -> tuple[np.ndarray, np.ndarray, int]:
    """How the attention of ``counts[b]`` new tokens after ``starts[b]`` is cut.

    Returns ``(units, merges, partial_rows)``, int32 ``[n, 8]`` and ``[m, 8]``. The rows of a KV head
    (``counts[b] * gq``, token-major) are cut into tiles, a tile's 64-token groups into parts; a
    unit is one part of one tile: ``(sequence, first row, rows, part, parts, partial slot, kind, alone)``,
    alone 1 for the only tile of its sequence. Cut tiles leave one partial per row and part, which the
    merge entries ``(sequence's first packed token, first row, rows, parts, slot, slots from part to part,
    0, 0)`` join, eight rows each. The longest units come first."""
    rows = np.array(counts, dtype=np.int64) * gq
    big_from = BIG_FROM_Q4 if q4 else BIG_FROM
    wide = bool((rows > big_from).any())
    size = np.where(rows > big_from, TILE_ROWS[ROWS256], TILE_ROWS[ROWS32])
    n_tiles = -(-rows // size)
    seq = np.repeat(np.arange(len(rows)), n_tiles)
    if not len(seq):
        return np.zeros((0, UNIT_INTS), np.int32), np.zeros((0, UNIT_INTS), np.int32), 0
    row0 = (np.arange(len(seq)) - np.repeat(np.cumsum(n_tiles) - n_tiles, n_tiles)) * size[seq]
    have = np.minimum(size[seq], rows[seq] - row0)
    kind = np.where(size[seq] == TILE_ROWS[ROWS256], ROWS256, np.where(have <= TILE_ROWS[ROWS16], ROWS16, ROWS32))
    steps = (np.array(starts, dtype=np.int64)[seq] + (row0 + have - 1) // gq) // GT + 1
    parts = (_parts_q4 if q4 else _parts)(steps, kind, have, hkv, wide)
    # one entry a unit
    tile = np.repeat(np.arange(len(seq)), parts)
    part = np.arange(len(tile)) - np.repeat(np.cumsum(parts) - parts, parts)
    slots = np.where(parts > 1, parts * have, 0)
    slot = np.cumsum(slots) - slots
    if q4 and wide:
        rounds, round_us, start = _wide_q4(steps, kind)
        cost = (rounds * round_us / parts + start)[tile]
    else:
        cost = (steps * np.where(kind == ROWS256, STEP_US, GROUP_US) / parts)[tile]  # (only its order counts)
    alone = (n_tiles[seq] == 1).astype(np.int64)
    units = np.stack([seq[tile], row0[tile], have[tile], part, parts[tile], slot[tile], kind[tile], alone[tile]], 1)
    units = units[np.argsort(-cost, kind="stable")]
    # the cut tiles' rows, eight a merge entry
    cut = np.nonzero(parts > 1)[0]
    n_merges = -(-have[cut] // MERGE_ROWS)
    t = np.repeat(cut, n_merges)
    r = (np.arange(len(t)) - np.repeat(np.cumsum(n_merges) - n_merges, n_merges)) * MERGE_ROWS
    first = (np.cumsum(counts) - np.array(counts))[seq]  # the sequence's first packed token
    zero = np.zeros_like(t)
    merges = np.stack([first[t], row0[t] + r, np.minimum(MERGE_ROWS, have[t] - r), parts[t], slot[t] + r, have[t], zero, zero], 1)
    return units.astype(np.int32), merges.astype(np.int32), int(slots.sum())


def _parts(steps: np.ndarray, kind: np.ndarray, rows: np.ndarray, hkv: int, wide: bool) -> np.ndarray:
    """Into how many parts each tile is cut: the cut with the least estimated time among those whose parts take at
    most the longest tile's time divided by 1, 1.5, 2, 3, .. A launch takes as long as its longest unit, or all of them
    over the workgroups that run at once, plus the partials' traffic and second launch."""
    small = kind != ROWS256
    waves, slots = (8, CUS) if wide else (4, 2 * CUS)
    rounds = -(-steps // waves)  # of a small unit: its waves take a group each
    most = np.minimum(MAX_PARTS, np.where(small, np.maximum(1, steps // SMALL_PART), steps))
    us = np.where(small, rounds * (waves * GROUP_US), steps * STEP_US)
    # (far more tiles than slots are not cut)
    cuts = np.array(CUTS if len(steps) * hkv < 16 * slots else CUTS[:1])[:, None]
    parts = np.clip(np.ceil(us * (cuts / us.max())).astype(np.int64), 1, most)
    unit = np.where(small, -(-rounds // parts) * (waves * GROUP_US), us / parts) + UNIT_US
    partials = (np.where(parts > 1, parts, 0) @ rows) * hkv
    time = np.maximum(unit.max(1), (unit * parts).sum(1) * (hkv / slots)) + np.where(partials > 0, MERGE_US + partials * PARTIAL_US, 0.0)
    return parts[time.argmin()]


# The 4-bit pages: rows from which tiles are ROWS256 (all as ROWS256 / as ROWS32): 96 rows over 32000 tokens 46 / 41 us, 8 times
# 128 rows over 4000 47 / 42, 200 rows over 8000 30 / 27; and, in launches of small units (ROWS16, ROWS32), what they take in
# us: a round of four waves alone on a CU, and beside another workgroup there; a unit's start and end; the second launch, and
# each part of its longest row.
BIG_FROM_Q4 = 200
ALONE_Q4, SHARED_Q4, START_Q4 = (1.6, 2.35), (1.5, 2.0), (5.0, 7.0)
MERGE_Q4, MERGE_PART_Q4 = 3.0, 0.1
# Launches with wide tiles, by kind: a round of eight waves or a wide tile's step, and a unit's start and end.
WIDE_STEP_Q4, WIDE_START_Q4 = (2.5, 3.2, 1.9), (7.0, 8.0, 10.0)
WIDE_CUTS_Q4 = (1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 8, 12, 16, 24, 32, 64, 128, 256)


def _parts_q4(steps: np.ndarray, kind: np.ndarray, rows: np.ndarray, hkv: int, wide: bool) -> np.ndarray:
    """:func:`_parts` for 4-bit pages: the least time among the same cuts, by what their units were measured at. Of 20 batches (1 to 64
    sequences of 1 to 50 rows over 500 to 131000 tokens, prompts and chunks) 18 get a cut within 7% of the best, all within 12%."""
    if wide:
        return _parts_q4_wide(steps, kind, rows, hkv)
    slow = (kind == ROWS32).astype(np.int64)
    rounds = -(-steps // 4)
    most = np.minimum(MAX_PARTS, np.maximum(1, steps // SMALL_PART))
    round_us = np.array(ALONE_Q4)[slow]
    us = rounds * round_us
    # (far more tiles than slots are not cut)
    cuts = np.array(CUTS if len(steps) * hkv < 32 * CUS else CUTS[:1])[:, None]
    parts = np.clip(np.ceil(us * (cuts / us.max())).astype(np.int64), 1, most)
    alone = -(-rounds // parts)
    # all of it over the CUs, as far as the units fill them evenly
    k = parts.sum(1) * (hkv / CUS)
    uneven = np.where(k <= 2.1, 1.1 * np.maximum(1.0, np.ceil(k - 0.1) / k), 1.2 + 0.03 * k)
    total = (alone * np.array(SHARED_Q4)[slow] * parts).sum(1) * (hkv / CUS)
    cut_rows = (np.where(parts > 1, parts, 0) @ rows) * hkv
    merges = np.where(cut_rows > 0, MERGE_Q4 + MERGE_PART_Q4 * parts.max(1) + cut_rows * PARTIAL_US, 0.0)
    time = START_Q4[int(slow.max())] + np.maximum((alone * round_us).max(1), total * uneven) + merges
    return parts[time.argmin()]


def _wide_q4(steps: np.ndarray, kind: np.ndarray) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
    """In a launch with wide tiles: each tile's rounds (of eight waves; a wide tile's steps), a round's price, the start's."""
    return np.where(kind == ROWS256, steps, -(-steps // 8)), np.array(WIDE_STEP_Q4)[kind], np.array(WIDE_START_Q4)[kind]


def _parts_q4_wide(steps: np.ndarray, kind: np.ndarray, rows: np.ndarray, hkv: int) -> np.ndarray:
    """The same for launches with wide tiles, one workgroup a CU, the longest units first: where they are up to twice the CUs, the
    shortest follow the units that end first. Of 17 batches (prompts and chunks, alone and beside up to 40 sequences of 1 to
    4 rows) 15 get a cut within 4% of the best, all within 14%; by _parts' prices 12 sequences of 8000 tokens beside a prompt
    take 49 us instead of 33, one of 30000 33 instead of 21."""
    small = kind != ROWS256
    rounds, round_us, start = _wide_q4(steps, kind)
    us = rounds * round_us
    most = np.minimum(MAX_PARTS, np.where(small, np.maximum(1, steps // SMALL_PART), steps))
    longest = int((us + start).argmax())
    cuts = np.array(WIDE_CUTS_Q4 if len(steps) * hkv < 16 * CUS else WIDE_CUTS_Q4[:1])[:, None]
    target = np.maximum(us[longest] / cuts + start[longest] - start, 1.0)
    parts = np.clip(np.ceil(us / target - 1e-9).astype(np.int64), 1, most)
    unit = np.where(small, -(-rounds // parts), rounds / parts) * round_us + start
    n, last = parts.sum(1) * hkv, unit.max(1)
    cut_rows = (np.where(parts > 1, parts, 0) @ rows) * hkv
    merges = np.where(cut_rows > 0, MERGE_US + cut_rows * PARTIAL_US, 0.0)
    time = np.maximum(last, (unit * parts).sum(1) * (hkv / CUS)) + np.where(n > 2 * CUS, unit.min(1), 0.0) + merges
    for c in np.nonzero((n > CUS) & (n <= 2 * CUS))[0]:
        each = np.sort(np.repeat(unit[c], parts[c] * hkv))[::-1]
        time[c] = max(time[c], (each[CUS:] + each[2 * CUS - n[c]:CUS][::-1]).max() + merges[c])
    return parts[time.argmin()]


def _packed(counts: list[int]) -> tuple[np.ndarray, np.ndarray]:
    n = np.array(counts, dtype=np.int64)
    if sum(counts) >= 1 << 24:
        raise ValueError(f"{sum(counts)} tokens in one call; less than 2^24 are possible")
    cu = np.concatenate(([0], np.cumsum(n)))
    return cu.astype(np.int32), np.repeat(np.arange(len(counts), dtype=np.int32), n)


def span_plan(counts: list[int], starts: list[int], pos: torch.Tensor) -> SpanPlan:
    cu, seq_of = _packed(counts)
    first = torch.tensor(starts, dtype=torch.int64).to(pos.device)
    ints = torch.from_numpy(np.concatenate((cu, seq_of))).to(pos.device)
    return SpanPlan(counts, int(cu[-1]), pos, first, ints[:len(cu)], ints[len(cu):])


def chunk_plan(counts: list[int], lengths: list[int], pos: torch.Tensor, gq: int, hkv: int, q4: bool = False) -> ChunkPlan:
    cu, seq_of = _packed(counts)
    units, merges, rows = plan_units(lengths, counts, gq, hkv, q4)
    # one copy to the device; the entries are 32 bytes, so that each of them stays aligned
    ints = torch.from_numpy(np.concatenate((units.ravel(), merges.ravel(), cu, seq_of))).to(pos.device)
    new = torch.tensor(counts, dtype=torch.int64).to(pos.device)
    u, m = units.size, units.size + merges.size
    return ChunkPlan(counts, int(cu[-1]), pos, pos[:len(counts)], ints[m:m + len(cu)], ints[m + len(cu):], new,
                     ints[:u].view(-1, UNIT_INTS), ints[u:m].view(-1, UNIT_INTS),
                     int(_lib.load().nkv_paged_chunks_workspace_bytes(hkv, rows)), bool((units[:, 6] == ROWS256).any()),
                     int(units[:, 6].max(initial=ROWS16)))


def launch(device: torch.device, name: str, *args) -> None:
    """``_lib.call`` on the current stream of ``device`` (a tensor's, so it has an index), whichever device is
    current."""
    index = device.index
    if index == torch._C._cuda_getDevice():  # (current_device() without the check that CUDA is set up, and below)
        rc = getattr(_lib.load(), name)(*args, torch._C._cuda_getCurrentRawStream(index))
        if rc:
            _lib.fail(name, rc)
        return
    with torch.cuda.device(device):
        _lib.call(name, *args, _lib.stream_ptr(device))


def of_cache(plan: SpanPlan, pos: torch.Tensor) -> None:
    if plan.pos is not pos:
        raise ValueError("the plan was made by another cache")


def step_of_cache(plan: SpanPlan, pos: torch.Tensor) -> None:
    """``plan`` must be a step's plan (``plan_chunks``) of the cache: one of ``plan_read`` names cached tokens, which a
    step would overwrite."""
    of_cache(plan, pos)
    if not isinstance(plan, ChunkPlan):
        raise ValueError("the plan was made by plan_read; a step takes one of plan_chunks")


def heads_of(x: torch.Tensor, name: str, tokens: int, heads: int, device: torch.device) -> None:
    """``x`` must be fp16 ``[>= tokens, heads, 128]`` on ``device``."""
    shape = x.shape
    if len(shape) != 3 or shape[0] < tokens or shape[1:] != (heads, D) or x.dtype != torch.float16 or x.device != device:
        raise ValueError(f"{name} must be fp16 [{tokens}, {heads}, {D}] on {device} (more tokens may follow), "
                         f"got {tuple(shape)} {x.dtype} on {x.device}")


def rows_in_place(x: torch.Tensor) -> bool:
    """Whether the kernels can take ``x`` ``[tokens, heads, 128]`` where it is: rows of 128 elements that start
    on 16 bytes."""
    token, head, element = x.stride()
    return element == 1 and token % 8 == 0 and head % 8 == 0 and x.data_ptr() % 16 == 0


def _extent(x: torch.Tensor) -> tuple[int, int]:
    """The bytes from ``x``'s first to behind its last element (no negative strides in torch)."""
    if x.numel() == 0:
        return x.data_ptr(), x.data_ptr()
    last = sum((n - 1) * s for n, s in zip(x.shape, x.stride()))
    return x.data_ptr(), x.data_ptr() + (last + 1) * x.element_size()


def overlap(x: torch.Tensor, y: torch.Tensor) -> bool:
    (a0, a1), (b0, b1) = _extent(x), _extent(y)
    return a0 < b1 and b0 < a1


def distinct_rows(x: torch.Tensor) -> bool:
    """Whether no two elements of ``x`` ``[tokens, heads, 128]`` (unit last stride) share memory: one of the two
    outer dimensions lies within the other's stride."""
    (n, h, d), (st, sh, _) = x.shape, x.stride()
    if x.numel() == 0:
        return True
    inner_heads = (h == 1 or sh >= d) and (n == 1 or st >= (h - 1) * sh + d)
    inner_tokens = (n == 1 or st >= d) and (h == 1 or sh >= (n - 1) * st + d)
    return inner_heads or inner_tokens
