"""Host side of the paged caches' calls over several tokens per sequence: the cut of the attention into
work units, the packing, and what the entry points refuse before any launch (CPU)."""

from __future__ import annotations

import random

import numpy as np
import pytest

from nova_amd import _lib
from nova_amd import chunks as C

OK, INVALID, UNSUPPORTED = _lib.NKV_OK, _lib.NKV_ERR_INVALID, _lib.NKV_ERR_UNSUPPORTED


@pytest.fixture(scope="module")
def lib():
    return _lib.load(require_gpu=False)


def _cases():
    rng = random.Random(5)
    yield [0], [1], 1, 1
    yield [63, 64, 65], [1, 1, 1], 4, 8
    yield [14336], [2048], 4, 8
    yield [100000], [1], 16, 1
    yield [0, 0, 0], [0, 5, 0], 7, 4
    yield [200, 1000, 64], [384, 1, 129], 5, 2
    for _ in range(60):
        n = rng.randint(1, 40)
        yield ([rng.choice([0, rng.randint(0, 9000)]) for _ in range(n)], [rng.choice([0, 1, 4, rng.randint(1, 700)]) for _ in range(n)],
               rng.choice([1, 2, 3, 4, 5, 7, 8, 16]), rng.choice([1, 2, 4, 8]))


@pytest.mark.parametrize("starts,counts,gq,hkv", list(_cases()))
def test_units_cover_each_row_and_part_once(starts, counts, gq, hkv):
    units, merges, slots = C.plan_units(starts, counts, gq, hkv)
    assert units.dtype == merges.dtype == np.int32 and units.shape[1] == merges.shape[1] == C.UNIT_INTS
    tiles = {}
    for seq, row0, rows, part, parts, slot, kind, alone in units.tolist():
        assert 0 <= part < parts <= C.MAX_PARTS and rows <= C.TILE_ROWS[kind] and alone == (rows == counts[seq] * gq)
        tiles.setdefault((seq, row0, rows, parts, slot, kind), []).append(part)
    seen = {}
    for (seq, row0, rows, parts, slot, kind), got in tiles.items():
        assert sorted(got) == list(range(parts))
        seen.setdefault(seq, []).extend(range(row0, row0 + rows))
    for b, n in enumerate(counts):
        assert sorted(seen.get(b, [])) == list(range(n * gq)), b
    # the partials of cut tiles lie apart, within the slots; each of their rows is merged once
    used = []
    for (seq, row0, rows, parts, slot, kind) in tiles:
        if parts > 1:
            used += range(slot, slot + parts * rows)
    assert sorted(used) == list(range(slots))
    first = np.concatenate(([0], np.cumsum(counts)))
    want = {(first[seq], row0 + r, parts, slot + r, rows) for seq, row0, rows, parts, slot, _ in tiles if parts > 1 for r in range(rows)}
    got = [(f, row0 + r, parts, slot + r, stride) for f, row0, rows, parts, slot, stride, _, _ in merges.tolist()
           for r in range(rows)]
    assert len(got) == len(set(got)) and set(got) == want
    assert all(rows <= C.MERGE_ROWS for rows in merges[:, 2])


def test_packing():
    cu, seq_of = C._packed([3, 0, 1, 2])
    assert cu.tolist() == [0, 3, 3, 4, 6] and seq_of.tolist() == [0, 0, 0, 2, 3, 3]
    assert cu.dtype == seq_of.dtype == np.int32
    with pytest.raises(ValueError, match="2\\^24"):
        C._packed([1 << 24])  # (refused before the tokens are listed)


def test_counts_are_checked():
    assert C.check_counts([0, 3], 2) == [0, 3]
    for bad in ([], [1, 1, 1], [1, -1]):
        with pytest.raises(ValueError):
            C.check_counts(bad, 2)


def test_overlap_and_distinct_rows():
    import torch

    x = torch.empty(64, 6, 128, dtype=torch.float16)
    assert C.overlap(x[:10], x[9:]) and not C.overlap(x[:10], x[10:])
    assert C.distinct_rows(x) and C.distinct_rows(x.transpose(0, 1)) and C.distinct_rows(x[:, 2:4])
    assert C.distinct_rows(x[:0]) and C.distinct_rows(x[::3])
    assert not C.distinct_rows(x[:1].expand(5, 6, 128)) and not C.distinct_rows(x[:, :1].expand(64, 6, 128))


# ---- refusals of the C entries (every pointer is a dummy that is never followed: each call fails, or has no tokens)

PTR = 1 << 20


def _append(lib, **kw):
    a = dict(qkv=PTR, dtype=0, rs=48 * 128, tokens=4, pages=PTR, table=PTR, ts=4, np=8, seq_of=PTR, cu=PTR, start=PTR, nseq=2,
             hq=32, hkv=8, d=128, qg=PTR, kg=PTR, eps=1e-6, inv=PTR, q=PTR, q_rs=32 * 128, stream=None)
    a.update(kw)
    return lib.nkv_paged_append_chunks_tok(*a.values())


def _attend(lib, **kw):
    a = dict(q=PTR, q_ts=4096, q_hs=128, tokens=4, pages=PTR, table=PTR, ts=4, np=8, cu=PTR, start=PTR, nseq=2, hq=32, hkv=8,
             d=128, units=PTR, n_units=1, wide=0, merges=None, n_merges=0, out=PTR, o_ts=4096, o_hs=128, lse=None, ws=None, ws_bytes=0,
             stream=None)
    a.update(kw)
    return lib.nkv_paged_attn_chunks_tok(*a.values())


def _read(lib, **kw):
    a = dict(pages=PTR, table=PTR, ts=4, np=8, seq_of=PTR, cu=PTR, start=PTR, tokens=4, nseq=2, hkv=8, d=128, k=PTR, v=PTR, dtype=0,
             stream=None)
    a.update(kw)
    return lib.nkv_paged_read_tok(*a.values())


def _read_t64(lib, **kw):
    a = dict(pages=PTR, table=PTR, ts=4, np=8, rings=PTR, length=PTR, seq_of=PTR, cu=PTR, start=PTR, tokens=4, nseq=2, hkv=8, d=128,
             k=PTR, v=PTR, dtype=0, stream=None)
    a.update(kw)
    return lib.nkv_paged_read_t64(*a.values())


SHARED = [(dict(nseq=0), INVALID), (dict(nseq=1 << 15), INVALID), (dict(hkv=0), INVALID), (dict(ts=0), INVALID), (dict(np=0), INVALID),
          (dict(tokens=-1), INVALID), (dict(tokens=1 << 24), INVALID), (dict(d=64), UNSUPPORTED), (dict(table=None), INVALID),
          (dict(cu=None), INVALID), (dict(start=None), INVALID), (dict(pages=None), INVALID), (dict(pages=PTR + 8), UNSUPPORTED),
          (dict(tokens=0, cu=None), OK)]


@pytest.mark.parametrize("kw,rc", SHARED + [
    (dict(qkv=None), INVALID), (dict(seq_of=None), INVALID), (dict(dtype=3), INVALID), (dict(hq=30), INVALID),
    (dict(hq=136, rs=152 * 128, q_rs=136 * 128), INVALID), (dict(rs=47 * 128), INVALID), (dict(rs=48 * 128 + 4), UNSUPPORTED),
    (dict(q_rs=31 * 128), INVALID), (dict(q=None), INVALID), (dict(qg=None), INVALID), (dict(kg=None), INVALID),
    (dict(q=PTR + 2), UNSUPPORTED), (dict(qkv=PTR + 2), UNSUPPORTED), (dict(kg=PTR + 2), UNSUPPORTED)])
def test_append_refusals(lib, kw, rc):
    assert _append(lib, **kw) == rc
    assert rc == OK or lib.nkv_last_error()


@pytest.mark.parametrize("kw,rc", SHARED + [
    (dict(q=None), INVALID), (dict(units=None), INVALID), (dict(out=None), INVALID), (dict(hq=30), INVALID), (dict(n_units=-1), INVALID),
    (dict(n_units=1 << 20), INVALID), (dict(n_merges=1 << 62, merges=PTR, ws=PTR, ws_bytes=1 << 40), INVALID), (dict(n_merges=1), INVALID), (dict(n_merges=1, merges=PTR), INVALID),
    (dict(q_ts=4), UNSUPPORTED), (dict(q_hs=4), UNSUPPORTED), (dict(o_ts=4), UNSUPPORTED), (dict(o_hs=4), UNSUPPORTED),
    (dict(out=PTR + 2), UNSUPPORTED), (dict(n_units=0), OK)])
def test_attend_refusals(lib, kw, rc):
    assert _attend(lib, **kw) == rc
    assert rc == OK or lib.nkv_last_error()


@pytest.mark.parametrize("call,more", [(_read, []), (_read_t64, [(dict(rings=None), INVALID), (dict(length=None), INVALID)])])
def test_read_refusals(lib, call, more):
    for kw, rc in SHARED + more + [(dict(seq_of=None), INVALID), (dict(dtype=7), INVALID), (dict(k=None), INVALID),
                                   (dict(v=PTR + 4), UNSUPPORTED)]:
        assert call(lib, **kw) == rc, kw


def test_workspace_bytes(lib):
    assert lib.nkv_paged_chunks_workspace_bytes(8, 100) == 8 * 100 * 132 * 4
    assert lib.nkv_paged_chunks_workspace_bytes(8, 0) == 0
