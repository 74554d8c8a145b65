"""Host side of the 4-bit format (CPU): what the entry points refuse before any launch, the layouts of the header."""

from __future__ import annotations

import random

import numpy as np
import pytest
import torch

from nova_amd import _lib
from nova_amd import chunks as C
from nova_amd import gemv as G
from nova_amd import q4
from nova_amd.paged import PAGE_BYTES_Q4

OK, INVALID, UNSUPPORTED = _lib.NKV_OK, _lib.NKV_ERR_INVALID, _lib.NKV_ERR_UNSUPPORTED
PTR = 1 << 20  # never followed: each call fails, or has nothing to do


@pytest.fixture(scope="module")
def lib():
    return _lib.load(require_gpu=False)


def _quantize(lib, **kw):
    a = dict(x=PTR, dtype=0, rows=4, n=64, w4=PTR, stream=None)
    a.update(kw)
    return lib.nkv_quantize_q4(*a.values())


def _dequantize(lib, **kw):
    a = dict(w4=PTR, rows=4, n=64, x=PTR, dtype=0, stream=None)
    a.update(kw)
    return lib.nkv_dequantize_q4(*a.values())


@pytest.mark.parametrize("call", [_quantize, _dequantize])
@pytest.mark.parametrize("kw,rc", [
    (dict(dtype=3), INVALID), (dict(rows=-1), INVALID), (dict(n=0), INVALID), (dict(n=48), INVALID), (dict(n=-32), INVALID),
    (dict(rows=1 << 40), INVALID), (dict(rows=1 << 30, n=128), INVALID), (dict(rows=1 << 39, n=1 << 39), INVALID),
    (dict(x=None), INVALID), (dict(w4=None), INVALID), (dict(x=PTR + 8), UNSUPPORTED), (dict(w4=PTR + 4), UNSUPPORTED), (dict(rows=0, x=None), OK)])
def test_quantizer_refusals(lib, call, kw, rc):
    assert call(lib, **kw) == rc
    assert rc == OK or lib.nkv_last_error()


def _gemv(lib, **kw):
    a = dict(x=PTR, dtype=0, tokens=2, gamma=None, eps=1e-6, w4=PTR, out=64, n_in=64, residual=None, y=PTR, ws=None, ws_bytes=0, stream=None)
    a.update(kw)
    return lib.nkv_gemv_q4(*a.values())


def _swiglu(lib, **kw):
    a = dict(x=PTR, dtype=0, tokens=2, gamma=None, eps=1e-6, w4=PTR, out=64, n_in=64, y=PTR, ws=None, ws_bytes=0, stream=None)
    a.update(kw)
    return lib.nkv_swiglu_gemv_q4(*a.values())


@pytest.mark.parametrize("call", [_gemv, _swiglu])
@pytest.mark.parametrize("kw,rc", [
    (dict(dtype=2), INVALID), (dict(dtype=-1), INVALID), (dict(tokens=-1), INVALID), (dict(tokens=1 << 20), INVALID),
    (dict(out=0), INVALID), (dict(out=1 << 27), INVALID), (dict(n_in=0), INVALID), (dict(n_in=40), INVALID),
    (dict(n_in=(1 << 20) + 32), INVALID), (dict(x=None), INVALID), (dict(w4=None), INVALID),
    (dict(y=None), INVALID), (dict(x=PTR + 2), UNSUPPORTED), (dict(w4=PTR + 8), UNSUPPORTED), (dict(gamma=PTR + 2), UNSUPPORTED),
    (dict(ws=PTR + 8), UNSUPPORTED), (dict(tokens=17, n_in=2592, out=40000, gamma=PTR), INVALID), (dict(tokens=17, dtype=1, n_in=2592, out=40000, ws=PTR, ws_bytes=42 * 4096 + 67), INVALID),
    (dict(tokens=0, x=None), OK)])
def test_product_refusals(lib, call, kw, rc):
    assert call(lib, **kw) == rc
    assert rc == OK or lib.nkv_last_error()


def test_product_workspace(lib):
    """None where one launch makes xn (passes of 4 tokens, 10240 inputs in a power of two of tokens, gates and ups in tiles of
    their own, few workgroups if passes), or where x is taken as it is; else xn in tiles of 16 tokens and blocks of 128 inputs
    (in two parts for a norm of fp16), and a word a token."""
    need = lib.nkv_gemv_q4_workspace_bytes
    assert need(1, 4, 100000, 2560, 1, 0) == need(0, 2, 100000, 2560, 1, 0) == need(1, 2, 100, 5120, 1, 0) == need(0, 1, 160, 10240, 1, 1) == need(1, 3, 16, 32, 0, 1) == 0
    assert need(0, 16, 100, 9728, 0, 0) == need(0, 1, 100, 40000, 0, 1) == need(0, 0, 100, 64, 1, 0) == 0
    assert need(0, 8, 2048, 2560, 1, 0) == need(1, 16, 1024, 2560, 0, 0) == need(1, 64, 256, 64, 1, 1) == 0
    assert need(0, 3, 4112, 128, 1, 0) == 2 * 4096 + 12 and need(0, 8, 2049, 128, 1, 0) == need(1, 9, 1376, 256, 1, 0) - 4 == 2 * 4096 + 32
    assert need(0, 1, 100, 64, 1, 1) == 8192 + 4 and need(1, 1, 100, 64, 1, 1) == 4096 + 4 and need(0, 5, 4100, 160, 1, 0) == 4 * 4096 + 20
    assert need(1, 1, 100, 10272, 0, 0) == 81 * 4096 + 4 and need(0, 17, 100, 64, 0, 0) == 2 * 4096 + 68
    assert need(0, 65, 5000, 128, 1, 0) == 12 * 4096 + 260  # (two passes of 48)


def test_weight_bytes(lib):
    need = lib.nkv_q4_weight_bytes
    assert need(16, 128) == 1152 and need(17, 128) == need(16, 160) == 2304 and need(6144, 2560) == 384 * 20 * 1152
    assert need(0, 128) == need(16, 0) == 0


def _paged_quantize(lib, **kw):
    a = dict(x=PTR, dtype=0, hs=64 * 128, hkv=2, n=64, which=0, pages=PTR, row=PTR, first=0, np=4, stream=None)
    a.update(kw)
    return lib.nkv_paged_quantize_q4(*a.values())


@pytest.mark.parametrize("kw,rc", [
    (dict(dtype=3), INVALID), (dict(hkv=0), INVALID), (dict(n=-1), INVALID), (dict(which=2), INVALID), (dict(first=-1), INVALID),
    (dict(np=0), INVALID), (dict(x=None), INVALID), (dict(pages=None), INVALID), (dict(row=None), INVALID),
    (dict(x=PTR + 8), UNSUPPORTED), (dict(pages=PTR + 8), UNSUPPORTED), (dict(hs=63 * 128), UNSUPPORTED),
    (dict(hs=64 * 128 + 4), UNSUPPORTED), (dict(n=0, x=None), OK)])
def test_paged_quantizer_refusals(lib, kw, rc):
    assert _paged_quantize(lib, **kw) == rc
    assert rc == OK or lib.nkv_last_error()


def _append(lib, **kw):
    a = dict(qkv=PTR, dtype=0, rs=48 * 128, tokens=4, pages=PTR, table=PTR, ts=4, np=8, seq_of=PTR, cu=PTR, start=PTR, nseq=2,
             hq=32, hkv=8, d=128, qg=PTR, kg=PTR, eps=1e-6, inv=PTR, q=PTR, q_rs=32 * 128, stream=None)
    a.update(kw)
    return lib.nkv_paged_append_chunks_q4(*a.values())


def _attend(lib, **kw):
    a = dict(q=PTR, q_ts=4096, q_hs=128, tokens=4, pages=PTR, table=PTR, ts=4, np=8, cu=PTR, start=PTR, nseq=2, hq=32, hkv=8,
             d=128, units=PTR, n_units=1, wide=0, merges=None, n_merges=0, out=PTR, o_ts=4096, o_hs=128, lse=None, ws=None, ws_bytes=0,
             stream=None)
    a.update(kw)
    return lib.nkv_paged_attn_chunks_q4(*a.values())


def _read(lib, **kw):
    a = dict(pages=PTR, table=PTR, ts=4, np=8, seq_of=PTR, cu=PTR, start=PTR, tokens=4, nseq=2, hkv=8, d=128, k=PTR, v=PTR, dtype=0,
             stream=None)
    a.update(kw)
    return lib.nkv_paged_read_q4(*a.values())


SHARED = [(dict(nseq=0), INVALID), (dict(nseq=1 << 15), INVALID), (dict(hkv=0), INVALID), (dict(ts=0), INVALID), (dict(np=0), INVALID),
          (dict(tokens=-1), INVALID), (dict(tokens=1 << 24), INVALID), (dict(d=64), UNSUPPORTED), (dict(table=None), INVALID),
          (dict(cu=None), INVALID), (dict(start=None), INVALID), (dict(pages=None), INVALID), (dict(pages=PTR + 8), UNSUPPORTED),
          (dict(tokens=0, cu=None), OK)]
OWN = {_append: [(dict(qkv=None), INVALID), (dict(dtype=3), INVALID), (dict(hq=30), INVALID), (dict(rs=47 * 128), INVALID),
                 (dict(rs=48 * 128 + 4), UNSUPPORTED), (dict(qg=None), INVALID), (dict(q=PTR + 2), UNSUPPORTED)],
       _attend: [(dict(q=None), INVALID), (dict(units=None), INVALID), (dict(hq=136), INVALID), (dict(n_units=1 << 20), INVALID),
                 (dict(n_merges=1, merges=PTR), INVALID), (dict(q_ts=4), UNSUPPORTED), (dict(out=PTR + 2), UNSUPPORTED),
                 (dict(n_units=0), OK)],
       _read: [(dict(seq_of=None), INVALID), (dict(dtype=7), INVALID), (dict(k=None), INVALID), (dict(v=PTR + 4), UNSUPPORTED)]}


@pytest.mark.parametrize("call", list(OWN))
def test_paged_refusals(lib, call):
    for kw, rc in SHARED + OWN[call]:
        assert call(lib, **kw) == rc, kw
        assert rc == OK or lib.nkv_last_error()


def test_weights_of_the_host_are_refused():
    with pytest.raises(ValueError):
        q4.quantize_q4(torch.zeros(4, 64))
    with pytest.raises(ValueError):
        q4.Q4Weight(torch.zeros(1152, dtype=torch.uint8), (4, 64))
    with pytest.raises(ValueError):
        G.rms_gemv_q4(torch.zeros(64, dtype=torch.float16), torch.zeros(4, 64))
    with pytest.raises(ValueError):
        G.swiglu_gemv_q4(torch.zeros(64, dtype=torch.float16), torch.zeros(4, 64))


def test_scale_places_are_one_each():
    """The header's places of a page's 256 scales, each taken once."""
    k = [64 * r + t for t in range(64) for r in range(4)]
    v = [64 * r + t // 8 * 8 + 2 * (t % 4) + t // 4 % 2 for t in range(64) for r in range(4)]
    assert sorted(k) == sorted(v) == list(range(256))
    assert PAGE_BYTES_Q4 == 2 * (64 * 64 + 512) == 9216


def test_values_are_fp16_numbers():
    """A scale of 8 significant bits (denormal: what fp16 keeps of them) times a code is an fp16 number."""
    m = torch.arange(128, 256, dtype=torch.float64) / 128
    s = (m[:, None] * 2.0 ** torch.arange(-24, 14, dtype=torch.float64)).to(torch.float16)
    s = s[7 * s.double() <= 65504].double()
    for c in range(8):
        assert torch.equal((c * s).to(torch.float16).double(), c * s)


def _batches():
    rng = random.Random(11)
    yield [0], [1], 1, 1
    yield [63, 64, 65], [1, 1, 1], 4, 8
    yield [131000] * 4, [1] * 4, 4, 2
    yield [8192], [51], 4, 8  # 204 rows: one tile of 256
    yield [8192], [50], 4, 8  # 200: seven of 32
    yield [1500, 4097, 700, 0, 6000, 3333], [384, 1, 129, 257, 5, 1], 4, 8
    yield [0, 0], [0, 0], 4, 8
    for _ in range(60):
        n = rng.randint(1, 40)
        yield ([rng.choice([0, rng.randint(0, 9000), rng.randint(0, 200000)]) for _ in range(n)],
               [rng.choice([0, 1, 4, rng.randint(1, 60), rng.randint(1, 700)]) for _ in range(n)], rng.choice([1, 2, 3, 4, 5, 7, 8, 16]),
               rng.choice([1, 2, 4, 8]))


@pytest.mark.parametrize("starts,counts,gq,hkv", list(_batches()))
def test_units_of_the_4_bit_cache(starts, counts, gq, hkv):
    """Each row and part once, the parts' slots apart, their rows merged once; tiles of 256 rows only beyond 200."""
    units, merges, slots = C.plan_units(starts, counts, gq, hkv, q4=True)
    rows_of, used, cut = {}, [], {}
    for seq, row0, rows, part, parts, slot, kind, alone in units.tolist():
        assert 0 <= part < parts <= C.MAX_PARTS and 0 < rows <= C.TILE_ROWS[kind] and alone == (rows == counts[seq] * gq)
        assert (kind == C.ROWS256) == (counts[seq] * gq > C.BIG_FROM_Q4)
        rows_of.setdefault(seq, []).extend((row, part, parts) for row in range(row0, row0 + rows))
        if parts > 1:
            used.extend(range(slot + part * rows, slot + (part + 1) * rows))
            cut[seq, row0] = rows, parts, slot
    for b, n in enumerate(counts):
        got = rows_of.get(b, [])
        assert len(got) == len(set(got)) and {r for r, _, _ in got} == set(range(n * gq))
        of_row = {}
        for row, part, parts in got:
            of_row.setdefault((row, parts), []).append(part)
        assert len(of_row) == n * gq and all(sorted(p) == list(range(parts)) for (_, parts), p in of_row.items())
    assert sorted(used) == list(range(slots))
    first = np.concatenate(([0], np.cumsum(counts)))
    want = {(first[seq], row0 + r, parts, slot + r, rows) for (seq, row0), (rows, parts, slot) in cut.items() for r in range(rows)}
    got = [(f, row0 + r, parts, slot + r, stride) for f, row0, rows, parts, slot, stride, _, _ in merges.tolist() for r in range(rows)]
    assert len(got) == len(set(got)) and set(got) == want
