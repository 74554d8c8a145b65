"""GPU tests of the paged caches' calls over several tokens per sequence (``append_chunks``,
``attend_chunks``, ``read``) against plain computations in 64 bits.

Tolerances, from the roundings of the operators (u = 2^-11, half a step of fp16):

- queries: fp32 sums and one rounding to fp16. The fp32 steps of a norm and a rotation stay below 32 half
  steps of fp32 relative to the row's largest value: ``u |x| + 2^-19 max|row|``.
- codes: with the scale s = max|x| / 127 in fp32 from values that are each 2^-19 max|row| off, x / s moves
  by at most 2 * 127 * 2^-19 < 2^-11 of a code: the code is the rounding of some value that close.
- attention: the codes are exact, each weight times its V scale is rounded to fp16 (u), a score is off by
  d = 130 * 2^-24 * sum|q k| / sqrt(128) (fp32 sums; it moves a weight and the sum of weights), an exponential by
  2^-22, a sum over up to 10000 tokens (no more than 256 additions one after another in a lane or an accumulator,
  two sums, the joins) by 600 * 2^-24 < u / 8, and the output is rounded once:
  ``|err| <= u |out| + (u + u / 4 + 2 d) max|v| + 2^-24``.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from nova_amd import chunks as C
from nova_amd.paged import GT, PAGE_BYTES_TOK, PagedKVInt8Cache, PagedKVInt8TokCache

pytestmark = pytest.mark.gpu

D = 128
U16 = 2.0 ** -11
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def _randn(shape, seed, scale=1.0, dtype=torch.float16):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def _cache(lens, room, hq, hkv, seed, layers=1, cls=PagedKVInt8TokCache, fill=True):
    """A cache whose sequences hold ``lens`` tokens of random keys and values, its pages handed out in a
    scrambled order and every other byte of the pool garbage."""
    need = [-(-(n + r) // GT) for n, r in zip(lens, room)]
    cache = cls(layers, hkv, D, hq, max_seqs=len(lens), num_pages=sum(need) + 5, max_pages_per_seq=max(need) + 2)
    rng = np.random.default_rng(seed)
    cache._free = [int(x) for x in rng.permutation(cache.num_pages)]
    g = torch.Generator(device="cuda").manual_seed(seed)
    for pool in cache.pages:
        pool.copy_(torch.randint(0, 256, pool.shape, generator=g, device="cuda", dtype=torch.uint8))
    for b, n in enumerate(lens):
        for layer in range(layers):
            if n and fill:
                cache.prefill(b, layer, _randn((1, hkv, n, D), seed + 10 * b + layer, 1.0).cuda(),
                              _randn((1, hkv, n, D), seed + 10 * b + layer + 5, 0.7).cuda())
        cache.pool.set_length(b, 0)
        cache.reserve(b, n + room[b])
        cache.pool.set_length(b, n)
        cache.pos[b] = n
    return cache


def _codes(cache, layer, b, n):
    """Sequence b's first n tokens from the bytes of its pages: K, V codes ``[n, H_kv, 128]`` and scales
    ``[n, H_kv]`` as float64 numpy arrays."""
    pages = cache.pages[layer].cpu().numpy()
    row = cache.page_table[b].cpu().numpy()
    out = []
    groups = -(-n // GT)
    rows = pages[row[:groups]] if groups else pages[:0]  # [G, H, PAGE]
    for which in (0, 1):
        c = rows[:, :, which * 8192:(which + 1) * 8192].view(np.int8).reshape(groups, cache.num_kv_heads, GT, D).transpose(0, 2, 1, 3)
        s = np.ascontiguousarray(rows[:, :, 16384 + which * 128:16384 + (which + 1) * 128]).view(np.float16).transpose(0, 2, 1)
        out += [c.reshape(groups * GT, cache.num_kv_heads, D)[:n].astype(np.float64), s.reshape(groups * GT, cache.num_kv_heads)[:n].astype(np.float64)]
    return out


def _values(cache, layer, b, n):
    kc, ks, vc, vs = _codes(cache, layer, b, n)
    with np.errstate(invalid="ignore"):
        return kc * ks[..., None], vc * vs[..., None]


def _attend64(q, k, v, start, gq, u=1.25 * U16):
    """Softmax attention of tokens at positions start .. over k, v ``[n, H_kv, 128]`` in 64 bits: output,
    log-sum-exp and the bound of the module's docstring."""
    m, hq, _ = q.shape
    out, lse, tol = np.zeros((m, hq, D)), np.full((m, hq), -np.inf), np.zeros((m, hq, D))
    for i in range(m):
        n = start + i + 1
        for h in range(hq):
            kk, vv = k[:n, h // gq], v[:n, h // gq]
            s = kk @ q[i, h] / np.sqrt(D)
            top = s.max()
            p = np.exp(s - top)
            out[i, h] = p @ vv / p.sum()
            lse[i, h] = top + np.log(p.sum())
            d = 130 * 2.0 ** -24 * (np.abs(kk) @ np.abs(q[i, h])).max() / np.sqrt(D)
            tol[i, h] = U16 * np.abs(out[i, h]) + (u + 2 * d) * np.abs(vv).max() + 2.0 ** -24
    return out, lse, tol


def _check_attention(cache, layer, plan, q, out, lse, starts):
    gq, at = cache.num_q_heads // cache.num_kv_heads, 0
    q64, out, lse = q.double().cpu().numpy(), out.double().cpu().numpy(), None if lse is None else lse.double().cpu().numpy()
    assert np.isfinite(out[:plan.total]).all()
    for b, n in enumerate(plan.counts):
        if n:
            k, v = _values(cache, layer, b, starts[b] + n)
            want, wl, tol = _attend64(q64[at:at + n], k, v, starts[b], gq)
            err = np.abs(out[at:at + n] - want)
            assert (err <= tol).all(), f"sequence {b}: off by {(err / tol).max():.2f} of the bound"
            if lse is not None:
                # a score is off by d, the sum of weights by u and 2^-13 (the exponentials and fp32 sums)
                assert np.abs(lse[at:at + n] - wl).max() <= 2e-3, f"sequence {b}: lse"
        at += n


# ---------------------------------------------------------------- append


def _rotated(x, gamma, eps, inv_freq, pos):
    x = x.astype(np.float64)
    if gamma is not None:
        x = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps) * gamma
    if inv_freq is not None:
        a = pos[:, None].astype(np.float64) * inv_freq.astype(np.float64)
        c, s = np.cos(a)[:, None], np.sin(a)[:, None]
        x = np.concatenate((x[..., :64] * c - x[..., 64:] * s, x[..., 64:] * c + x[..., :64] * s), -1)
    return x


@pytest.mark.parametrize("lens,counts,hq,hkv,dtype,norm,rope,pad", [
    ([0], [1], 1, 1, torch.float16, True, True, 0),
    ([5, 63, 64, 200], [1, 1, 1, 1], 32, 8, torch.float16, True, True, 0),
    ([5, 63, 0, 200], [130, 1, 0, 65], 32, 8, torch.float16, True, True, 3),
    ([1000, 0], [700, 500], 28, 4, torch.bfloat16, True, True, 0),
    ([17], [129], 16, 1, torch.float32, True, True, 2),
    ([40, 9], [70, 3], 6, 2, torch.float16, True, False, 0),
    ([40, 9], [70, 3], 6, 2, torch.bfloat16, False, True, 0),
])
def test_append_against_64_bits(lens, counts, hq, hkv, dtype, norm, rope, pad):
    print(f"case append lens={lens} counts={counts} hq={hq} hkv={hkv} {dtype}", flush=True)
    cache = _cache(lens, counts, hq, hkv, 3)
    before = cache.pages[0].clone()
    plan = cache.plan_chunks(counts)
    heads = hq + 2 * hkv
    qkv = _randn((plan.total + pad, heads * D), 4, 0.8, dtype).cuda()
    gq = (1 + _randn((D,), 5, 0.2, torch.float32)).to(dtype).cuda() if norm else None
    gk = (1 + _randn((D,), 6, 0.2, torch.float32)).to(dtype).cuda() if norm else None
    inv = (1e6 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)).float().cuda() if rope else None
    q_out = torch.full((plan.total + pad, hq, D), 7.0, dtype=torch.float16, device="cuda")
    q = cache.append_chunks(plan, qkv, 0, gq, gk, 1e-6, inv, q_out=q_out)
    torch.cuda.synchronize()
    assert q is q_out and bool((q_out[plan.total:] == 7.0).all())
    x = qkv.double().cpu().numpy()[:plan.total].reshape(plan.total, heads, D)
    pos = np.concatenate([np.arange(n) + s for s, n in zip(lens, counts)])
    f = lambda t: None if t is None else t.double().cpu().numpy()  # noqa: E731
    want_q = _rotated(x[:, :hq], f(gq), 1e-6, f(inv), pos)
    want_k = _rotated(x[:, hq:hq + hkv], f(gk), 1e-6, f(inv), pos)
    err = np.abs(q.double().cpu().numpy()[:plan.total] - want_q)
    top = np.abs(want_q).max(-1, keepdims=True)
    assert (err <= U16 * np.abs(want_q) + 2.0 ** -19 * top + 2.0 ** -25).all()
    at = 0
    for b, n in enumerate(counts):
        kc, ks, vc, vs = (z[lens[b]:] for z in _codes(cache, 0, b, lens[b] + n))
        for codes, scales, want in ((kc, ks, want_k[at:at + n]), (vc, vs, x[at:at + n, hq + hkv:])):
            s = np.abs(want).max(-1) / 127
            assert (np.abs(scales - s) <= (U16 + 2.0 ** -18) * s + 2.0 ** -25).all()
            assert (np.abs(codes - want / s[..., None]) <= 0.5 + 2.0 ** -10).all()
        at += n
    # nothing but the new tokens' rows changed
    cache2 = _cache(lens, counts, hq, hkv, 3)
    assert torch.equal(cache2.pages[0], before)
    pages, old = cache.pages[0].clone(), before
    for b, n in enumerate(counts):
        for p in range(lens[b], lens[b] + n):
            pg, r = int(cache.page_table[b, p // GT]), p % GT
            for a, w in ((r * D, D), (8192 + r * D, D), (16384 + 2 * r, 2), (16512 + 2 * r, 2)):
                pages[pg, :, a:a + w] = old[pg, :, a:a + w]
    assert torch.equal(pages, old)


def test_append_without_norm_and_rotation_gives_the_quantizers_bits():
    from nova_amd.kvtok import quantize_tok

    for dtype in (torch.float16, torch.bfloat16, torch.float32):
        cache = _cache([30], [100], 4, 2, 8)
        plan = cache.plan_chunks([100])
        qkv = _randn((100, 8 * D), 9, 2.0, dtype)
        qkv[3, 4 * D:5 * D] = 0.0
        qkv[4, 5 * D] = 60000.0
        qkv = qkv.cuda()
        q = cache.append_chunks(plan, qkv, 0)
        assert torch.equal(q.view(100, 4 * D), qkv[:, :4 * D].half())
        for which in (0, 1):
            part = qkv[:, (4 + 2 * which) * D:(6 + 2 * which) * D].view(100, 2, D).transpose(0, 1).contiguous()
            wc, ws = quantize_tok(part)
            got = _codes(cache, 0, 0, 130)
            assert np.array_equal(got[2 * which][30:], wc.transpose(0, 1).cpu().numpy().astype(np.float64))
            assert np.array_equal(got[2 * which + 1][30:], ws.transpose(0, 1).cpu().double().numpy())


def test_append_rotates_at_far_positions():
    """Position 1,000,000 and beyond: an angle in fp32 would be off by up to 0.03."""
    start = 1_000_003
    cache = _cache([0], [1], 2, 1, 12, fill=False)
    cache = PagedKVInt8TokCache(1, 1, D, 2, max_seqs=1, num_pages=-(-(start + 40) // GT), max_pages_per_seq=-(-(start + 40) // GT))
    cache.reserve(0, start + 33)
    cache.pool.set_length(0, start)
    cache.pos[0] = start
    plan = cache.plan_chunks([33])
    qkv = _randn((33, 4 * D), 13).cuda()
    inv = (1e6 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)).float().cuda()
    q = cache.append_chunks(plan, qkv, 0, inv_freq=inv)
    pos = np.arange(33) + start
    x = qkv.double().cpu().numpy().reshape(33, 4, D)
    want = _rotated(x[:, :2], None, 0, inv.double().cpu().numpy(), pos)
    top = np.abs(x[:, :2]).max()
    assert (np.abs(q.double().cpu().numpy() - want) <= U16 * np.abs(want) + 2.0 ** -19 * top).all()


def test_append_in_place_and_strided():
    lens, counts, hq, hkv = [70, 3], [40, 90], 8, 2
    base = _randn((140, 14 * D), 20)
    inv = (1e4 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)).float().cuda()
    gam = [(1 + _randn((D,), 5 + i, 0.2, torch.float32)).half().cuda() for i in range(2)]
    a, b = _cache(lens, counts, hq, hkv, 21), _cache(lens, counts, hq, hkv, 21)
    pa, pb = a.plan_chunks(counts), b.plan_chunks(counts)
    plain = base[:, :12 * D].contiguous().cuda()
    q = a.append_chunks(pa, plain, 0, *gam, 1e-6, inv)
    wide = base.cuda()
    view = wide[:, :12 * D]
    own = view[:, :hq * D].unflatten(1, (hq, D))
    got = b.append_chunks(pb, view, 0, *gam, 1e-6, inv, q_out=own)
    assert got.data_ptr() == wide.data_ptr() and torch.equal(got[:130], q)
    assert torch.equal(wide[:, hq * D:], base[:, hq * D:].cuda()) and torch.equal(wide[130:], base[130:].cuda())
    assert torch.equal(a.pages[0], b.pages[0])
    # rows that cannot be read in place are copied
    odd = torch.empty(140, 12 * D + 1, dtype=torch.float16, device="cuda")[:, 1:]
    odd.copy_(plain)
    c = _cache(lens, counts, hq, hkv, 21)
    assert torch.equal(c.append_chunks(c.plan_chunks(counts), odd, 0, *gam, 1e-6, inv), q)
    assert torch.equal(a.pages[0], c.pages[0])


def test_rows_that_start_between_are_copied():
    """Contiguous tensors whose first element is not on 16 bytes."""
    cache = _held_with_step([70, 10], [30, 5], 8, 2, 22)
    plan = cache.plan_chunks([30, 5])
    qkv = _randn((35, 12 * D), 23).cuda()
    q = cache.append_chunks(plan, qkv, 0)
    pages, out = cache.pages[0].clone(), cache.attend_chunks(plan, q, 0)
    odd = torch.empty(35 * 12 * D + 3, dtype=torch.float16, device="cuda")[3:].view(35, 12 * D)
    odd.copy_(qkv)
    assert odd.is_contiguous() and torch.equal(cache.append_chunks(plan, odd, 0, eps=np.float32(1e-6)), q)
    assert torch.equal(cache.pages[0], pages)
    odd_q = torch.empty(35 * 8 * D + 1, dtype=torch.float16, device="cuda")[1:].view(35, 8, D)
    odd_q.copy_(q)
    assert torch.equal(cache.attend_chunks(plan, odd_q, 0), out)


def test_append_skips_tokens_without_a_page():
    cache = _cache([10, 50], [200, 30], 4, 2, 30)
    plan = cache.plan_chunks([200, 30])
    cache.page_table[0, 1] = -1
    cache.page_table[1].fill_(1 << 20)  # no page of this pool
    before = cache.pages[0].clone()
    qkv = _randn((230, 8 * D), 31).cuda()
    cache.append_chunks(plan, qkv, 0)
    torch.cuda.synchronize()
    changed = (cache.pages[0] != before).flatten(1).any(1).nonzero().flatten().tolist()
    assert sorted(changed) == sorted(int(cache.page_table[0, g]) for g in (0, 2, 3))


# ---------------------------------------------------------------- attention


ATTEND = [
    ([0], [1], 1, 1),
    ([0, 1, 62, 63, 64], [1, 1, 1, 1, 1], 4, 4),
    ([63, 64, 65, 127], [2, 1, 70, 1], 32, 8),
    ([200, 0, 5, 31], [4, 4, 0, 4], 32, 8),
    ([700], [1], 16, 1),
    ([2500, 90], [1, 3], 14, 2),
    ([0], [97], 5, 1),
    ([100, 333], [40, 64], 8, 1),
    ([0, 129], [65, 130], 7, 7),
    ([4000], [9], 12, 4),
    # 64 rows of a sequence and fewer are tiles of 32, more are tiles of 256
    ([900], [64], 1, 1),
    ([900, 30], [65, 64], 1, 1),
    ([500], [255], 1, 1),
    ([500], [257], 1, 1),
    ([5000, 700, 60], [40, 2, 17], 16, 2),
    ([9000], [33], 2, 1),
]


@pytest.mark.parametrize("lens,counts,hq,hkv", ATTEND)
def test_attend_against_64_bits(lens, counts, hq, hkv):
    print(f"case attend lens={lens} counts={counts} hq={hq} hkv={hkv}", flush=True)
    total = [a + n for a, n in zip(lens, counts)]
    cache = _cache(total, [0] * len(lens), hq, hkv, 40)
    for b, n in enumerate(lens):
        cache.pool.set_length(b, n)
        cache.pos[b] = n
    plan = cache.plan_chunks(counts)
    q = _randn((plan.total + 2, hq, D), 41, 1.5).cuda()
    out = torch.full((plan.total + 2, hq, D), 9.0, dtype=torch.float16, device="cuda")
    lse = torch.full((plan.total + 2, hq), 9.0, device="cuda")
    got = cache.attend_chunks(plan, q, 0, out=out, lse=lse)
    torch.cuda.synchronize()
    assert got is out and bool((out[plan.total:] == 9.0).all()) and bool((lse[plan.total:] == 9.0).all())
    _check_attention(cache, 0, plan, q, out, lse, lens)
    assert torch.equal(cache.attend_chunks(plan, q, 0), out[:plan.total])


def _held_with_step(lens, counts, hq, hkv, seed):
    cache = _cache([a + n for a, n in zip(lens, counts)], [0] * len(lens), hq, hkv, seed)
    for b, n in enumerate(lens):
        cache.pool.set_length(b, n)
        cache.pos[b] = n
    return cache


def test_attend_reads_any_strides_and_writes_any():
    lens, counts, hq, hkv = [70, 10], [30, 5], 8, 2
    cache = _held_with_step(lens, counts, hq, hkv, 42)
    plan = cache.plan_chunks(counts)
    q = _randn((35, hq, D), 43).cuda()
    want = cache.attend_chunks(plan, q, 0)
    by_head = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(cache.attend_chunks(plan, by_head, 0), want)
    room = torch.empty(35, hq + 3, D + 8, dtype=torch.float16, device="cuda")
    wide = room[:, 1:hq + 1, :D]
    wide.copy_(q)
    assert torch.equal(cache.attend_chunks(plan, wide, 0), want)
    odd = torch.empty(35, hq, D + 1, dtype=torch.float16, device="cuda")[..., 1:]
    odd.copy_(q)
    assert torch.equal(cache.attend_chunks(plan, odd, 0), want)
    out = torch.zeros(hq, 35, D, dtype=torch.float16, device="cuda").transpose(0, 1)
    cache.attend_chunks(plan, q, 0, out=out)
    assert torch.equal(out, want)


def test_masked_places_may_hold_anything():
    """Infinite and NaN scales behind the sequence's end, and in tokens that a query comes before, change
    nothing for it; the queries that do attend such a token give NaN."""
    lens, counts, hq, hkv = [60, 100], [70, 20], 8, 2
    cache = _held_with_step(lens, counts, hq, hkv, 44)
    plan = cache.plan_chunks(counts)
    q = _randn((90, hq, D), 45).cuda()
    want = cache.attend_chunks(plan, q, 0).clone()
    for bad in (float("inf"), float("nan"), -float("inf")):
        cache2 = _held_with_step(lens, counts, hq, hkv, 44)
        halves = cache2.pages[0].view(torch.float16)
        last = int(cache2.page_table[0, 2])   # tokens 128 .. 191, the sequence ends at 129
        for which in (0, 1):
            halves[last, :, 8192 + 64 * which + 2:8192 + 64 * which + 64] = bad
        mid = int(cache2.page_table[1, 1])    # tokens 64 .. 127: position 110 is the chunk's eleventh token
        halves[mid, 0, 8192 + 64 + 110 - 64] = bad
        got = cache2.attend_chunks(cache2.plan_chunks(counts), q, 0)
        assert torch.equal(got[:70], want[:70])
        assert torch.equal(got[70:80], want[70:80]) and torch.equal(got[:, 4:], want[:, 4:])
        assert bool(got[80:, :4].isnan().all())


def test_groups_without_a_page_take_no_part():
    lens, counts, hq, hkv = [300, 40], [5, 3], 4, 2
    cache = _held_with_step(lens, counts, hq, hkv, 46)
    plan = cache.plan_chunks(counts)
    q = _randn((8, hq, D), 47).cuda()
    k, v = _values(cache, 0, 0, 305)
    cache.page_table[0, 2] = -1
    cache.page_table[1].fill_(-1)
    lse = torch.empty(8, hq, device="cuda")
    out = cache.attend_chunks(plan, q, 0, lse=lse).double().cpu().numpy()
    keep = np.r_[0:128, 192:305]
    for i in range(5):
        n = int((keep < 301 + i).sum())
        want, _, tol = _attend64(q[i:i + 1].double().cpu().numpy(), k[keep[:n]], v[keep[:n]], n - 1, 2)
        assert (np.abs(out[i] - want[0]) <= tol[0]).all()
    assert (out[5:] == 0).all() and bool((lse[5:] == -float("inf")).all())


@pytest.mark.parametrize("counts", [[3, 2], [40, 70]])
def test_masked_places_of_few_rows_and_of_many(counts):
    lens, hq, hkv = [60, 150], 4, 1
    cache = _held_with_step(lens, counts, hq, hkv, 144)
    plan = cache.plan_chunks(counts)
    q = _randn((plan.total, hq, D), 145).cuda()
    want = cache.attend_chunks(plan, q, 0).clone()
    halves = cache.pages[0].view(torch.float16)
    for b, n in enumerate(counts):  # everything behind each sequence's last token
        end = lens[b] + n
        page = int(cache.page_table[b, (end - 1) // GT])
        for bad in (float("inf"), float("nan"), 60000.0):
            for which in (0, 1):
                halves[page, :, 8192 + 64 * which + (end - 1) % GT + 1:8192 + 64 * which + 64] = bad
            assert torch.equal(cache.attend_chunks(plan, q, 0), want)


@pytest.mark.parametrize("lens,counts,hq,hkv", [([0, 130], [1, 2], 4, 2), ([500], [9], 4, 1), ([0, 200], [90, 40], 4, 2), ([1500], [70], 2, 1)])
@pytest.mark.parametrize("scales", [(2.0 ** -24, 2.0 ** -20), (2.0 ** -17, 2.0 ** -16), (2.0 ** -24, 500.0), (500.0, 2.0 ** -22)])
def test_values_of_any_size(lens, counts, hq, hkv, scales):
    """Values so small that their scales are fp16 denormals, and sequences whose values grow or shrink by many
    powers of two from the first to the last token, lose nothing that the bound does not allow."""
    cache = _held_with_step(lens, counts, hq, hkv, 146)
    halves = cache.pages[0].view(torch.float16)
    first, last = (np.log2(x) for x in scales)
    for b, n in enumerate(counts):
        end = lens[b] + n
        s = torch.from_numpy(2.0 ** (first + (last - first) * np.arange(end) / max(1, end - 1))).half().cuda()
        for g in range(-(-end // GT)):
            part = s[g * GT:(g + 1) * GT]
            halves[int(cache.page_table[b, g]), :, 8192 + 64:8192 + 64 + len(part)] = part
    plan = cache.plan_chunks(counts)
    q = _randn((plan.total, hq, D), 147, 1.5).cuda()
    lse = torch.empty(plan.total, hq, device="cuda")
    _check_attention(cache, 0, plan, q, cache.attend_chunks(plan, q, 0, lse=lse), lse, lens)


@pytest.mark.parametrize("counts", [[3, 4], [40, 30]])
def test_a_query_that_is_not_finite_spoils_its_own_row(counts):
    lens, hq, hkv = [300, 90], 4, 1
    cache = _held_with_step(lens, counts, hq, hkv, 154)
    plan = cache.plan_chunks(counts)
    q = _randn((plan.total, hq, D), 155).cuda()
    want = cache.attend_chunks(plan, q, 0)
    bad = q.clone()
    bad[1, 2, 7], bad[plan.total - 1, 0, 100], bad[0, 3, 5] = float("nan"), float("inf"), -float("inf")
    got = cache.attend_chunks(plan, bad, 0)
    rows = torch.zeros(plan.total, hq, dtype=torch.bool, device="cuda")
    rows[1, 2] = rows[plan.total - 1, 0] = rows[0, 3] = True
    assert torch.equal(got[~rows], want[~rows]) and bool(got[rows].isnan().all())


def test_scores_that_grow_by_much():
    """Keys whose scores rise by hundreds from group to group: what was summed before vanishes, and the
    last tokens hold all of the weight."""
    for counts in ([2, 1], [70, 30]):
        lens, hq, hkv = [700, 300], 4, 1
        cache = _held_with_step(lens, counts, hq, hkv, 148)
        halves = cache.pages[0].view(torch.float16)
        for b in range(2):
            for g in range(-(-(lens[b] + counts[b]) // GT)):
                halves[int(cache.page_table[b, g]), :, 8192:8192 + 64] = 2.0 ** (g - 6)
        plan = cache.plan_chunks(counts)
        q = _randn((plan.total, hq, D), 149, 1.0).cuda()
        out = cache.attend_chunks(plan, q, 0)
        _check_attention(cache, 0, plan, q, out, None, lens)


def test_many_rows_over_missing_pages():
    lens, counts, hq, hkv = [700, 130], [40, 70], 8, 2
    cache = _held_with_step(lens, counts, hq, hkv, 150)
    plan = cache.plan_chunks(counts)
    assert plan.wide
    q = _randn((110, hq, D), 151).cuda()
    k, v = _values(cache, 0, 0, 740)
    cache.page_table[0, 0] = -1
    cache.page_table[0, 4:6] = 1 << 20
    cache.page_table[1].fill_(-1)
    lse = torch.empty(110, hq, device="cuda")
    out = cache.attend_chunks(plan, q, 0, lse=lse).double().cpu().numpy()
    keep = np.r_[64:256, 384:740]
    for i in range(40):
        n = int((keep < 701 + i).sum())
        want, _, tol = _attend64(q[i:i + 1].double().cpu().numpy(), k[keep[:n]], v[keep[:n]], n - 1, 4)
        assert (np.abs(out[i] - want[0]) <= tol[0]).all()
    assert (out[40:] == 0).all() and bool((lse[40:] == -float("inf")).all())


@pytest.mark.parametrize("counts", [[3, 1], [80, 40]])
def test_a_plan_outlives_its_lengths(counts):
    """A plan made at one length serves others, shorter (some parts have nothing to do) and longer."""
    hq, hkv = 4, 1
    made = [2500, 900]
    cache = _held_with_step(made, counts, hq, hkv, 152)
    plan = cache.plan_chunks(counts)
    assert plan.ws_bytes > 0
    q = _randn((plan.total, hq, D), 153, 1.5).cuda()
    for lens in ([0, 0], [1, 700], [63, 65], [2499, 130]):
        cache.pos[:2] = torch.tensor(lens)
        lse = torch.empty(plan.total, hq, device="cuda")
        _check_attention(cache, 0, plan, q, cache.attend_chunks(plan, q, 0, lse=lse), lse, lens)
    late = _held_with_step(made, counts, hq, hkv, 152)
    late.pos[:2] = torch.tensor([3, 70])
    for b, n in enumerate((3, 70)):
        late.pool.set_length(b, n)
    early = late.plan_chunks(counts)
    late.pos[:2] = torch.tensor(made)
    _check_attention(late, 0, early, q, late.attend_chunks(early, q, 0), None, made)


def test_one_token_each_agrees_with_the_decode_step():
    lens, hq, hkv = [70, 1000, 64, 4100, 1, 63], 32, 8
    a, b = (_cache(lens, [1] * 6, hq, hkv, 50) for _ in range(2))
    a.plan()
    q, k, v = (_randn((6, h, 1, D), 51 + i).cuda() for i, h in enumerate((hq, hkv, hkv)))
    want = a.decode_step(k, v, q, 0)
    plan = b.plan_chunks([1] * 6)
    qkv = torch.cat([x.view(6, -1) for x in (q, k, v)], 1)
    got = b.attend_chunks(plan, b.append_chunks(plan, qkv, 0), 0)
    assert torch.equal(a.pages[0], b.pages[0])
    _check_attention(b, 0, plan, q[:, :, 0], got, None, lens)
    # the decode step rounds keys and values to fp16 (3 u max|v| with its output), the chunk its weights
    err = (got.float() - want[:, :, 0].float()).abs().max()
    assert float(err) <= 4 * U16 * 3.5


def test_refusals():
    cache = _cache([10, 20], [100, 100], 8, 2, 60)
    with pytest.raises(ValueError):
        cache.plan_chunks([1, 1, 1])
    with pytest.raises(ValueError):
        cache.plan_chunks([1, -1])
    owned = [list(o) for o in cache._owned]
    with pytest.raises(RuntimeError, match="exhausted"):
        cache.plan_chunks([400, 900])
    assert owned == [list(o) for o in cache._owned]
    cache._free = list(range(cache.num_pages, cache.num_pages + 100))
    with pytest.raises(ValueError, match="max_pages_per_seq"):
        cache.plan_chunks([1, 400])
    cache._free = []
    plan = cache.plan_chunks([30, 40])
    qkv = _randn((70, 12 * D), 61).cuda()
    good = dict(q_gamma=torch.ones(D, dtype=torch.float16, device="cuda"), k_gamma=torch.ones(D, dtype=torch.float16, device="cuda"))
    for kw in (dict(qkv=qkv[:69]), dict(qkv=qkv[:, :-128]), dict(qkv=qkv.double()), dict(qkv=qkv.cpu()),
               dict(q_gamma=None), dict(k_gamma=good["k_gamma"].float()), dict(k_gamma=good["k_gamma"][:64]),
               dict(inv_freq=torch.ones(64, dtype=torch.float16, device="cuda")), dict(inv_freq=torch.ones(63, device="cuda")),
               dict(q_out=torch.empty(70, 8, D, device="cuda")), dict(q_out=torch.empty(69, 8, D, dtype=torch.float16, device="cuda")),
               dict(q_out=qkv[:, D:9 * D].unflatten(1, (8, D))),
               dict(q_out=torch.empty(1, 8, D, dtype=torch.float16, device="cuda").expand(70, 8, D))):
        with pytest.raises(ValueError):
            cache.append_chunks(**{**dict(plan=plan, qkv=qkv, layer=0, **good), **kw})
    q = _randn((70, 8, D), 62).cuda()
    for kw in (dict(query=q[:69]), dict(query=q[:, :7]), dict(query=q.float()), dict(query=q.cpu()), dict(out=q), dict(out=q[:69]),
               dict(out=q.float()), dict(out=torch.empty(70, 8, D + 1, dtype=torch.float16, device="cuda")[..., :D]),
               dict(out=torch.empty(1, 8, D, dtype=torch.float16, device="cuda").expand(70, 8, D)),
               dict(lse=torch.empty(70, 8, dtype=torch.float16, device="cuda")), dict(lse=torch.empty(70, 7, device="cuda"))):
        with pytest.raises(ValueError):
            cache.attend_chunks(**{**dict(plan=plan, query=q, layer=0), **kw})
    for accepted in ([31, 0], [1], [-1, 0]):
        with pytest.raises(ValueError):
            cache.advance_chunks(plan, accepted)
    with pytest.raises(RuntimeError, match="reserved"):
        cache.note_chunks(plan, 50)
    with pytest.raises(ValueError):
        cache.plan_read([11, 1])
    with pytest.raises(ValueError):
        cache.plan_read([1, 1], [10, 0])
    with pytest.raises(ValueError):
        cache.plan_read([1, 1], [0])
    span = cache.plan_read([5, 6])
    with pytest.raises(ValueError):
        cache.read(span, 0, torch.float64)
    k = torch.empty(11, 2, D, dtype=torch.float16, device="cuda")
    for out in ((k, k), (k, k[:10]), (k, k.float()), (k, torch.empty(11, 2, 2 * D, dtype=torch.float16, device="cuda")[..., ::2])):
        with pytest.raises(ValueError):
            cache.read(span, 0, out=out)


def test_plans_of_other_caches_are_refused():
    a, b = _cache([10, 20], [100, 100], 8, 2, 64), _cache([10, 20], [100, 100], 8, 2, 64)
    small = _cache([40], [10], 8, 2, 65)
    plan, span = a.plan_chunks([3, 4]), a.plan_read([5, 6])
    qkv, q = _randn((7, 12 * D), 66).cuda(), _randn((7, 8, D), 67).cuda()
    for call in (lambda: b.append_chunks(plan, qkv, 0), lambda: b.attend_chunks(plan, q, 0), lambda: b.read(plan, 0),
                 lambda: b.advance_chunks(plan), lambda: small.read(span, 0), lambda: b.read(span, 0)):
        with pytest.raises(ValueError, match="another cache"):
            call()
    with pytest.raises(ValueError, match="steps"):
        a.note_chunks(plan, -1)


def test_steps_of_no_tokens():
    cache = _cache([10, 20], [64, 64], 8, 2, 63)
    plan = cache.plan_chunks([0, 0])
    before = cache.pages[0].clone()
    q = cache.append_chunks(plan, torch.empty(0, 12 * D, dtype=torch.float16, device="cuda"), 0)
    out = cache.attend_chunks(plan, q, 0)
    k, v = cache.read(plan, 0)
    cache.advance_chunks(plan)
    assert q.shape == out.shape == (0, 8, D) and k.shape == v.shape == (0, 2, D)
    assert torch.equal(cache.pages[0], before) and cache.pos.tolist() == [10, 20]


# ---------------------------------------------------------------- read


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens,counts,starts,hkv", [
    ([1], None, None, 1), ([64, 130, 63], None, None, 8), ([300, 5, 200], [100, 0, 150], [150, 5, 50], 2), ([700], [1], [699], 3)])
def test_read_tok(lens, counts, starts, hkv, dtype):
    cache = _cache(lens, [3] * len(lens), hkv, hkv, 70)
    plan = cache.plan_read(counts, starts)
    counts = lens if counts is None else counts
    starts = [0] * len(lens) if starts is None else starts
    room = tuple(torch.full((plan.total + 2, hkv, D), 5.0, dtype=dtype, device="cuda") for _ in range(2))
    k, v = cache.read(plan, 0, dtype, out=room)
    assert bool((k[plan.total:] == 5.0).all()) and bool((v[plan.total:] == 5.0).all())
    at = 0
    for b, (s, n) in enumerate(zip(starts, counts)):
        kc, ks, vc, vs = _codes(cache, 0, b, s + n)
        for got, c, sc in ((k, kc, ks), (v, vc, vs)):
            want = torch.from_numpy(c[s:] * sc[s:, :, None]).float().to(dtype)  # (exact in fp32)
            assert torch.equal(got[at:at + n].cpu(), want)
        at += n
    k2, v2 = cache.read(plan, 0, dtype)
    assert torch.equal(k2, k[:plan.total]) and torch.equal(v2, v[:plan.total])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens,counts,starts", [([1], None, None), ([64, 130, 63], None, None), ([300, 64, 200], [100, 3, 110], [200, 61, 50])])
def test_read_t64(lens, counts, starts, dtype):
    hkv = 2
    cache = _cache(lens, [3] * len(lens), hkv, hkv, 80, cls=PagedKVInt8Cache)
    plan = cache.plan_read(counts, starts)
    counts = lens if counts is None else counts
    starts = [0] * len(lens) if starts is None else starts
    k, v = cache.read(plan, 0, dtype)
    pages, at = cache.pages[0].cpu(), 0
    for b, (s, n) in enumerate(zip(starts, counts)):
        for got, which in ((k, 0), (v, 1)):
            for t in range(s, s + n):
                if t < lens[b] // GT * GT:
                    pg = pages[int(cache.page_table[b, t // GT])]
                    c = pg[:, which * 8192 + (t % GT) * D:][:, :D].float()
                    r = pg[:, 16384 + which * 512:16384 + (which + 1) * 512].contiguous().view(torch.float16).float()
                    want = (c.double() * r[:, :D].double() + r[:, D:].double()).float().to(dtype)
                else:
                    want = cache.rings[0][b, :, which, t % GT].cpu().float().to(dtype)
                assert torch.equal(got[at + t - s].cpu(), want), (b, t, which)
        at += n


def test_read_of_missing_pages_is_zero():
    cache = _cache([200], [3], 2, 2, 85)
    plan = cache.plan_read()
    k0, v0 = cache.read(plan, 0)
    cache.page_table[0, 1] = -1
    k, v = cache.read(plan, 0)
    assert bool((k[64:128] == 0).all()) and bool((v[64:128] == 0).all())
    for new, old in ((k, k0), (v, v0)):
        assert torch.equal(new[:64], old[:64]) and torch.equal(new[128:], old[128:])


# ---------------------------------------------------------------- together


def _layer_inputs(total, hq, hkv, layers, seed):
    return [_randn((total, (hq + 2 * hkv) * D), seed + i, 0.8).cuda() for i in range(layers)]


def test_a_batch_served_in_mixed_steps():
    """Two layers, three sequences: prompts in chunks beside decode tokens, drafted tokens of which some are
    kept, then the one-token decode step, all over the same pages; every output against 64 bits."""
    hq, hkv, layers = 8, 2, 2
    cache = _cache([0, 0, 0], [400, 300, 200], hq, hkv, 90, layers=layers, fill=False)
    inv = (1e4 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)).float().cuda()
    gam = [(1 + _randn((D,), 91 + i, 0.2, torch.float32)).half().cuda() for i in range(2)]
    lens = [0, 0, 0]
    steps = [([100, 64, 1], None), ([130, 1, 60], None), ([1, 90, 1], None), ([4, 4, 4], [1, 4, 2]), ([1, 0, 5], None)]
    for i, (counts, accepted) in enumerate(steps):
        plan = cache.plan_chunks(counts)
        for layer, qkv in enumerate(_layer_inputs(plan.total, hq, hkv, layers, 100 + 10 * i)):
            q = cache.append_chunks(plan, qkv, layer, *gam, 1e-6, inv)
            out = cache.attend_chunks(plan, q, layer)
            _check_attention(cache, layer, plan, q, out, None, lens)
            k, v = cache.read(plan, layer)
            at = 0
            for b, n in enumerate(counts):
                wk, wv = _values(cache, layer, b, lens[b] + n)
                assert np.array_equal(k[at:at + n].cpu().numpy(), wk[lens[b]:].astype(np.float16))
                assert np.array_equal(v[at:at + n].cpu().numpy(), wv[lens[b]:].astype(np.float16))
                at += n
        cache.advance_chunks(plan, accepted)
        lens = [a + n for a, n in zip(lens, accepted or counts)]
        assert cache.pos.tolist() == lens == cache._len
    cache.plan()
    q, k, v = (_randn((3, h, 1, D), 200 + h).cuda() for h in (hq, hkv, hkv))
    out = cache.decode_step(k, v, q, 1)
    for b in range(3):
        kk, vv = _values(cache, 1, b, lens[b] + 1)
        # (the decode step rounds keys and values to fp16, too)
        want, _, tol = _attend64(q[b, :, 0][None].double().cpu().numpy(), kk, vv, lens[b], hq // hkv, 3 * U16)
        assert (np.abs(out[b, :, 0].double().cpu().numpy() - want[0]) <= tol[0]).all()


def test_a_captured_step_follows_the_sequences():
    """One capture of append, attend, read and the advance, replayed while the sequences grow across pages,
    against eager calls; the eager work between the replays shares the plan."""
    hq, hkv, counts, lens, steps = 8, 2, [4, 1, 7], [50, 700, 0], 12
    a, b = (_cache(lens, [n * (steps + 1) for n in counts], hq, hkv, 110) for _ in range(2))
    pa, pb = a.plan_chunks(counts), b.plan_chunks(counts)
    inv = (1e4 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)).float().cuda()
    x = torch.empty(pa.total, 12 * D, dtype=torch.float16, device="cuda")
    x.copy_(_randn(x.shape, 111))

    def step(c, p):
        q = c.append_chunks(p, x, 0, inv_freq=inv)
        return q, c.attend_chunks(p, q, 0), *c.read(p, 0)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            got = step(b, pb)
            b.pos[:3].add_(pb.new)
    torch.cuda.current_stream().wait_stream(side)
    for i in range(steps):
        x.copy_(_randn(x.shape, 112 + i))
        graph.replay()
        want = step(a, pa)
        a.advance_chunks(pa)
        b.note_chunks(pb)
        torch.cuda.synchronize()
        for w, g in zip(want, got):
            assert torch.equal(w, g), i
        assert torch.equal(a.pages[0], b.pages[0]) and torch.equal(a.pos, b.pos) and a._len == b._len


def test_a_captured_step_of_many_rows_follows_the_sequences():
    """As above, with rows of every kind, and two graphs of one plan replayed side by side on two streams."""
    hq, hkv, counts, lens, steps = 8, 2, [40, 1, 9, 0], [0, 1000, 70, 5], 4
    a, b = (_cache(lens, [n * (steps + 1) for n in counts], hq, hkv, 160) for _ in range(2))
    pa, pb = a.plan_chunks(counts), b.plan_chunks(counts)
    assert pa.wide and pa.ws_bytes > 0
    x = torch.empty(pa.total, 12 * D, dtype=torch.float16, device="cuda")
    q2 = torch.empty(pa.total, hq, D, dtype=torch.float16, device="cuda")

    def step(c, p):
        q = c.append_chunks(p, x, 0)
        return q, c.attend_chunks(p, q, 0)

    graphs, outs = [], []
    for f in (lambda: step(b, pb), lambda: (q2, b.attend_chunks(pb, q2, 0))):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(f())
        graphs.append(g)
    side = torch.cuda.Stream()
    for i in range(steps):
        x.copy_(_randn(x.shape, 161 + i))
        q2.copy_(_randn(q2.shape, 171 + i))
        want = step(a, pa)
        graphs[0].replay()
        torch.cuda.synchronize()
        other = a.attend_chunks(pa, q2, 0)
        side.wait_stream(torch.cuda.current_stream())
        for _ in range(3):
            graphs[0].replay()
            with torch.cuda.stream(side):
                graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(want[0], outs[0][0]) and torch.equal(want[1], outs[0][1]) and torch.equal(other, outs[1][1])
        for c, p in ((a, pa), (b, pb)):
            c.advance_chunks(p)


def test_two_streams_share_a_plan():
    lens, counts, hq, hkv = [3000, 500, 1200], [3, 9, 1], 32, 8
    cache = _held_with_step(lens, counts, hq, hkv, 120)
    plan = cache.plan_chunks(counts)
    assert plan.ws_bytes > 0
    qs = [_randn((13, hq, D), 121 + i).cuda() for i in range(4)]
    want = [cache.attend_chunks(plan, q, 0).clone() for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[] for _ in qs]
    for _ in range(5):
        for i, q in enumerate(qs):
            with torch.cuda.stream(streams[i % 2]):
                got[i].append(cache.attend_chunks(plan, q, 0))
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        assert all(torch.equal(w, o) for o in outs)


def test_pages_beyond_four_gigabytes():
    """A pool of more than 2^32 bytes: tokens in its last pages."""
    hq, hkv, n = 2, 1, 100
    pages = (1 << 32) // PAGE_BYTES_TOK + 64
    cache = PagedKVInt8TokCache(1, hkv, D, hq, max_seqs=1, num_pages=pages, max_pages_per_seq=4)
    cache._free = [5, pages - 2, pages - 1]
    plan = cache.plan_chunks([n])
    assert cache._owned[0] == [pages - 1, pages - 2]
    qkv = _randn((n, 4 * D), 131).cuda()
    q = cache.append_chunks(plan, qkv, 0)
    out = cache.attend_chunks(plan, q, 0)
    _check_attention(cache, 0, plan, q, out, None, [0])
    k, _ = cache.read(plan, 0)
    assert np.array_equal(k.cpu().numpy(), _values(cache, 0, 0, n)[0].astype(np.float16))
    assert int(cache.pages[0][:pages - 2].count_nonzero()) == 0


# ---------------------------------------------------------------- tokens that a row does not attend


@pytest.mark.parametrize("small", [2.0 ** -9, 2.0 ** -12, 2.0 ** -20])
@pytest.mark.parametrize("lens,counts,hq,hkv", [
    ([10], [4], 4, 1),      # 16 rows
    ([30], [8], 8, 2),      # 16 and 16 rows of two heads
    ([70], [9], 3, 1),      # 27 rows
    ([128], [16], 4, 1),    # two tiles of 32 rows
    ([300, 7], [6, 20], 4, 1),
    ([20], [40], 4, 1),     # a wide tile in one group
    ([0], [130], 2, 1),     # a wide tile that begins with masked places, and one of 4 rows
    ([500, 33], [70, 5], 2, 1),
])
def test_a_later_tokens_scale_changes_nothing_before_it(lens, counts, hq, hkv, small):
    """V scales that are large or not finite, in tokens of the same step: the rows before such a token give the bits
    that they give beside an ordinary one, within the bound of the values that they attend."""
    cache = _held_with_step(lens, counts, hq, hkv, 180)
    halves = cache.pages[0].view(torch.float16)
    for b in range(len(lens)):
        for g in range(-(-(lens[b] + counts[b]) // GT)):
            halves[int(cache.page_table[b, g]), :, 8192 + 64:] = small
    plan = cache.plan_chunks(counts)
    q = _randn((plan.total, hq, D), 181, 1.5).cuda()
    want = cache.attend_chunks(plan, q, 0).clone()
    q64, gq, at = q.double().cpu().numpy(), hq // hkv, 0
    for b, n in enumerate(counts):
        for j in sorted({1, n * 3 // 4, n - 1}):
            k, v = _values(cache, 0, b, lens[b] + j)
            exact, _, tol = _attend64(q64[at:at + j], k, v, lens[b], gq)
            page, place = int(cache.page_table[b, (lens[b] + j) // GT]), (lens[b] + j) % GT
            for bad in (float("inf"), float("nan"), -float("inf"), 60000.0, 500.0, -500.0):
                print(f"case sequence {b} token {j} scale {bad}", flush=True)
                halves[page, :, 8192 + 64 + place] = bad
                got = cache.attend_chunks(plan, q, 0)
                err = np.abs(got[at:at + j].double().cpu().numpy() - exact)
                assert (err <= tol).all(), f"off by {(err / tol).max():.2f} of the bound"
                others = torch.ones(plan.total, dtype=torch.bool, device="cuda")
                others[at + j:at + n] = False
                assert torch.equal(got[others], want[others])
                if abs(bad) == 500.0:
                    k2, v2 = _values(cache, 0, b, lens[b] + n)
                    late, _, tol2 = _attend64(q64[at + j:at + n], k2, v2, lens[b] + j, gq)
                    assert (np.abs(got[at + j:at + n].double().cpu().numpy() - late) <= tol2).all()
                elif not np.isfinite(bad):
                    assert not bool(got[at + j:at + n].isfinite().any())
            halves[page, :, 8192 + 64 + place] = small
        at += n


@pytest.mark.parametrize("tokens", [131072, 1 << 20])
@pytest.mark.parametrize("n", [1, 20])
def test_sums_over_long_contexts_keep_their_precision(n, tokens):
    """A plan made while the sequence was short leaves all of a long context to one unit of four waves. Queries of zero
    give every token the same weight, a power of two, so that nothing but the sums' roundings is left: values of one
    code, +1 or -1, times a scale of each head, come out as they are. Half a step of the sum of P times a code and of
    the sum of P, for each of their additions (up to four in a matrix instruction, which takes 32 tokens), with the
    codes' offset of 128 in them for at most 16 groups; a lane's sum of weights, one addition a group; the output."""
    hkv = 8
    cache = PagedKVInt8TokCache(1, hkv, D, hkv, max_seqs=1, num_pages=8, max_pages_per_seq=tokens // GT)
    plan = cache.plan_chunks([n])
    assert len(plan.units) == 1 and not plan.wide
    cache.page_table[0] = torch.arange(tokens // GT, dtype=torch.int32) % 8
    scales = torch.tensor([0.02, 0.0123, 0.7, 1.001, 0.333, 0.00731, 0.05, 0.11]).half()
    sign = torch.where(torch.arange(D) % 2 == 0, 1, -1).to(torch.int8)
    pool = cache.pages[0]
    pool[:, :, 8192:16384] = sign.repeat(GT).view(torch.uint8).cuda()
    pool.view(torch.float16)[:, :, 8192:8192 + GT] = 1.0
    pool.view(torch.float16)[:, :, 8192 + GT:] = scales.cuda()[:, None]
    cache.pos[0] = tokens - n
    out = cache.attend_chunks(plan, torch.zeros(n, hkv, D, dtype=torch.float16, device="cuda"), 0).double().cpu().numpy()
    want = scales.double().numpy()[:, None] * sign.double().numpy()
    groups, held = tokens // GT // 4, 16  # of a wave; that the offset's share stays for
    adds = 4 * (groups + 2 * held * GT + 2 * held * GT) + groups / 2 + groups / held + 16
    err = np.abs(out - want) / np.abs(want)
    print(f"off by {err.max() / U16:.2f} half steps of fp16, allowed {1 + adds * 2.0 ** -24 / U16:.2f}", flush=True)
    assert (err <= U16 + adds * 2.0 ** -24).all()


def test_plans_to_read_are_no_steps():
    cache = _cache([70, 20], [10, 10], 8, 2, 190)
    span = cache.plan_read([5, 6], [60, 0])
    qkv, q = _randn((11, 12 * D), 191).cuda(), _randn((11, 8, D), 192).cuda()
    before, lens = cache.pages[0].clone(), list(cache._len)
    for call in (lambda: cache.append_chunks(span, qkv, 0), lambda: cache.attend_chunks(span, q, 0),
                 lambda: cache.advance_chunks(span), lambda: cache.advance_chunks(span, [1, 1]), lambda: cache.note_chunks(span)):
        with pytest.raises(ValueError, match="plan_read"):
            call()
    assert torch.equal(cache.pages[0], before) and cache._len == lens and cache.pos.tolist() == lens
    plan = cache.plan_chunks([3, 2])  # a step's plan reads what the step stored
    cache.append_chunks(plan, qkv[:5], 0)
    assert cache.read(plan, 0)[0].shape == (5, 2, D)


# ---------------------------------------------------------------- the forms that the call's size chooses


@pytest.mark.parametrize("lens,counts,hq,hkv,dtype,norm,rope,pad", [
    # from 256 tokens all heads of a token in one workgroup; more than 64 of them (32 of fp32) in several rounds of loads
    ([30], [300], 64, 8, torch.float16, True, True, 1),
    ([3], [260], 72, 8, torch.bfloat16, True, True, 0),
    ([0], [300], 40, 4, torch.float32, True, True, 0),
    # from 2048 tokens the queries pass the caches
    ([0, 100], [2000, 61], 32, 8, torch.float16, True, True, 2),
    ([5], [2100], 4, 2, torch.bfloat16, False, True, 0),
    ([0], [2050], 8, 2, torch.float32, True, False, 0),
])
def test_append_of_many_tokens(lens, counts, hq, hkv, dtype, norm, rope, pad):
    test_append_against_64_bits(lens, counts, hq, hkv, dtype, norm, rope, pad)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cls", [PagedKVInt8TokCache, PagedKVInt8Cache])
@pytest.mark.parametrize("lens,counts,starts,hkv", [
    ([700, 129, 333], None, None, 8),                            # four tokens a workgroup, the last one less
    ([2000, 1500, 64], [1900, 0, 63], [37, 1, 1], 3),
    ([9000, 77, 8000], None, None, 8),                           # sixteen, the last one less
    ([5000, 16000, 700], [4801, 15900, 3], [199, 50, 640], 7)])
def test_read_of_many_tokens(lens, counts, starts, hkv, cls, dtype):
    cache = _cache(lens, [3] * len(lens), hkv, hkv, 200, cls=cls)
    plan = cache.plan_read(counts, starts)
    counts = lens if counts is None else counts
    starts = [0] * len(lens) if starts is None else starts
    assert plan.total * hkv > 4096
    print(f"case read {cls.__name__} {lens} {dtype}: {plan.total} tokens", flush=True)
    room = tuple(torch.full((plan.total + 3, hkv, D), 5.0, dtype=dtype, device="cuda") for _ in range(2))
    cache.read(plan, 0, dtype, out=room)
    assert all(bool((x[plan.total:] == 5.0).all()) for x in room)
    at = 0
    for b, (first, n) in enumerate(zip(starts, counts)):
        end = first + n
        pages = cache.pages[0][cache.page_table[b, :-(-end // GT)].long()]
        for got, which in zip(room, (0, 1)):
            codes = pages[:, :, 8192 * which:8192 * (which + 1)]
            if cls is PagedKVInt8TokCache:
                scales = pages[:, :, 16384 + 128 * which:16384 + 128 * (which + 1)].contiguous().view(torch.float16)
                x = codes.contiguous().view(torch.int8).unflatten(2, (GT, D)).float() * scales[..., None].float()  # (exact)
            else:
                step, low = pages[:, :, 16384 + 512 * which:16384 + 512 * (which + 1)].contiguous().view(torch.float16).split(D, 2)
                x = (codes.unflatten(2, (GT, D)).double() * step[:, :, None].double() + low[:, :, None].double()).float()
            x = x.transpose(1, 2).flatten(0, 1)
            if cls is PagedKVInt8Cache and end > lens[b] // GT * GT:
                left = lens[b] - lens[b] // GT * GT
                x[lens[b] // GT * GT:][:left] = cache.rings[0][b, :, which, :left].transpose(0, 1).float()
            assert torch.equal(got[at:at + n], x[first:end].to(dtype)), (b, which)
        at += n


@pytest.mark.parametrize("lens,counts,hq", [
    ([20500], [3], 16),             # four waves of 81 groups each, rows in tiles of 32 and 16
    ([20500], [1], 2),
    ([6100, 36000], [70, 3], 2),    # a wide tile over 96 groups, and eight waves of 71 groups beside it
    ([36000, 10], [9, 300], 3),
])
def test_waves_of_more_groups_than_page_ids_at_once(lens, counts, hq):
    """A plan made while the sequences were short cuts nothing: each wave takes more groups than it holds page ids for.
    Each query is one and a half times a key of its own, spread over all groups, so that this token has most of the weight.
    (A lane's and an accumulator's additions stay within the 256 of the bound.)"""
    cache = _held_with_step(lens, counts, hq, 1, 210)
    for b in range(len(lens)):
        cache.pool.set_length(b, 0)
    plan = cache.plan_chunks(counts)
    units = plan.units.cpu()
    assert bool((units[units[:, 0] == int(np.argmax(lens)), 4] == 1).all())
    q, at = torch.empty(plan.total, hq, D, dtype=torch.float16), 0
    for b, n in enumerate(counts):
        k, _ = _values(cache, 0, b, lens[b] + n)
        token = (np.arange(n * hq) * (lens[b] / (n * hq)) + 31).astype(np.int64) % (lens[b] + 1)
        q[at:at + n] = torch.from_numpy(1.5 * k[token, 0]).half().view(n, hq, D)
        at += n
    lse = torch.empty(plan.total, hq, device="cuda")
    out = cache.attend_chunks(plan, q.cuda(), 0, lse=lse)
    _check_attention(cache, 0, plan, q, out, lse, lens)
