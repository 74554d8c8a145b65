"""GPU tests of the 4-bit format: quantizers, products with 4-bit weights, and the paged 4-bit cache's append, attention
and read, against plain computations in 64 bits.

Tolerances, from the roundings of the operators (u = 2^-11, half a step of fp16; U the output type's half step):

- codes and scales: the format's arithmetic is fp32 division and rounding, which numpy repeats bit for bit.
- products: xn is rounded to 11 bits at least (u; x itself where it is fp16 without a norm), its fp32 norm is 2^-20 off, the sums
  of in / 4 products a wave (each addition 2^-24) and the waves' are fp32, the output is rounded once:
  ``|err| <= U |y| + (e + (in / 4 + 40) 2^-24) sum|W xn| + 540 2^-24 sum(s |xn|) + 2^-35 max|xn| sum|W|``, e = u + 2^-19
  with a norm, u for bf16 (whose small values fall to denormals: half a step is 2^-25, of inputs held over 16 2^-21, the
  largest at least 2^14), else 0; the third term: codes held with an offset of 8, 15 at most, give a group's sum of 32 and
  its offset 36 additions of 2^-24 times 15 s |xn|. SwiGLU: the gate's and up's errors g', u' pass on as
  1.1 |u| g' + |silu| u' + g' u', the exponential's as 2^-20 |act|.
- append: fp32 norm and rotation 2^-19 of the row's largest off; a scale of 8
  significant bits (neighbours 2^-7 of a power of two apart: half a step is 2^-8 relative, at most) is within
  2^-8 + 2^-17 of amax / 7; a code is within half of the value over the stored scale, moved by
  8 * 2^-19 (the value) + 2^-20 (the quotient); beyond 7.5 it is clamped (a scale is at most 2^-8 too small: 7.03).
- attention: keys and values are exact operands, each weight is rounded to fp16 (u), a score is off by
  d = 2^-24 (130 sum|q k| + 540 sum(s |q|)) / sqrt(128) (fp32 sums; the second term: codes held with an offset of 8, 15 at
  most, give a group's sum of 32 channels and its offset 36 additions; it moves a weight and the sum of weights), an exponential by
  2^-22, a sum over up to 10000 tokens (at most 640 additions one after another in a lane or an accumulator, the joins)
  by 700 * 2^-24 < u / 8, weights below 2^-36 of the largest fall to 0 (10000 of them: 2^-22), and the output is rounded
  once: ``|err| <= u |out| + (u + u / 4 + 2 d) max|v| + 2^-24``.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from nova_amd import chunks as C
from nova_amd import gemv as G
from nova_amd.paged import GT, PAGE_BYTES_Q4, PagedKVInt8TokCache, PagedKVQ4Cache
from nova_amd.q4 import Q4Weight, dequantize_q4, quantize_q4

pytestmark = pytest.mark.gpu

D = 128
U16 = 2.0 ** -11
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def _randn(shape, seed, scale=1.0, dtype=torch.float16):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def _quantized(x: torch.Tensor):
    """The format in numpy's fp32: codes -7 .. 7 (float64) of ``x``'s shape and scales (fp16) of its groups."""
    v = x.float().cpu().numpy().reshape(-1, 32)
    with np.errstate(all="ignore"):
        amax = np.abs(v).max(1)  # (NaN passes on)
        s = np.maximum(amax / np.float32(7), np.float32(2.0 ** -24))
        s8 = torch.from_numpy(s).to(torch.bfloat16).float().numpy()
        s16 = np.where(np.float32(7) * s8 <= 65504, s8, np.where(np.isnan(amax), np.nan, np.inf)).astype(np.float16)
        code = np.clip(np.rint(v / s16.astype(np.float32)[:, None]), -7, 7)
    return code.astype(np.float64).reshape(x.shape), s16.reshape(*x.shape[:-1], x.shape[-1] // 32)


def _unpacked(codes: np.ndarray) -> np.ndarray:
    return np.stack((codes & 15, codes >> 4), -1).reshape(*codes.shape[:-1], 2 * codes.shape[-1]).astype(np.float64) - 8


def _weight_parts(w):
    """Codes ``[out, in]`` (float64) and scales ``[out, in / 32]`` of a weight, from its blocks as the header has them; and
    whether what is behind the last row and column has no scale."""
    (rows, n), tiles, nb = w.shape, -(-w.shape[0] // 16), -(-w.shape[1] // 128)
    data = w.data.cpu().numpy().reshape(tiles, nb, 1152)
    words = np.ascontiguousarray(data[:, :, :1024]).view(np.uint32).reshape(tiles, nb, 4, 16, 4)  # g, row, word
    codes = np.empty((tiles, 16, nb, 4, 4, 8))
    for e in range(8):
        codes[..., e] = ((words >> (4 * (e // 2 + 4 * (e % 2)))) & 15).transpose(0, 3, 1, 2, 4).astype(np.float64) - 8
    scales = np.ascontiguousarray(data[:, :, 1024:]).view(np.float16).reshape(tiles, nb, 4, 16).transpose(0, 3, 1, 2).reshape(tiles * 16, nb * 4)
    rest = np.ones(scales.shape, bool)
    rest[:rows, :n // 32] = False
    return codes.reshape(tiles * 16, nb * 128)[:rows, :n], scales[:rows, :n // 32], bool((scales[rest] == 0).all())


# ---------------------------------------------------------------- quantizers


@pytest.mark.parametrize("shape,dtype,scale", [((1, 32), torch.float16, 1.0), ((7, 96), torch.bfloat16, 3.0), ((333, 1056), torch.float16, 0.02),
                                               ((64, 2560), torch.float32, 100.0), ((5, 64), torch.float16, 1e-6),
                                               ((9, 64), torch.float32, 1e-9)])
def test_quantize_gives_the_formats_bits(shape, dtype, scale):
    x = _randn(shape, 1, scale, dtype)
    x[0, :32] = 0.0
    if shape[0] > 4:
        x[1, 3] = 7.0 * scale  # ties: halves of an exact scale
        x[1, :32] = (torch.arange(32) % 15 - 7).float().to(dtype) * 0.5
        x[2, 5] = 65504.0 if dtype == torch.float16 else 3e38
        x[3, 6], x[3, 40] = float("inf"), float("nan")
    w = quantize_q4(x.cuda())
    want, s16 = _quantized(x)
    codes, scales, rest = _weight_parts(w)
    assert w.shape == shape and rest and np.array_equal(scales, s16, equal_nan=True)
    fine = np.repeat(np.isfinite(s16.astype(np.float64)), 32, -1)
    assert np.array_equal(codes[fine], want[fine])
    with np.errstate(all="ignore"):
        value = want * np.repeat(s16.astype(np.float64), 32, -1)
    for to in (torch.float16, torch.bfloat16, torch.float32):
        got = dequantize_q4(w, to).double().cpu().numpy()
        exact = torch.from_numpy(value).to(to).double().numpy()
        assert np.array_equal(got[fine], exact[fine])
        assert not np.isfinite(got[~fine]).any()
    if dtype == torch.float16:
        assert np.array_equal(dequantize_q4(w).double().cpu().numpy()[fine], value[fine])


def test_quantize_takes_views_and_refuses():
    x = _randn((64, 128), 2).cuda()
    for view in (x.t(), x[:, 64:], x[::3], x.flatten()[3:3 + 32 * 64].view(32, 64)):
        a, b = quantize_q4(view), quantize_q4(view.contiguous().clone())
        assert torch.equal(a.data, b.data)
    assert quantize_q4(x[:0]).shape == (0, 128)
    for bad in (x[:, :40], x[0], x.int(), x[:, :0]):
        with pytest.raises(ValueError):
            quantize_q4(bad)
    w = quantize_q4(x)
    with pytest.raises(ValueError):
        dequantize_q4(w, torch.int8)
    for data, shape in ((w.data[:-1], (64, 128)), (w.data, (64, 256)), (w.data, (64, 100)), (w.data.cpu(), (64, 128)),
                        (w.data.view(torch.int8), (64, 128))):
        with pytest.raises(ValueError):
            Q4Weight(data, shape)


# ---------------------------------------------------------------- products


def _normed(x, gamma, eps):
    x = x.astype(np.float64)
    return x if gamma is None else x / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps) * gamma


def _linear64(x, w, s, gamma, eps, exact_x):
    """``W xn`` in 64 bits and the bound of all but the output's rounding; s: the scales of w's groups."""
    xn = _normed(x, gamma, eps)
    y = xn @ w.T
    e = 0.0 if exact_x else U16 + (2.0 ** -19 if gamma is not None else 0.0)
    tol = (e + (w.shape[1] / 4 + 40) * 2.0 ** -24) * (np.abs(xn) @ np.abs(w).T)
    tol += 540 * 2.0 ** -24 * (np.abs(xn).reshape(len(x), -1, 32).sum(-1) @ s.astype(np.float64).T)
    return y, tol + 2.0 ** -35 * np.abs(xn).max(-1, keepdims=True) * np.abs(w).sum(-1)


def _f(t):
    return None if t is None else t.double().cpu().numpy()


def _check_product(x, w, gamma, eps, residual, got, gated=False):
    assert got.dtype == x.dtype
    w64, x64 = _f(dequantize_q4(w, torch.float32)), _f(x).reshape(-1, x.shape[-1])
    y, tol = _linear64(x64, w64, _weight_parts(w)[1], _f(gamma), eps, gamma is None and x.dtype == torch.float16)
    if gated:
        n = y.shape[1] // 2
        g, up, tg, tu = y[:, :n], y[:, n:], tol[:, :n], tol[:, n:]
        silu = g / (1 + np.exp(-g))
        y = silu * up
        tol = 1.1 * np.abs(up) * tg + np.abs(silu) * tu + 1.1 * tg * tu + 2.0 ** -20 * np.abs(y)
    if residual is not None:
        y = y + _f(residual).reshape(y.shape)
        tol = tol + 2.0 ** -24 * np.abs(y)
    out = _f(got).reshape(y.shape)
    u = HALF[x.dtype]
    assert np.isfinite(out).all()
    err = np.abs(out - y) / (u * np.abs(y) + tol * (1 + u) + 2.0 ** -25)
    assert (err <= 1).all(), f"off by {err.max():.3f} of the bound"


PRODUCTS = [
    (1, 1, 32, torch.float16, False, False), (1, 16, 64, torch.bfloat16, True, True), (2, 17, 96, torch.float16, True, False),
    (3, 333, 1056, torch.bfloat16, True, True), (1, 6144, 2560, torch.float16, True, False), (8, 2560, 9728, torch.float16, False, True),
    (16, 100, 512, torch.float16, True, True), (17, 100, 544, torch.float16, True, False), (33, 50, 4096, torch.bfloat16, False, False),
    (64, 1000, 1024, torch.float16, True, True), (130, 40, 160, torch.bfloat16, True, True), (5, 31, 12800, torch.bfloat16, True, False),
    (1, 48, 40000, torch.float16, True, True), (16, 33, 20000, torch.float16, False, False), (7, 4096, 128, torch.float16, True, False),
    (15, 129, 608, torch.float16, False, True), (31, 2100, 416, torch.bfloat16, True, False), (48, 640, 2560, torch.float16, False, True),
    # the largest calls of one launch, and the next ones
    (8, 4096, 160, torch.float16, True, False), (8, 4100, 160, torch.bfloat16, True, True), (30, 1040, 96, torch.float16, True, True),
    (4, 48, 2560, torch.bfloat16, True, False), (4, 48, 2592, torch.float16, True, False), (2, 32, 5120, torch.float16, True, True),
    (1, 32, 10240, torch.float16, True, True), (1, 32, 10272, torch.bfloat16, True, True), (16, 528, 288, torch.float16, False, True),
    (17, 8224, 256, torch.float16, False, True), (40, 8300, 256, torch.bfloat16, True, False), (64, 8200, 224, torch.float16, True, False),
    (65, 70, 640, torch.float16, True, False), (11, 70, 4096, torch.bfloat16, True, True),
    (8, 40, 2560, torch.float16, True, False), (8, 40, 2592, torch.bfloat16, True, False), (1, 20, 20480, torch.bfloat16, True, False),
    (1, 20, 20512, torch.bfloat16, False, True), (9, 70, 640, torch.float16, True, False), (2, 70, 5152, torch.float16, True, True),
    (3, 70, 2720, torch.float16, True, False), (4, 70, 2528, torch.float16, True, False), (6, 70, 96, torch.bfloat16, True, False), (60, 90, 1184, torch.float16, True, False),
]


@pytest.mark.parametrize("tokens,n_out,n_in,dtype,norm,residual", PRODUCTS)
def test_gemv_against_64_bits(tokens, n_out, n_in, dtype, norm, residual):
    print(f"case gemv tokens={tokens} out={n_out} in={n_in} {dtype}", flush=True)
    w = quantize_q4(_randn((n_out, n_in), 3, n_in ** -0.5, dtype).cuda())
    x = _randn((tokens, n_in), 4, 3.0 if norm else 0.6, dtype).cuda()
    gamma = (1 + _randn((n_in,), 5, 0.2, torch.float32)).to(dtype).cuda() if norm else None
    res = _randn((tokens, n_out), 6, 1.0, dtype).cuda() if residual else None
    got = G.rms_gemv_q4(x, w, gamma, 1e-6, res)
    _check_product(x, w, gamma, 1e-6, res, got)
    # rows behind the last token stay, the residual may be the output, the same call gives the same bits
    room = torch.full((tokens + 2, n_out), 9.0, dtype=dtype, device="cuda")
    if res is not None:
        room[:tokens] = res
    assert G.rms_gemv_q4(x, w, gamma, 1e-6, None if res is None else room[:tokens], out=room[:tokens]).data_ptr() == room.data_ptr()
    assert torch.equal(room[:tokens], got) and bool((room[tokens:] == 9.0).all())


@pytest.mark.parametrize("tokens,n_out,n_in,dtype,norm,residual", PRODUCTS)
def test_swiglu_against_64_bits(tokens, n_out, n_in, dtype, norm, residual):
    print(f"case swiglu tokens={tokens} inter={n_out} in={n_in} {dtype}", flush=True)
    w = quantize_q4(_randn((2 * n_out, n_in), 7, 1.5 * n_in ** -0.5, dtype).cuda())
    x = _randn((tokens, n_in), 8, 2.0, dtype).cuda()
    gamma = (1 + _randn((n_in,), 9, 0.2, torch.float32)).to(dtype).cuda() if norm else None
    _check_product(x, w, gamma, 1e-6, None, G.swiglu_gemv_q4(x, w, gamma, 1e-6), gated=True)


def test_a_tokens_result_is_its_own():
    """A token's values do not hang on its neighbours', finite or not."""
    w = quantize_q4(_randn((300, 640), 10, 0.05).cuda())
    gamma = (1 + _randn((640,), 11, 0.2, torch.float32)).half().cuda()
    x = _randn((16, 640), 12, 2.0).cuda()
    want = G.rms_gemv_q4(x, w, gamma)
    spoilt = x.clone()
    spoilt[3, 5], spoilt[7, 600] = float("nan"), float("inf")
    got = G.rms_gemv_q4(spoilt, w, gamma)
    keep = [t for t in range(16) if t not in (3, 7)]
    assert torch.equal(got[keep], want[keep])
    assert bool(got[[3, 7]].isnan().all())
    for t in (0, 9):  # (the number of tokens chooses the kernel, and so the order of the sums)
        _check_product(x[t:t + 1], w, gamma, 1e-6, None, G.rms_gemv_q4(x[t:t + 1].contiguous(), w, gamma))


@pytest.mark.parametrize("dtype,size", [(torch.bfloat16, 1e30), (torch.bfloat16, 1e-30), (torch.float16, 60000.0), (torch.float16, 1e-6)])
def test_inputs_of_any_size(dtype, size):
    """The norm takes inputs of any size (bf16 far beyond fp16's range, fp16's own largest and denormals); without one a bf16
    input keeps its range."""
    x = (_randn((3, 256), 13, 1.0, torch.float32).clamp(-1, 1) * size).to(dtype).cuda()
    w = quantize_q4(_randn((40, 256), 14, 0.06).cuda())
    gamma = (1 + _randn((256,), 15, 0.2, torch.float32)).to(dtype).cuda()
    if size < 1e19:  # (the mean of squares fits fp32)
        _check_product(x, w, gamma, 1e-12, None, G.rms_gemv_q4(x, w, gamma, 1e-12))
    if dtype == torch.bfloat16:
        _check_product(x, w, None, 0, None, G.rms_gemv_q4(x, w))
    big = (gamma.float() * 30000).to(dtype)
    y = _randn((3, 256), 16, 1.0, dtype).cuda()
    if dtype == torch.bfloat16:
        _check_product(y, w, big, 1e-6, None, G.rms_gemv_q4(y, w, big))
    z = torch.zeros(2, 256, dtype=dtype, device="cuda")
    assert bool((G.rms_gemv_q4(z, w, gamma) == 0).all())


def test_product_refusals():
    w = quantize_q4(_randn((64, 128), 17).cuda())
    x = _randn((4, 128), 18).cuda()
    res = _randn((4, 64), 19).cuda()
    gamma = torch.ones(128, dtype=torch.float16, device="cuda")
    wide = torch.zeros(4, 256, dtype=torch.float16, device="cuda")
    for args in [(x.float(),), (x[:, :64].contiguous(),), (x.t(),), (wide[:, :128],), (x.cpu(),), (x.flatten()[1:129],)]:
        with pytest.raises(ValueError):
            G.rms_gemv_q4(*args, w)
    for kw in [dict(gamma=gamma.float()), dict(gamma=gamma[:64]), dict(gamma=gamma.bfloat16()), dict(residual=res[:3]),
               dict(residual=res.bfloat16()), dict(residual=res.t()), dict(out=res[:2]), dict(out=res.float()), dict(out=res.t()),
               dict(out=x.flatten()[:256].view(4, 64)), dict(out=w.data.view(torch.float16)[:256].view(4, 64))]:
        with pytest.raises(ValueError):
            G.rms_gemv_q4(x, w, **kw)
    room = torch.zeros(5 * 64, dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError):
        G.rms_gemv_q4(x, w, residual=room[:256].view(4, 64), out=room[64:].view(4, 64))
    with pytest.raises(ValueError):
        G.swiglu_gemv_q4(x, quantize_q4(_randn((63, 128), 20).cuda()))
    with pytest.raises(ValueError):
        G.rms_gemv_q4(x, x)
    assert G.rms_gemv_q4(x[:0], w).shape == (0, 64) and G.rms_gemv_q4(x[0], w).shape == (64,)
    assert G.rms_gemv_q4(x.view(2, 2, 128), w).shape == (2, 2, 64)


# ---------------------------------------------------------------- the cache


def _cache(lens, room, hq, hkv, seed, layers=1, cls=PagedKVQ4Cache, fill=True):
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


def _held_with_step(lens, counts, hq, hkv, seed):
    cache = _cache([a + n for a, n in zip(lens, counts)], [0] * len(lens), hq, hkv, seed)
    for b, n in enumerate(lens):
        cache.pool.set_length(b, n)
        cache.pos[b] = n
    return cache


_T, _R = np.arange(64)[:, None], np.arange(4)[None]
PLACE = (64 * _R + _T, 64 * _R + _T // 8 * 8 + 2 * (_T % 4) + _T // 4 % 2)


def _bytes(which, slot):
    """Where a token's 64 bytes of codes and its four scales (two bytes each) are in a page of one KV head."""
    scales = [8192 + 1024 * which // 2 + 2 * int(p) for p in PLACE[which][slot]]
    return [(4096 * which + 64 * slot, 64)] + [(s, 2) for s in scales]


def _codes(cache, layer, b, n):
    """Sequence b's first n tokens from the bytes of its pages: K codes ``[n, H_kv, 128]`` and scales ``[n, H_kv, 4]``,
    V's, as float64 numpy arrays."""
    row = cache.page_table[b].cpu().numpy()
    groups = -(-n // GT)
    rows = cache.pages[layer][torch.from_numpy(row[:groups].astype(np.int64)).cuda()].cpu().numpy()  # [G, H, PAGE]
    h, out = cache.num_kv_heads, []
    for which in (0, 1):
        c = _unpacked(rows[:, :, 4096 * which:4096 * (which + 1)].reshape(groups, h, GT, 64))
        if which == 0:  # (K's words 4 j + g and 4 g + j in each other's place)
            c = c.reshape(groups, h, GT, 4, 4, 8).swapaxes(3, 4).reshape(groups, h, GT, D)
        s = np.ascontiguousarray(rows[:, :, 8192 + 512 * which:8704 + 512 * which]).view(np.float16)[:, :, PLACE[which]]
        out += [c.transpose(0, 2, 1, 3).reshape(groups * GT, h, D)[:n], s.astype(np.float64).transpose(0, 2, 1, 3).reshape(groups * GT, h, 4)[:n]]
    return out


def _values(cache, layer, b, n):
    kc, ks, vc, vs = _codes(cache, layer, b, n)
    with np.errstate(invalid="ignore"):
        return kc * np.repeat(ks, 32, -1), vc * np.repeat(vs, 32, -1)


def _attend64(q, k, v, ks, start, gq, u=1.25 * U16):
    """Softmax attention of tokens at positions start .. over k, v ``[n, H_kv, 128]`` in 64 bits: output,
    log-sum-exp and the bound of the module's docstring. ks: K's scales ``[n, H_kv, 4]``."""
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
            d = 2.0 ** -24 / np.sqrt(D) * (130 * np.abs(kk) @ np.abs(q[i, h])
                                           + 540 * ks[:n, h // gq] @ np.abs(q[i, h]).reshape(4, 32).sum(1)).max()
            tol[i, h] = U16 * np.abs(out[i, h]) + (u + 2 * d) * np.abs(vv).max() + 2.0 ** -24
    return out, lse, tol


def _check_attention(cache, layer, plan, q, out, lse, starts):
    gq, at = cache.num_q_heads // cache.num_kv_heads, 0
    q64, out, lse = _f(q), _f(out), _f(lse)
    assert np.isfinite(out[:plan.total]).all()
    for b, n in enumerate(plan.counts):
        if n:
            k, v = _values(cache, layer, b, starts[b] + n)
            want, wl, tol = _attend64(q64[at:at + n], k, v, _codes(cache, layer, b, starts[b] + n)[1], starts[b], gq)
            err = np.abs(out[at:at + n] - want)
            assert (err <= tol).all(), f"sequence {b}: off by {(err / tol).max():.2f} of the bound"
            if lse is not None:
                # a score is off by d, the sum of weights by 2^-13 (the exponentials and fp32 sums)
                assert np.abs(lse[at:at + n] - wl).max() <= 2e-3, f"sequence {b}: lse"
        at += n


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_prefill_gives_the_quantizers_bits(dtype):
    cache = _cache([0, 0], [300, 70], 4, 2, 1)
    before = cache.pages[0].clone()
    for b, n in ((0, 197), (1, 64)):
        k, v = _randn((1, 2, n, D), 2 + b, 1.0, dtype), _randn((1, 2, n, D), 4 + b, 5.0, dtype)
        k[0, 0, 3], k[0, 1, 5, 7] = 0.0, 30000.0
        cache.prefill(b, 0, k.cuda(), v.transpose(1, 2).contiguous().transpose(1, 2).cuda())
        assert cache._len[b] == n and int(cache.pos[b]) == n
        got = _codes(cache, 0, b, n)
        for which, x in enumerate((k, v)):
            code, s16 = _quantized(x[0])
            assert np.array_equal(got[2 * which], code.transpose(1, 0, 2)) and np.array_equal(got[2 * which + 1], s16.astype(np.float64).transpose(1, 0, 2))
    # nothing but those tokens' bytes changed
    pages = cache.pages[0].clone()
    for b, n in ((0, 197), (1, 64)):
        for p in range(n):
            for which in (0, 1):
                for a, w in _bytes(which, p % GT):
                    pages[int(cache.page_table[b, p // GT]), :, a:a + w] = before[int(cache.page_table[b, p // GT]), :, a:a + w]
    assert torch.equal(pages, before)


# ---------------------------------------------------------------- append


def _rotated(x, gamma, eps, inv_freq, pos):
    x = _normed(x, gamma, eps)
    if inv_freq is not None:
        a = pos[:, None].astype(np.float64) * inv_freq.astype(np.float64)
        c, s = np.cos(a)[:, None], np.sin(a)[:, None]
        x = np.concatenate((x[..., :64] * c - x[..., 64:] * s, x[..., 64:] * c + x[..., :64] * s), -1)
    return x


def _inv_freq(theta=1e6):
    return (theta ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)).float().cuda()


@pytest.mark.parametrize("lens,counts,hq,hkv,dtype,norm,rope,pad", [
    ([0], [1], 1, 1, torch.float16, True, True, 0),
    ([5, 63, 64, 200], [1, 1, 1, 1], 32, 8, torch.float16, True, True, 0),
    ([5, 63, 0, 200], [130, 1, 0, 65], 32, 8, torch.float16, True, True, 3),
    ([1000, 0], [700, 500], 28, 4, torch.bfloat16, True, True, 0),
    ([17], [129], 16, 1, torch.float32, True, True, 2),
    ([40, 9], [70, 3], 6, 2, torch.float16, True, False, 0),
    ([40, 9], [70, 3], 6, 2, torch.bfloat16, False, True, 0),
    ([100], [2100], 4, 2, torch.float16, True, True, 0),
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
    inv = _inv_freq() if rope else None
    q_out = torch.full((plan.total + pad, hq, D), 7.0, dtype=torch.float16, device="cuda")
    q = cache.append_chunks(plan, qkv, 0, gq, gk, 1e-6, inv, q_out=q_out)
    torch.cuda.synchronize()
    assert q is q_out and bool((q_out[plan.total:] == 7.0).all())
    x = _f(qkv)[:plan.total].reshape(plan.total, heads, D)
    pos = np.concatenate([np.arange(n) + s for s, n in zip(lens, counts)])
    want_q = _rotated(x[:, :hq], _f(gq), 1e-6, _f(inv), pos)
    want_k = _rotated(x[:, hq:hq + hkv], _f(gk), 1e-6, _f(inv), pos)
    err = np.abs(_f(q)[:plan.total] - want_q)
    assert (err <= U16 * np.abs(want_q) + 2.0 ** -19 * np.abs(want_q).max(-1, keepdims=True) + 2.0 ** -25).all()
    at = 0
    for b, n in enumerate(counts):
        kc, ks, vc, vs = (z[lens[b]:] for z in _codes(cache, 0, b, lens[b] + n))
        for codes, scales, want in ((kc, ks, want_k[at:at + n]), (vc, vs, x[at:at + n, hq + hkv:])):
            amax = np.abs(want).reshape(*want.shape[:2], 4, 32).max(-1)
            assert (np.abs(scales - amax / 7) <= (2.0 ** -8 + 2.0 ** -17) * amax / 7 + 2.0 ** -24).all()
            quotient = np.clip(want / np.repeat(scales, 32, -1), -7, 7)
            row = np.abs(want).max(-1, keepdims=True) / np.repeat(scales, 32, -1)
            assert (np.abs(codes - quotient) <= 0.5 + 2.0 ** -20 * 8 + 2.0 ** -19 * row).all()
        at += n
    # nothing but the new tokens' rows changed
    pages, old = cache.pages[0].clone(), before
    for b, n in enumerate(counts):
        for p in range(lens[b], lens[b] + n):
            pg = int(cache.page_table[b, p // GT])
            for which in (0, 1):
                for a, w in _bytes(which, p % GT):
                    pages[pg, :, a:a + w] = old[pg, :, a:a + w]
    assert torch.equal(pages, old)


def test_append_without_norm_and_rotation_gives_the_quantizers_bits():
    for dtype in (torch.float16, torch.bfloat16, torch.float32):
        cache = _cache([30], [100], 4, 2, 8)
        plan = cache.plan_chunks([100])
        qkv = _randn((100, 8 * D), 9, 2.0, dtype)
        qkv[3, 4 * D:5 * D] = 0.0
        qkv[4, 5 * D] = 60000.0
        q = cache.append_chunks(plan, qkv.cuda(), 0)
        assert torch.equal(q.view(100, 4 * D), qkv[:, :4 * D].half().cuda())
        got = _codes(cache, 0, 0, 130)
        for which in (0, 1):
            code, s16 = _quantized(qkv[:, (4 + 2 * which) * D:(6 + 2 * which) * D].reshape(100, 2, D))
            assert np.array_equal(got[2 * which][30:], code) and np.array_equal(got[2 * which + 1][30:], s16.astype(np.float64))


def test_append_in_place_strided_and_without_a_page():
    lens, counts, hq, hkv = [70, 3], [40, 90], 8, 2
    base = _randn((140, 14 * D), 20)
    gam = [(1 + _randn((D,), 5 + i, 0.2, torch.float32)).half().cuda() for i in range(2)]
    a, b = _cache(lens, counts, hq, hkv, 21), _cache(lens, counts, hq, hkv, 21)
    pa, pb = a.plan_chunks(counts), b.plan_chunks(counts)
    plain = base[:, :12 * D].contiguous().cuda()
    q = a.append_chunks(pa, plain, 0, *gam, 1e-6, _inv_freq())
    wide = base.cuda()
    own = wide[:, :hq * D].unflatten(1, (hq, D))
    got = b.append_chunks(pb, wide[:, :12 * D], 0, *gam, 1e-6, _inv_freq(), q_out=own)
    assert got.data_ptr() == wide.data_ptr() and torch.equal(got[:130], q) and torch.equal(a.pages[0], b.pages[0])
    c = _cache(lens, counts, hq, hkv, 21)
    pc = c.plan_chunks(counts)
    c.page_table[0, 1] = -1
    c.page_table[1].fill_(1 << 20)  # no page of this pool
    before = c.pages[0].clone()
    c.append_chunks(pc, plain, 0)
    torch.cuda.synchronize()
    assert torch.equal(c.pages[0], before)


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
    ([900], [64], 1, 1),
    ([900, 30], [65, 64], 1, 1),
    ([500], [255], 1, 1),
    ([500], [257], 1, 1),
    ([5000, 700, 60], [40, 2, 17], 16, 2),
    ([9000], [33], 2, 1),
    ([3000, 0, 64], [300, 31, 1], 3, 3),
]


@pytest.mark.parametrize("lens,counts,hq,hkv", ATTEND)
def test_attend_against_64_bits(lens, counts, hq, hkv):
    print(f"case attend lens={lens} counts={counts} hq={hq} hkv={hkv}", flush=True)
    cache = _held_with_step(lens, counts, hq, hkv, 40)
    plan = cache.plan_chunks(counts)
    q = _randn((plan.total + 2, hq, D), 41, 1.5).cuda()
    out = torch.full((plan.total + 2, hq, D), 9.0, dtype=torch.float16, device="cuda")
    lse = torch.full((plan.total + 2, hq), 9.0, device="cuda")
    got = cache.attend_chunks(plan, q, 0, out=out, lse=lse)
    torch.cuda.synchronize()
    assert got is out and bool((out[plan.total:] == 9.0).all()) and bool((lse[plan.total:] == 9.0).all())
    _check_attention(cache, 0, plan, q, out, lse, lens)
    assert torch.equal(cache.attend_chunks(plan, q, 0), out[:plan.total])


def test_attend_reads_any_strides_and_writes_any():
    lens, counts, hq, hkv = [70, 10], [30, 5], 8, 2
    cache = _held_with_step(lens, counts, hq, hkv, 42)
    plan = cache.plan_chunks(counts)
    q = _randn((35, hq, D), 43).cuda()
    want = cache.attend_chunks(plan, q, 0)
    by_head = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(cache.attend_chunks(plan, by_head, 0), want)
    wide = torch.zeros(35, hq, 2 * D, dtype=torch.float16, device="cuda")
    wide[..., :D] = q
    other = torch.zeros(hq, 35, 2 * D, dtype=torch.float16, device="cuda").transpose(0, 1)[..., D:]
    assert torch.equal(cache.attend_chunks(plan, wide[..., :D], 0, out=other), want)
    odd = torch.empty(35 * hq * D + 1, dtype=torch.float16, device="cuda")[1:].view(35, hq, D)
    odd.copy_(q)
    assert torch.equal(cache.attend_chunks(plan, odd, 0), want)


@pytest.mark.parametrize("counts", [[3, 1], [33, 70], [140, 65]])
def test_masked_places_may_hold_anything(counts):
    """Rows of a page behind the sequence's last token, and later tokens of the step, are infinite or NaN: rows that do not
    attend them stay as they are; those that do are not finite."""
    lens, hq, hkv = [100, 62], 8, 2
    cache = _held_with_step(lens, counts, hq, hkv, 50)
    plan = cache.plan_chunks(counts)
    q = _randn((plan.total, hq, D), 51, 1.5).cuda()
    lse = torch.empty(plan.total, hq, device="cuda")
    want = cache.attend_chunks(plan, q, 0, lse=lse).clone()
    want_lse = lse.clone()
    for bits in (0x7c00, 0xfc00, 0x7e00, 0x7bff):
        held = cache.pages[0].clone()
        for b, n in enumerate(counts):
            end = lens[b] + n
            for p in range(end, -(-end // GT) * GT):
                for which in (0, 1):
                    for a, w in _bytes(which, p % GT):
                        held[int(cache.page_table[b, p // GT]), :, a:a + w].view(torch.int16 if w == 2 else torch.uint8).fill_(
                            (bits if bits < 0x8000 else bits - 0x10000) if w == 2 else 0x5a)
        cache.pages[0], good = held, cache.pages[0]
        got = cache.attend_chunks(plan, q, 0, lse=lse)
        assert torch.equal(got, want) and torch.equal(lse, want_lse)
        # the last token of each sequence's step: only its own rows may change
        for b, n in enumerate(counts):
            p = lens[b] + n - 1
            a, w = _bytes(1, p % GT)[2]
            held[int(cache.page_table[b, p // GT]), 0, a:a + w].view(torch.int16).fill_(bits if bits < 0x8000 else bits - 0x10000)
        got = cache.attend_chunks(plan, q, 0)
        last = np.cumsum(counts) - 1
        others = [t for t in range(plan.total) if t not in last]
        assert torch.equal(got[others], want[others])
        if bits != 0x7bff:
            assert not bool(got[list(last), :hq // hkv].isfinite().all(-1).any())
        assert torch.equal(got[:, hq // hkv:], want[:, hq // hkv:])
        cache.pages[0] = good


@pytest.mark.parametrize("counts", [[2, 1], [40, 300]])
def test_groups_without_a_page_take_no_part(counts):
    lens, hq, hkv = [300, 200], 4, 2
    cache = _held_with_step(lens, counts, hq, hkv, 60)
    plan = cache.plan_chunks(counts)
    q = _randn((plan.total, hq, D), 61, 1.5).cuda()
    cache.page_table[0, 2] = -1
    cache.page_table[0, 3] = cache.num_pages  # no page of this pool
    cache.page_table[1] = -1
    lse = torch.empty(plan.total, hq, device="cuda")
    out = cache.attend_chunks(plan, q, 0, lse=lse)
    assert bool((out[counts[0]:] == 0).all()) and bool((lse[counts[0]:] == -np.inf).all())
    table = cache.page_table[0].clone()
    cache.page_table[0, 2:4] = cache.page_table[0, 0]  # (any page: its tokens are left out below)
    k, v = _values(cache, 0, 0, lens[0] + counts[0])
    ks = _codes(cache, 0, 0, lens[0] + counts[0])[1]
    cache.page_table[0] = table
    keep = np.r_[0:128, 256:lens[0] + counts[0]]
    want, _, tol = _attend64(_f(q)[:counts[0]], k[keep], v[keep], ks[keep], lens[0] - 128, hq // hkv)
    assert (np.abs(_f(out)[:counts[0]] - want) <= tol).all()


@pytest.mark.parametrize("counts", [[1], [20], [150]])
def test_values_and_scores_of_any_size(counts):
    """Values near fp16's largest and down to its denormals, scores that grow and fall by much along the context."""
    lens, hq, hkv = [640], 4, 2
    n = lens[0] + counts[0]
    for size, grow in ((9000.0, 1.0), (3e-6, 1.0), (1.0, 40.0)):
        cache = _held_with_step(lens, counts, hq, hkv, 70)
        ramp = torch.linspace(1, grow, n)[None, None, :, None]
        k = (_randn((1, hkv, n, D), 71, 1.0, torch.float32) * ramp).half().cuda()
        v = (_randn((1, hkv, n, D), 72, 1.0, torch.float32) * size).clamp(-65000, 65000).half().cuda()
        cache.prefill(0, 0, k, v)
        cache.pool.set_length(0, lens[0])
        cache.pos[0] = lens[0]
        plan = cache.plan_chunks(counts)
        q = _randn((plan.total, hq, D), 73, 1.5).cuda()
        lse = torch.empty(plan.total, hq, device="cuda")
        out = cache.attend_chunks(plan, q, 0, lse=lse)
        _check_attention(cache, 0, plan, q, out, None, lens)


@pytest.mark.parametrize("counts", [[5], [40], [130]])
def test_a_query_that_is_not_finite_spoils_its_own_row(counts):
    cache = _held_with_step([130], counts, 4, 2, 80)
    plan = cache.plan_chunks(counts)
    q = _randn((plan.total, 4, D), 81, 1.5).cuda()
    want = cache.attend_chunks(plan, q, 0)
    for bad in (float("nan"), float("inf")):
        spoilt = q.clone()
        spoilt[2, 1, 17] = bad
        got = cache.attend_chunks(plan, spoilt, 0)
        assert bool(got[2, 1].isnan().all())
        got[2, 1] = want[2, 1]
        assert torch.equal(got, want)


@pytest.mark.parametrize("counts", [[3, 1], [90, 70]])
def test_a_plan_outlives_its_lengths(counts):
    lens, hq, hkv = [50, 700], 8, 2
    cache = _held_with_step([200, 900], counts, hq, hkv, 90)
    for b, n in enumerate(lens):
        cache.pool.set_length(b, n)
    plan = cache.plan_chunks(counts)  # planned at the shorter lengths
    for b, n in enumerate([200, 900]):
        cache.pool.set_length(b, n)
        cache.pos[b] = n
    q = _randn((plan.total, hq, D), 91, 1.5).cuda()
    out = cache.attend_chunks(plan, q, 0)
    _check_attention(cache, 0, plan, q, out, None, [200, 900])


def test_pages_beyond_four_gigabytes():
    hkv, start = 8, 200
    page = hkv * PAGE_BYTES_Q4
    n_pages = (1 << 32) // page + 8
    cache = PagedKVQ4Cache(1, hkv, D, 16, max_seqs=1, num_pages=n_pages, max_pages_per_seq=8)
    cache._free = list(range(n_pages - 1, n_pages - 6, -1))[::-1]  # the last pages of the pool
    k, v = _randn((1, hkv, start + 3, D), 95).cuda(), _randn((1, hkv, start + 3, D), 96).cuda()
    cache.prefill(0, 0, k, v)
    cache.pool.set_length(0, start)
    cache.pos[0] = start
    plan = cache.plan_chunks([3])
    qkv = _randn((3, 32 * D), 97).cuda()
    q = cache.append_chunks(plan, qkv, 0)
    _check_attention(cache, 0, plan, q, cache.attend_chunks(plan, q, 0), None, [start])
    span = cache.plan_read([3], [start - 3])
    got = cache.read(span, 0)
    kk, vv = _values(cache, 0, 0, start)
    assert np.array_equal(_f(got[0]), kk[start - 3:]) and np.array_equal(_f(got[1]), vv[start - 3:])


@pytest.mark.parametrize("n,counts", [(1 << 20, [1]), (1 << 18, [70])])
def test_sums_over_long_contexts_keep_their_precision(n, counts):
    """All tokens weigh alike: the output is the mean of V, whose tokens share one page. Sums in fp32: at most 2 half steps
    more than the output's rounding (as many additions one after another as a wave has tokens, 2^-25 each on average)."""
    cache = PagedKVQ4Cache(1, 1, D, 2, max_seqs=1, num_pages=1, max_pages_per_seq=n // GT + 4)
    cache.prefill(0, 0, torch.zeros(1, 1, 63, D).half().cuda(), torch.zeros(1, 1, 63, D).half().cuda())
    cache.pages[0][:, :, 4096:8192] = 0x9a  # V codes 2 and 1
    cache.pages[0][:, :, 8192:].view(torch.float16).fill_(0.5)
    cache.page_table[0].fill_(0)
    cache.pool.owned[0] = [0] * (n // GT + 4)
    cache.pool.length[0] = n
    cache.pos[0] = n
    plan = cache.plan_chunks(counts)
    out = cache.attend_chunks(plan, torch.ones(plan.total, 2, D, dtype=torch.float16, device="cuda"), 0)
    want = torch.tensor([1.0, 0.5], device="cuda").repeat(64)
    assert bool(((out.double() - want).abs() <= 3 * U16 * want).all())


# ---------------------------------------------------------------- read


@pytest.mark.parametrize("lens,counts,starts,hkv,dtype", [
    ([1], [1], [0], 1, torch.float16), ([200, 75], [200, 75], [0, 0], 8, torch.float16),
    ([100, 0, 333, 64], [90, 0, 100, 64], [5, 0, 129, 0], 2, torch.bfloat16), ([4097], [3001], [60], 4, torch.float32),
    ([9000, 9000], [8000, 8999], [500, 0], 8, torch.float16)])
def test_read(lens, counts, starts, hkv, dtype):
    cache = _cache(lens, [0] * len(lens), hkv, hkv, 100)
    plan = cache.plan_read(counts, starts)
    k, v = (torch.full((plan.total + 1, hkv, D), 9.0, dtype=dtype, device="cuda") for _ in range(2))
    cache.read(plan, 0, dtype, out=(k, v))
    want = [_values(cache, 0, b, n) for b, n in enumerate(lens)]
    for got, which in ((k, 0), (v, 1)):
        ref = np.concatenate([w[which][s:s + n] for w, s, n in zip(want, starts, counts)])
        assert torch.equal(got[:plan.total].cpu(), torch.from_numpy(ref).to(dtype)) and bool((got[plan.total:] == 9.0).all())
    cache.page_table[0, 0] = -1
    got = cache.read(plan, 0, dtype)
    gone = max(0, min(GT, starts[0] + counts[0]) - starts[0])
    assert bool((got[0][:gone] == 0).all()) and torch.equal(got[1][gone:], v[gone:plan.total])


# ---------------------------------------------------------------- as it is used


def test_refusals():
    cache = _cache([70], [10], 8, 2, 110)
    plan = cache.plan_chunks([5])
    q = _randn((5, 8, D), 111).cuda()
    for call in (cache.plan, lambda: cache.decode_step(q, q, q, 0), lambda: cache.attend(q, 0)):
        with pytest.raises(NotImplementedError):
            call()
    other = _cache([70], [10], 8, 2, 110, cls=PagedKVInt8TokCache)
    with pytest.raises(ValueError):
        other.attend_chunks(plan, q, 0)
    for bad in (q[:4], q[:, :4], q.float(), q.cpu()):
        with pytest.raises(ValueError):
            cache.attend_chunks(plan, bad, 0)
    with pytest.raises(ValueError):
        cache.attend_chunks(plan, q, 0, out=q)
    with pytest.raises(ValueError):
        cache.attend_chunks(plan, q, 0, lse=torch.zeros(5, 7, device="cuda"))
    with pytest.raises(ValueError):
        cache.append_chunks(plan, _randn((5, 11 * D), 112).cuda(), 0)
    with pytest.raises(ValueError):
        cache.prefill(0, 0, q[None], q[None])
    with pytest.raises(RuntimeError):
        cache.plan_chunks([1000])


def test_a_captured_step_follows_the_sequences():
    """Projection, append, attention, projection with the residual, SwiGLU: captured once, replayed over growing sequences
    with eager work between, against the same calls made eagerly."""
    lens, counts, hq, hkv, hidden = [100, 7, 1000], [1, 3, 40], 8, 2, 512
    caches = [_cache(lens, [400] * 3, hq, hkv, 120) for _ in range(2)]
    w_qkv, w_o = quantize_q4(_randn((12 * D, hidden), 121, 0.05).cuda()), quantize_q4(_randn((hidden, hq * D), 122, 0.03).cuda())
    w_gu, w_down = quantize_q4(_randn((2 * 640, hidden), 123, 0.05).cuda()), quantize_q4(_randn((hidden, 640), 124, 0.04).cuda())
    gam = [(1 + _randn((n,), 125 + i, 0.2, torch.float32)).half().cuda() for i, n in enumerate((hidden, hidden, D, D))]
    x = torch.zeros(sum(counts), hidden, dtype=torch.float16, device="cuda")
    inv = _inv_freq()
    plans = [c.plan_chunks(counts) for c in caches]

    def step(cache, plan):
        qkv = G.rms_gemv_q4(x, w_qkv, gam[0])
        q = cache.append_chunks(plan, qkv, 0, gam[2], gam[3], 1e-6, inv)
        o = cache.attend_chunks(plan, q, 0)
        h = G.rms_gemv_q4(o.view(-1, hq * D), w_o, residual=x)
        act = G.swiglu_gemv_q4(h, w_gu, gam[1])
        y = G.rms_gemv_q4(act, w_down, residual=h)
        cache.pos[:3].add_(plan.new)
        return qkv, q, o, h, act, y

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(caches[0], plans[0])  # (loads what a capture may not)
    torch.cuda.current_stream().wait_stream(side)
    caches[0].pos[:3] = torch.tensor(lens, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(caches[0], plans[0])
    for r in range(4):
        x.copy_(_randn(x.shape, 130 + r).cuda())
        graph.replay()
        want = step(caches[1], plans[1])
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b), r
        assert torch.equal(caches[0].pages[0], caches[1].pages[0]) and torch.equal(caches[0].pos, caches[1].pos)
        start = [n + r * m for n, m in zip(lens, counts)]
        # each operator against 64 bits on the inputs that it had
        qkv, q, o, h, act, y = want
        _check_product(x, w_qkv, gam[0], 1e-6, None, qkv)
        _check_attention(caches[1], 0, plans[1], q, o, None, start)
        _check_product(o.view(-1, hq * D), w_o, None, 0, x, h)
        _check_product(h, w_gu, gam[1], 1e-6, None, act, gated=True)
        _check_product(act, w_down, None, 0, h, y)
        for c, p in zip(caches, plans):
            c.note_chunks(p)


def test_streams_other_than_the_tensors_own():
    cache = _held_with_step([500, 30], [2, 40], 8, 2, 140)
    plan = cache.plan_chunks([2, 40])
    q = _randn((42, 8, D), 141, 1.5).cuda()
    w = quantize_q4(_randn((300, 512), 142, 0.05).cuda())
    x = _randn((20, 512), 143).cuda()
    want, product = cache.attend_chunks(plan, q, 0), G.rms_gemv_q4(x, w)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append([(cache.attend_chunks(plan, q, 0), G.rms_gemv_q4(x, w)) for _ in range(5)])
    torch.cuda.synchronize()
    for outs in got:
        for a, b in outs:
            assert torch.equal(a, want) and torch.equal(b, product)


# ---------------------------------------------------------------- a decoder


def _decoder(cfg):
    """A decoder whose weights are values of the 4-bit format: the same weights in fp16 and in 4 bits."""
    from nova_amd.skeleton import SkeletonForCausalLM

    model = SkeletonForCausalLM(cfg, seed=3).half().cuda().eval()
    with torch.no_grad():
        for layer in model.model.layers:
            a, mlp = layer.attn, layer.mlp
            for lin in (a.q_proj, a.k_proj, a.v_proj, a.o_proj) + (() if mlp is None else (mlp.gate_proj, mlp.up_proj, mlp.down_proj)):
                lin.weight.copy_(dequantize_q4(quantize_q4(lin.weight.detach())))
        model.lm_head.weight.copy_(dequantize_q4(quantize_q4(model.lm_head.weight.detach())))
    return model


def _apart(a, b):
    return float((a.float() - b.float()).norm() / b.float().norm())


def _config(**more):
    from nova_amd.skeleton import SkeletonConfig

    return SkeletonConfig(**(dict(num_hidden_layers=3, num_attention_heads=8, num_key_value_heads=2, hidden_size=512, intermediate_size=992,
                                  vocab_size=300) | more))


@pytest.mark.parametrize("paged, bound", [(PagedKVInt8TokCache, 1e-2), (PagedKVQ4Cache, 0.125)])
def test_a_decoder_over_packed_batches(paged, bound):
    """Prompts, drafts and single tokens through forward_chunks with the weights in fp16 and in 4 bits, the same values. Some
    ten roundings a layer differ, by 2^-11 / sqrt(3) of the value each: over three layers 2e-3 of the logits' norm, five
    times that allowed. Behind them an 8-bit code turns for 2% of the channels, by 1 / 127 of the largest one: nothing.
    A 4-bit code's step is a seventh of the largest channel, 2.5 / 7 = 0.36 of the rms. Inputs off by d of their rms turn
    0.8 d / 0.36 of the codes by 0.36: keys and values off by sqrt(0.29 d). The first layer's inputs are the same and its
    products off by 2^-11 / sqrt(3): d = 3e-4, 0.01 behind it. The second layer's are off by 0.01 then: 0.054 behind it; the third's
    by 0.054 at most: 0.125. (That the first bound stood at 0.03 was a mistake: it took the first layer's d for all three.)"""
    cfg = _config()
    model = _decoder(cfg)
    with pytest.raises(ValueError):
        model.use_decode_kernels(weights="q3")
    counts, prompts = [5, 1, 70], [40, 3, 0]
    g = torch.Generator().manual_seed(5)
    ids = [torch.randint(0, cfg.vocab_size, (p + 3 * n,), generator=g).cuda() for p, n in zip(prompts, counts)]
    logits = {}
    for weights in ("fp16", "q4"):
        model.use_decode_kernels(weights=weights)
        cache = paged(3, 2, D, 8, 3, 40, 12)
        at, logits[weights] = [0, 0, 0], []
        for step in range(4):
            now = prompts if step == 0 else counts
            tokens = torch.cat([x[a:a + n] for x, a, n in zip(ids, at, now)])
            plan = cache.plan_chunks(now)
            logits[weights].append(model.forward_chunks(tokens, cache, plan))
            cache.advance_chunks(plan)
            at = [a + n for a, n in zip(at, now)]
    with pytest.raises(ValueError):
        model.forward_chunks(tokens[:-1], cache, plan)
    model.use_decode_kernels(False)
    with pytest.raises(RuntimeError):
        model.forward_chunks(tokens, cache, plan)
    for a, b in zip(logits["q4"], logits["fp16"]):
        assert a.shape == b.shape and a.shape[1] == cfg.vocab_size
        assert _apart(a, b) < bound


@pytest.mark.parametrize("intermediate", [992, 0])
def test_a_decoder_of_single_tokens(intermediate):
    """One-token steps over the int8 cache, captured, eager and with fp16 weights of the same values (the bound: above)."""
    from nova_amd.decode import GraphDecoder

    cfg = _config(intermediate_size=intermediate)
    model = _decoder(cfg)
    ids = torch.randint(0, cfg.vocab_size, (1, 100), generator=torch.Generator().manual_seed(9)).cuda()
    fed = torch.randint(0, cfg.vocab_size, (6, 1, 1), generator=torch.Generator().manual_seed(10)).cuda()
    logits = {}
    for weights, captured in (("fp16", True), ("q4", True), ("q4", False)):
        model.use_decode_kernels(weights=weights)
        dec = GraphDecoder(model, max_len=256, quant="int8")
        dec.prefill(ids)
        if captured:
            dec.capture(warmup=2)
        logits[weights, captured] = []
        for token in fed:
            dec.input_ids.copy_(token)
            if captured:
                dec.step()
                out = dec.logits
            else:
                with torch.inference_mode():
                    out = dec._body()
            logits[weights, captured].append(out.clone())
    model.use_decode_kernels(False)
    for plain, replayed, eager in zip(*logits.values()):
        assert torch.equal(replayed, eager)
        assert replayed.shape == plain.shape and _apart(replayed, plain) < 1e-2


class _NoCache:
    """The caller's cache of a prompt that is all there is."""

    pos = torch.zeros(1, dtype=torch.int64)

    def update(self, k, v, layer):
        return k, v


def test_packed_steps_are_the_torch_layers():
    """forward_chunks over the int8 cache against the torch layers over whole prompts. A cached value is off by 2.5 to 3 rms / 127 /
    sqrt(12) = 0.0066 of its rms: so are a score (by that much, the query's rms being 1) and what the weights gather, 0.0093 a
    layer together, 0.016 over three; twice that, and the roundings (above), are allowed."""
    cfg = _config()
    model = _decoder(cfg)
    lens = [40, 3, 131, 1]
    ids = [torch.randint(0, cfg.vocab_size, (n,), generator=torch.Generator().manual_seed(20 + n)).cuda() for n in lens]
    _NoCache.pos = _NoCache.pos.cuda()
    with torch.no_grad():
        want = [model(x[None], past_key_values=_NoCache())[0] for x in ids]
    model.use_decode_kernels()
    cache = PagedKVInt8TokCache(3, 2, D, 8, 4, 40, 12)
    got = [[] for _ in ids]
    for at, now in (([0, 0, 0, 0], [30, 2, 64, 0]), ([30, 2, 64, 0], [10, 1, 67, 1])):
        plan = cache.plan_chunks(now)
        out = model.forward_chunks(torch.cat([x[a:a + n] for x, a, n in zip(ids, at, now)]), cache, plan)
        cache.advance_chunks(plan)
        for b, part in enumerate(out.split(now)):
            got[b].append(part)
    for w, g in zip(want, got):
        assert _apart(torch.cat(g), w) < 0.034


def test_weights_are_quantized_as_they_are_now():
    cfg = _config(num_hidden_layers=1)
    model = _decoder(cfg).use_decode_kernels(weights="q4")
    with torch.no_grad():
        model.model.layers[0].attn.v_proj.weight.neg_()
        model.lm_head.weight.mul_(2)
    model.use_decode_kernels(weights="q4")
    layer = model.model.layers[0]
    assert torch.equal(dequantize_q4(layer.q4["qkv"]), layer.w_qkv) and torch.equal(dequantize_q4(model.lm_head_q4), model.lm_head.weight)
    with pytest.raises(ValueError):
        _decoder_of(hidden_size=500)


def _decoder_of(**more):
    from nova_amd.skeleton import SkeletonForCausalLM

    return SkeletonForCausalLM(_config(**more), seed=3).half().cuda().use_decode_kernels(weights="q4")


# where one form of the product ends and the next begins (256 workgroups of passes; two tokens' parts in one product)
EDGES = [(3, 4096, 96, torch.float16), (3, 4112, 96, torch.float16), (4, 4112, 96, torch.bfloat16), (8, 2048, 160, torch.float16),
         (8, 2064, 160, torch.bfloat16), (9, 1360, 224, torch.float16), (9, 1376, 224, torch.float16), (2, 4112, 96, torch.float16),
         # tiles of a workgroup: 513 to 768 tiles of 16 rows three, more four (two of 64 tokens in two parts)
         (17, 8192, 96, torch.float16), (17, 8208, 160, torch.float16), (33, 12288, 96, torch.bfloat16), (50, 8230, 64, torch.float16),
         (64, 12304, 96, torch.float16), (40, 12304, 96, torch.float16), (64, 12310, 160, torch.bfloat16), (10, 12320, 64, torch.float16),
         # .. and of gates and ups, of half as many outputs
         (5, 16416, 96, torch.bfloat16), (20, 24576, 64, torch.float16), (20, 24608, 64, torch.bfloat16), (32, 24608, 96, torch.float16),
         (16, 24608, 64, torch.float16), (20, 16394, 64, torch.float16),
         # passes of 16 to 64 tokens of one, two, three and four tiles of outputs, with and without rest
         (48, 2560, 320, torch.bfloat16), (49, 2500, 320, torch.bfloat16), (64, 2560, 256, torch.float16), (100, 1030, 96, torch.float16),
         (40, 6144, 96, torch.float16), (128, 2100, 160, torch.bfloat16), (200, 400, 96, torch.float16), (150, 16640, 64, torch.bfloat16),
         (130, 8200, 64, torch.float16), (257, 20, 64, torch.bfloat16),
         # more inputs than a token's waves hold: passes of two, of one
         (3, 100, 2592, torch.float16), (4, 100, 5120, torch.bfloat16), (7, 530, 4096, torch.float16), (5, 40, 5152, torch.float16),
         (12, 333, 9728, torch.float16), (13, 333, 9728, torch.float16), (2, 40, 10240, torch.bfloat16), (3, 40, 10272, torch.float16)]


@pytest.mark.parametrize("tokens,n_out,n_in,dtype", EDGES)
def test_products_at_the_edges_of_their_forms(tokens, n_out, n_in, dtype):
    x, gamma = _randn((tokens, n_in), 150 + tokens, dtype=dtype).cuda(), (1 + _randn((n_in,), 151, 0.2, torch.float32)).to(dtype).cuda()
    w = quantize_q4(_randn((n_out, n_in), 152, 0.05, dtype).cuda())
    _check_product(x, w, gamma, 1e-6, None, G.rms_gemv_q4(x, w, gamma))
    if n_out % 2 == 0:
        _check_product(x, w, gamma, 1e-6, None, G.swiglu_gemv_q4(x, w, gamma), gated=True)


def test_a_step_without_tokens():
    cache = _held_with_step([70, 0], [0, 0], 8, 2, 160)
    before = cache.pages[0].clone()
    plan = cache.plan_chunks([0, 0])
    q = cache.append_chunks(plan, torch.zeros(0, 12 * D, dtype=torch.float16, device="cuda"), 0)
    assert q.shape == (0, 8, D) and cache.attend_chunks(plan, q, 0).shape == (0, 8, D)
    assert torch.equal(cache.pages[0], before)
    w = quantize_q4(_randn((48, 64), 161).cuda())
    x = torch.zeros(0, 64, dtype=torch.float16, device="cuda")
    assert G.rms_gemv_q4(x, w).shape == (0, 48) and G.swiglu_gemv_q4(x, w).shape == (0, 24)


def test_a_captured_decoder_step_follows_the_sequences():
    """forward_chunks with 4-bit weights over 4-bit pages, captured once and replayed as the sequences grow, with eager steps
    of a second cache between."""
    cfg = _config(num_hidden_layers=2)
    model = _decoder(cfg).use_decode_kernels(weights="q4")
    prompts, counts = [100, 7, 0], [1, 3, 1]
    gen = torch.Generator().manual_seed(31)
    caches = [PagedKVQ4Cache(2, 2, D, 8, 3, 20, 6) for _ in range(2)]
    first = torch.randint(0, cfg.vocab_size, (sum(prompts),), generator=gen).cuda()
    for cache in caches:
        plan = cache.plan_chunks(prompts)
        model.forward_chunks(first, cache, plan)
        cache.advance_chunks(plan)
        for b in range(3):
            cache.reserve(b, prompts[b] + 40)
    plans = [cache.plan_chunks(counts) for cache in caches]
    tokens = torch.zeros(sum(counts), dtype=torch.int64, device="cuda")
    before = [p.clone() for p in caches[0].pages]

    def step():
        logits = model.forward_chunks(tokens, caches[0], plans[0])
        caches[0].pos[:3].add_(plans[0].new)
        return logits

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()  # (loads what a capture may not)
    torch.cuda.current_stream().wait_stream(side)
    caches[0].pos[:3] = torch.tensor(prompts, device="cuda")
    for page, held in zip(caches[0].pages, before):
        page.copy_(held)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for r in range(5):
        tokens.copy_(torch.randint(0, cfg.vocab_size, tokens.shape, generator=gen).cuda())
        graph.replay()
        caches[0].note_chunks(plans[0])
        want = model.forward_chunks(tokens, caches[1], plans[1])
        caches[1].advance_chunks(plans[1])
        torch.cuda.synchronize()
        assert torch.equal(out, want), r
        assert all(torch.equal(a, b) for a, b in zip(caches[0].pages, caches[1].pages)) and torch.equal(caches[0].pos, caches[1].pos)


@pytest.mark.parametrize("tokens", [1000, 2500])
def test_products_of_many_tokens(tokens):
    x, gamma = _randn((tokens, 160), 170, dtype=torch.float16).cuda(), (1 + _randn((160,), 171, 0.2, torch.float32)).half().cuda()
    w = quantize_q4(_randn((80, 160), 172, 0.05).cuda())
    _check_product(x, w, gamma, 1e-6, None, G.rms_gemv_q4(x, w, gamma))
    _check_product(x, w, gamma, 1e-6, None, G.swiglu_gemv_q4(x, w, gamma), gated=True)


def test_captured_steps_outlive_a_change_of_the_weights_mode():
    """A captured step goes on with its 4-bit weights while the decoder runs on fp16 ones, and with new values once they are
    quantized again."""
    from nova_amd.decode import GraphDecoder

    model = _decoder(_config(num_hidden_layers=2)).use_decode_kernels(weights="q4")
    ids = torch.randint(0, 300, (1, 70), generator=torch.Generator().manual_seed(9)).cuda()
    dec = GraphDecoder(model, max_len=256, quant="int8")
    dec.prefill(ids)
    dec.capture(warmup=2)
    start = [(t, t.clone()) for t in (dec.input_ids, dec.cache.pos, dec.cache._written, dec.cache._qlen)]

    def replay():
        for t, held in start:
            t.copy_(held)
        dec.step()
        torch.cuda.synchronize()
        return dec.logits.clone()

    want = replay()
    model.use_decode_kernels(weights="fp16")
    junk = [torch.full((1 << 20,), 7, dtype=torch.uint8, device="cuda") for _ in range(16)]  # (what was freed would be taken)
    assert torch.equal(replay(), want)
    model.use_decode_kernels(weights="q4")
    assert torch.equal(replay(), want)
    with torch.no_grad():
        model.lm_head.weight.mul_(2)
    model.use_decode_kernels(weights="q4")
    assert torch.equal(replay(), want * 2) and len(junk) == 16
    w = _randn((32, 64), 180).cuda()
    held = quantize_q4(w)
    assert quantize_q4(-w, out=held) is held and torch.equal(dequantize_q4(held), -dequantize_q4(quantize_q4(w)))
    for bad in (_randn((32, 96), 181).cuda(), _randn((16, 64), 181).cuda()):
        with pytest.raises(ValueError):
            quantize_q4(bad, out=held)
