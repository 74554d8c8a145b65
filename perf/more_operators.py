"""Operators of a serving step in 4 bits, as cases to measure.

One format for weights and cache: groups of 32 values of a row share a scale of 8 significant bits,
held in fp16, and each value is a code of -7 .. 7 (two in a byte).

- ``product``: a few tokens times a 4-bit weight, with the RMSNorm before and the residual after, or as
  the first half of a SwiGLU block;
- ``append``: the stacked q/k/v projections of a batch's new tokens get each query and key head's
  RMSNorm and the rotary embedding at the token's own position; the keys and values go into pages of
  64 tokens in 4 bits, and are read back (what a caller keeps as fp16);
- ``attend``: the new tokens attend causally over everything their sequence has in its pages;
- ``read``: spans of cached tokens leave the pages as fp16, bf16 or fp32.

``own`` false: elementary torch operations in 32 bits; true: the package's entry points.
"""

import math

import torch

own = False

D, GT, GROUP = 128, 64, 32
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
THETA, EPS = 1_000_000.0, 1e-6


# ---------------------------------------------------------------- cases


def listed():
    return [
        # one token's q/k/v projection behind the input norm
        {"name": "product_qkv_1", "op": "product", "form": "plain", "tokens": 1, "out": 6144, "in": 2560, "dtype": "fp16",
         "norm": True, "residual": False},
        # a small odd adapter, five tokens: the smallest call, latency
        {"name": "product_odd_5", "op": "product", "form": "plain", "tokens": 5, "out": 333, "in": 1056, "dtype": "bf16",
         "norm": True, "residual": True},
        # the down projection of eight decoding sequences, onto the residual stream
        {"name": "product_down_8", "op": "product", "form": "plain", "tokens": 8, "out": 2560, "in": 9728, "dtype": "fp16",
         "norm": False, "residual": True},
        # one token's gate and up projections
        {"name": "product_swiglu_1", "op": "product", "form": "swiglu", "tokens": 1, "out": 9728, "in": 2560, "dtype": "fp16",
         "norm": True, "residual": False},
        # the same for forty-eight tokens of a batch, bf16
        {"name": "product_swiglu_bf16_48", "op": "product", "form": "swiglu", "tokens": 48, "out": 9728, "in": 2560,
         "dtype": "bf16", "norm": True, "residual": False},
        # twelve conversations decode one token each: a launch and a read
        {"name": "append_decode_12", "op": "append", "hq": 32, "hkv": 8, "dtype": "fp16",
         "ctx": "113,4000,777,64,1999,63,250,8190,1024,512,31,2500", "new": ",".join(["1"] * 12)},
        # three prompts of a batch, one continued; a bf16 model with seven query heads to a key head
        {"name": "append_prompts_4k", "op": "append", "hq": 28, "hkv": 4, "dtype": "bf16",
         "ctx": "0,3000,129", "new": "2048,1003,1061"},
        # a decoding batch of thirty-two
        {"name": "attend_decode_32", "op": "attend", "hq": 32, "hkv": 8,
         "ctx": ",".join(str(64 + 261 * ((7 * i) % 32)) for i in range(32)), "new": ",".join(["1"] * 32)},
        # prompts' chunks and drafted tokens beside decoding sequences
        {"name": "attend_mixed_6", "op": "attend", "hq": 32, "hkv": 8,
         "ctx": "1500,4097,700,0,6000,3333", "new": "384,1,129,257,5,1"},
        # the largest: a 2048-token chunk late in a long prompt
        {"name": "attend_2048_over_14k", "op": "attend", "hq": 32, "hkv": 8, "ctx": "14336", "new": "2048"},
        # two short sequences leave the cache: latency
        {"name": "read_short", "op": "read", "hkv": 8, "dtype": "fp16", "ctx": "200,75", "new": "200,75"},
        # a batch's contexts, spans that start and end inside pages
        {"name": "read_8_long", "op": "read", "hkv": 8, "dtype": "bf16",
         "ctx": "4600,13700,9001,6144,8191,5005,12001,11111", "new": "4600,13601,9000,6144,8127,5005,12001,11000"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["product", "product", "append", "attend", "attend", "read"])
    if op == "product":
        case = {"op": op, "form": rng.choice(["plain", "plain", "swiglu"]), "tokens": _log_int(rng, 1, 64)}
        case["in"] = GROUP * _log_int(rng, 1, 304)
        most = min(20000, 50_000_000 // case["in"])
        case["out"] = _log_int(rng, 1, most // 2 if case["form"] == "swiglu" else most)
        case["dtype"] = rng.choice(["fp16", "fp16", "bf16"])
        case["norm"] = rng.random() < 0.6
        case["residual"] = case["form"] == "plain" and rng.random() < 0.5
        return case
    nseq = _log_int(rng, 1, 40)
    case = {"op": op}
    if op == "read":
        case["hkv"] = rng.choice([1, 2, 4, 8])
        case["dtype"] = rng.choice(["fp16", "bf16", "fp32"])
        ctx = [_log_int(rng, 1, min(13000, 60000 // nseq)) for _ in range(nseq)]
        new = [rng.randint(1, c) for c in ctx]
    else:
        case["hkv"] = rng.choice([1, 2, 4, 8])
        gq = rng.choice([g for g in (1, 2, 3, 4, 5, 7, 8, 16) if g * case["hkv"] <= 32])
        case["hq"] = gq * case["hkv"]
        if rng.random() < 0.5:  # a decoding or verifying batch: the same few tokens each
            new = [rng.randint(1, 8)] * nseq
        else:
            new = [_log_int(rng, 1, max(1, 2048 // nseq)) for _ in range(nseq)]
        room = min(14336, 160000 // nseq)
        ctx = [0 if rng.random() < 0.15 else _log_int(rng, 1, room) for _ in range(nseq)]
        if op == "append":
            case["dtype"] = rng.choice(["fp16", "bf16", "fp32"])
    case["ctx"] = ",".join(map(str, ctx))
    case["new"] = ",".join(map(str, new))
    return case


def _spans(case):
    """Per sequence: tokens its pages hold, the first token of the span, the span's tokens (the new ones; read:
    a stretch from the middle of the context)."""
    ctx, new = [int(x) for x in case["ctx"].split(",")], [int(x) for x in case["new"].split(",")]
    if case["op"] == "read":
        return ctx, [(c - n) // 2 for c, n in zip(ctx, new)], new
    return [c + n for c, n in zip(ctx, new)], ctx, new


# ---------------------------------------------------------------- the format


def _quantize(x):
    """Codes + 8 of ``x`` ``[.., n]`` packed ``[.., n / 2]`` and scales fp16 ``[.., n / 32]``."""
    x = x.float().unflatten(-1, (-1, GROUP))
    scale = (x.abs().amax(-1) / 7.0).clamp_min(2.0 ** -24).to(torch.bfloat16).to(torch.float16)
    code = ((x / scale.float()[..., None]).round().clamp(-7, 7) + 8).to(torch.uint8).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale


def _values(codes, scales):
    """What packed codes and their scales stand for, in fp32."""
    code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float() - 8
    return (code.unflatten(-1, (-1, GROUP)) * scales.float()[..., None]).flatten(-2)


# ---------------------------------------------------------------- inputs


def _randn(shape, seed, k):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed * 7919 + k), device="cuda")


def _gamma(n, seed, k, dtype):
    return (1.0 + 0.2 * _randn((n,), seed, k)).to(dtype)


def _product_inputs(case, seed):
    t, n_out, n_in, dt = case["tokens"], case["out"], case["in"], DTYPES[case["dtype"]]
    rows = 2 * n_out if case["form"] == "swiglu" else n_out
    w = _randn((rows, n_in), seed, 0)
    w[:, 3::61] *= 4.0  # input features with larger weights
    return {
        "w": (w * n_in ** -0.5).to(dt),
        "x": (_randn((t, n_in), seed, 1) * (3.0 if case["norm"] else 0.6)).to(dt),
        "gamma": _gamma(n_in, seed, 2, dt) if case["norm"] else None,
        "residual": _randn((t, n_out), seed, 3).to(dt) if case["residual"] else None,
    }


def _prepare_product(case, seed):
    state = {"op": "product", "form": case["form"], **_product_inputs(case, seed)}
    w = state.pop("w")
    if own:
        from nova_amd.q4 import quantize_q4

        state["w"] = quantize_q4(w)
    else:
        state["codes"], state["scales"] = _quantize(w)
    return state


def _prompts(case, seed, b, n):
    """Keys and values ``[1, H_kv, n, 128]`` of sequence b's first n tokens."""
    shape = (1, case["hkv"], n, D)
    k, v = _randn(shape, seed, 100 + 2 * b), _randn(shape, seed, 101 + 2 * b) * 0.7
    k[..., 5::37] *= 3.0  # a few channels stand out, as keys' do
    return k.half(), v.half()


def prepare(case, seed):
    op = case["op"]
    if op == "product":
        return _prepare_product(case, seed)
    hkv = case["hkv"]
    total, start, new = _spans(case)
    nseq, T = len(new), sum(new)
    need = [-(-t // GT) for t in total]
    n_pages, per_seq = sum(need) + 3, max(need) + 1
    order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).tolist()
    held = total if op != "append" else [0] * nseq  # (an append reads nothing of what is there)
    state = {"op": op, "hkv": hkv, "T": T}
    if own:
        from nova_amd.paged import PagedKVQ4Cache

        cache = PagedKVQ4Cache(1, hkv, D, case.get("hq", hkv), nseq, n_pages, per_seq)
        cache._free = order[::-1]  # pages are handed out from the end
        for b in range(nseq):
            cache.reserve(b, total[b])
            if held[b]:
                cache.prefill(b, 0, *_prompts(case, seed, b, held[b]))
            cache.pool.set_length(b, start[b] if op != "read" else total[b])
        cache.pos[:nseq] = torch.tensor(start if op != "read" else total, device="cuda")
        state["cache"] = cache
        state["plan"] = cache.plan_chunks(new) if op != "read" else cache.plan_read(new, start)
    else:
        table = torch.zeros((nseq, per_seq), dtype=torch.int64)
        pool = [torch.zeros((n_pages, hkv, GT, w), dtype=t, device="cuda")
                for w, t in ((D // 2, torch.uint8), (D // GROUP, torch.float16)) * 2]  # K codes and scales, V's
        at = 0
        for b, n in enumerate(need):
            ids = torch.tensor(order[at:at + n], dtype=torch.int64)
            table[b, :n] = ids
            at += n
            if held[b]:
                for which, x in enumerate(_prompts(case, seed, b, held[b])):
                    padded = torch.zeros((hkv, n * GT, D), dtype=torch.float16, device="cuda")
                    padded[:, :held[b]] = x[0]
                    for part, y in enumerate(_quantize(padded)):
                        pool[2 * which + part][ids.cuda()] = y.unflatten(1, (n, GT)).transpose(0, 1)
        # packed token t: its sequence, its row among the sequence's new tokens, its position
        seq = torch.repeat_interleave(torch.arange(nseq), torch.tensor(new))
        row = torch.arange(T) - torch.tensor([sum(new[:b]) for b in range(nseq)])[seq]
        state |= {"pool": pool, "table": table.cuda(), "nseq": nseq, "most": max(total), "rows": max(new)}
        state |= {"seq": seq.cuda(), "row": row.cuda(), "pos": (row + torch.tensor(start)[seq]).cuda()}
    if op == "append":
        hq, dt = case["hq"], DTYPES[case["dtype"]]
        state["hq"] = hq
        state["qkv"] = (_randn((T, (hq + 2 * hkv) * D), seed, 4) * 0.9).to(dt)
        state["q_gamma"], state["k_gamma"] = _gamma(D, seed, 5, dt), _gamma(D, seed, 6, dt)
        state["inv_freq"] = (THETA ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)).float().cuda()
    elif op == "attend":
        state["hq"] = case["hq"]
        state["q"] = (_randn((T, case["hq"], D), seed, 7) * 1.5).half()
    else:
        state["dtype"] = DTYPES[case["dtype"]]
    return state


# ---------------------------------------------------------------- one pass


def run(state):
    op = state["op"]
    if not own:
        return {"product": _product, "append": _append, "attend": _attend, "read": _read}[op](state)
    if op == "product":
        from nova_amd import gemv

        if state["form"] == "swiglu":
            return gemv.swiglu_gemv_q4(state["x"], state["w"], state["gamma"], EPS)
        return gemv.rms_gemv_q4(state["x"], state["w"], state["gamma"], EPS, state["residual"])
    cache, plan = state["cache"], state["plan"]
    if op == "append":
        q = cache.append_chunks(plan, state["qkv"], 0, q_gamma=state["q_gamma"], k_gamma=state["k_gamma"], eps=EPS,
                                inv_freq=state["inv_freq"])
        return (q, *cache.read(plan, 0))
    if op == "attend":
        return cache.attend_chunks(plan, state["q"], 0)
    return cache.read(plan, 0, state["dtype"])


def _rms(x, gamma):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * gamma.float()


def _product(s):
    x = s["x"].float()
    if s["gamma"] is not None:
        x = _rms(x, s["gamma"])
    y = x @ _values(s["codes"], s["scales"]).T
    if s["form"] == "swiglu":
        gate, up = y.chunk(2, -1)
        y = gate / (1 + torch.exp(-gate)) * up
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["x"].dtype)


def _rotate(x, cos, sin):
    lo, hi = x[..., :D // 2], x[..., D // 2:]
    return torch.cat((lo * cos - hi * sin, hi * cos + lo * sin), -1)


def _append(s):
    hq, hkv, T = s["hq"], s["hkv"], s["T"]
    x = s["qkv"].float().view(T, hq + 2 * hkv, D)
    angle = s["pos"].double()[:, None] * s["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    q = _rotate(_rms(x[:, :hq], s["q_gamma"]), cos, sin).half()
    k = _rotate(_rms(x[:, hq:hq + hkv], s["k_gamma"]), cos, sin)
    page, slot = s["table"][s["seq"], s["pos"] // GT], s["pos"] % GT
    for which, new in enumerate((k, x[:, hq + hkv:])):
        s["pool"][2 * which][page, :, slot], s["pool"][2 * which + 1][page, :, slot] = _quantize(new)
    return (q, *(_taken(s, which, torch.float16) for which in (0, 1)))


def _taken(s, which, dtype):
    page, slot = s["table"][s["seq"], s["pos"] // GT], s["pos"] % GT
    return _values(*(x[page, :, slot] for x in s["pool"][2 * which:2 * which + 2])).to(dtype)


def _attend(s):
    """Every sequence padded to the longest and to the most new tokens, in one product each way."""
    hq, hkv, nseq, most, rows = s["hq"], s["hkv"], s["nseq"], s["most"], s["rows"]
    gq, groups = hq // hkv, -(-most // GT)
    q = torch.zeros((nseq, rows, hq, D), device="cuda")
    q[s["seq"], s["row"]] = s["q"].float()
    at = torch.full((nseq, rows), -1, dtype=torch.int64, device="cuda")
    at[s["seq"], s["row"]] = s["pos"]
    q = q.view(nseq, rows, hkv, gq, D).permute(0, 2, 3, 1, 4).reshape(nseq * hkv, gq * rows, D)
    k, v = (_whole(s, which, groups) for which in (0, 1))
    scores = torch.bmm(q, k.transpose(1, 2).contiguous()).view(nseq, hkv, gq, rows, groups * GT)
    scores.mul_(1.0 / math.sqrt(D))
    scores.masked_fill_((torch.arange(groups * GT, device="cuda") > at[..., None])[:, None, None], -math.inf)
    scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = torch.bmm(scores.view(nseq * hkv, gq * rows, groups * GT), v).view(nseq, hkv, gq, rows, D) / total
    return out.permute(0, 3, 1, 2, 4).reshape(nseq, rows, hq, D)[s["seq"], s["row"]].half()


def _whole(s, which, groups):
    """``[sequences x H_kv, tokens, 128]`` of one tensor."""
    page = s["table"][:, :groups]
    x = _values(*(y[page] for y in s["pool"][2 * which:2 * which + 2]))
    return x.transpose(1, 2).reshape(-1, groups * GT, D)


def _read(s):
    return tuple(_taken(s, which, s["dtype"]) for which in (0, 1))


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    if case["op"] == "product":
        t, n_out, n_in = case["tokens"], case["out"], case["in"]
        rows = 2 * n_out if case["form"] == "swiglu" else n_out
        moved = rows * (n_in // 2 + n_in // GROUP * 2) + 2 * t * (n_in + n_out * (2 if case["residual"] else 1))
        return {"bytes": moved + (2 * n_in if case["norm"] else 0), "flops": 2 * t * rows * n_in}
    total, start, new = _spans(case)
    hkv, T, row = case["hkv"], sum(new), D // 2 + 2 * (D // GROUP)  # a token's bytes of a tensor and KV head
    if case["op"] == "append":
        hq, size = case["hq"], DTYPES[case["dtype"]].itemsize
        moved = T * ((hq + 2 * hkv) * D * size + hq * D * 2 + hkv * 2 * row)  # in, q out, pages
        moved += T * hkv * 2 * (row + D * 2)  # read back
        return {"bytes": moved, "flops": 12 * T * (hq + 2 * hkv) * D}
    if case["op"] == "attend":
        hq = case["hq"]
        pairs = sum(n * s + n * (n + 1) // 2 for s, n in zip(start, new))
        return {"bytes": 2 * T * hq * D * 2 + sum(total) * hkv * 2 * row, "flops": 4 * D * hq * pairs}
    size = DTYPES[case["dtype"]].itemsize
    return {"bytes": T * hkv * 2 * (row + D * size), "flops": 2 * T * hkv * 2 * D}


# ---------------------------------------------------------------- the definition in 64 bits


def _grid(x):
    """The nearest multiples of their group's scale, in 64 bits, for ``x`` ``[.., n]`` with n a multiple of 32."""
    g = x.double().reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    unit = torch.clamp(g.abs().max(-1, keepdim=True).values / 7, min=0.5 ** 24)
    m, e = torch.frexp(unit)
    unit = torch.ldexp(torch.round(m * 256) / 256, e).half().double()
    return (torch.clamp(torch.round(g / unit), -7, 7) * unit).reshape(x.shape)


def exact(case, seed):
    f64 = torch.float64
    if case["op"] == "product":
        s = _product_inputs(case, seed)
        x = s["x"].to(f64)
        if s["gamma"] is not None:
            x = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * s["gamma"].to(f64)
        y = torch.matmul(x, _grid(s["w"]).t())
        if case["form"] == "swiglu":
            y = y[:, :case["out"]] * torch.sigmoid(y[:, :case["out"]]) * y[:, case["out"]:]
        return y if s["residual"] is None else y + s["residual"].to(f64)
    total, start, new = _spans(case)
    hkv = case["hkv"]
    if case["op"] == "append":
        hq, dt, T = case["hq"], DTYPES[case["dtype"]], sum(new)
        x = (_randn((T, (hq + 2 * hkv) * D), seed, 4) * 0.9).to(dt).to(f64).reshape(T, -1, D)
        inv = (THETA ** (-torch.arange(0, D, 2, dtype=f64) / D)).float().cuda().to(f64)
        pos = torch.cat([torch.arange(a, a + n) for a, n in zip(start, new)]).cuda().to(f64)

        def turned(h, k):
            h = h / (h.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt() * _gamma(D, seed, k, dt).to(f64)
            z = torch.complex(h[..., :D // 2], h[..., D // 2:])
            a = pos[:, None] * inv[None]
            z = z * torch.polar(torch.ones_like(a), a)[:, None]
            return torch.cat((z.real, z.imag), -1)

        return (turned(x[:, :hq], 5), _grid(turned(x[:, hq:hq + hkv], 6)), _grid(x[:, hq + hkv:]))
    if case["op"] == "read":
        outs = [[], []]
        for b, (a, n) in enumerate(zip(start, new)):
            for which, x in enumerate(_prompts(case, seed, b, total[b])):
                outs[which].append(_grid(x[0, :, a:a + n]).transpose(0, 1))
        return tuple(torch.cat(o) for o in outs)
    hq, out, at = case["hq"], [], 0
    queries = (_randn((sum(new), hq, D), seed, 7) * 1.5).half().to(f64)
    for b, n in enumerate(new):
        k, v = (_grid(x[0]) for x in _prompts(case, seed, b, total[b]))
        hidden = torch.ones((n, total[b]), dtype=torch.bool, device="cuda").triu(start[b] + 1)
        heads = []
        for i in range(hq):
            w = queries[at:at + n, i] @ k[i // (hq // hkv)].T.contiguous() / D ** 0.5
            heads.append(torch.softmax(w.masked_fill(hidden, -math.inf), -1) @ v[i // (hq // hkv)])
        out.append(torch.stack(heads, 1))
        at += n
    return torch.cat(out)
