"""Operators of a serving step over the paged per-token cache, as cases to measure.

A batch of sequences of different lengths brings new tokens (a prompt's chunk, a decode token, a
few drafted tokens) in one packed tensor:

- ``append``: the stacked q/k/v projections of the new tokens get each query and key head's
  RMSNorm and the rotary embedding at the token's own position; the keys and values are quantized
  into their pages. The new keys and values are then read back (what a caller keeps as fp16).
- ``attend``: the new tokens attend causally over everything their sequence has in its pages.
- ``read``: spans of cached tokens leave the pages as fp16, bf16 or fp32, from the per-token
  symmetric pages or the int8t64 ones (whole groups from pages, newer tokens from the ring).

``own`` false: elementary torch operations in 32 bits; true: the package's entry points.
"""

import math

import torch

own = False

D, GT = 128, 64
CODES = GT * D
PAGE_TOK, PAGE_T64 = 2 * CODES + 2 * GT * 2, 2 * CODES + 4 * D * 2
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
THETA, EPS = 1_000_000.0, 1e-6


# ---------------------------------------------------------------- cases


def listed():
    return [
        # twelve conversations decode one token each: the smallest call, a launch and a read
        {"name": "append_decode_12", "op": "append", "hq": 32, "hkv": 8, "dtype": "fp16",
         "ctx": "113,4000,777,64,1999,63,250,8190,1024,512,31,2500", "new": ",".join(["1"] * 12)},
        # three prompts of a batch, one continued: an ordinary prefill step
        {"name": "append_prompts_4k", "op": "append", "hq": 32, "hkv": 8, "dtype": "fp16",
         "ctx": "0,3000,129", "new": "2048,1003,1061"},
        # a bf16 model with seven query heads to a key head
        {"name": "append_bf16_28_heads", "op": "append", "hq": 28, "hkv": 4, "dtype": "bf16",
         "ctx": "0,17,16001,640", "new": "700,33,1,295"},
        # drafted tokens verified: four a sequence over short and middle contexts
        {"name": "attend_verify_8x4", "op": "attend", "hq": 32, "hkv": 8,
         "ctx": "200,1000,64,3999,517,1300,2222,90", "new": ",".join(["4"] * 8)},
        # a decoding batch of thirty-two
        {"name": "attend_decode_32", "op": "attend", "hq": 32, "hkv": 8,
         "ctx": ",".join(str(64 + 261 * ((7 * i) % 32)) for i in range(32)), "new": ",".join(["1"] * 32)},
        # prompts' chunks beside decoding sequences
        {"name": "attend_mixed_6", "op": "attend", "hq": 32, "hkv": 8,
         "ctx": "1500,4097,700,0,6000,3333", "new": "384,1,129,257,5,1"},
        # prompts from nothing, seven query heads to a key head
        {"name": "attend_prompts_28_heads", "op": "attend", "hq": 28, "hkv": 4, "ctx": "0,0,0", "new": "1200,801,1057"},
        # the largest: a 2048-token chunk late in a long prompt
        {"name": "attend_2048_over_14k", "op": "attend", "hq": 32, "hkv": 8, "ctx": "14336", "new": "2048"},
        # two short sequences leave the cache: latency
        {"name": "read_tok_short", "op": "read", "format": "tok", "hkv": 8, "dtype": "fp16", "ctx": "200,75", "new": "200,75"},
        # a batch's whole contexts
        {"name": "read_tok_8_long", "op": "read", "format": "tok", "hkv": 8, "dtype": "bf16",
         "ctx": "4600,13700,9001,6144,8191,5005,12001,11111", "new": "4600,13700,9001,6144,8191,5005,12001,11111"},
        # int8t64 pages and rings, spans that start and end inside groups
        {"name": "read_t64_ragged", "op": "read", "format": "t64", "hkv": 8, "dtype": "fp32",
         "ctx": "2100,333,4097,64,31", "new": "2000,333,3001,64,20"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "read"])
    nseq = _log_int(rng, 1, 40)
    case = {"op": op}
    if op == "read":
        case["format"] = rng.choice(["tok", "t64"])
        case["hkv"] = rng.choice([1, 2, 4, 8])
        case["dtype"] = rng.choice(["fp16", "bf16", "fp32"])
        most = min(13000, 60000 // nseq)
        ctx = [_log_int(rng, 1, most) for _ in range(nseq)]
        new = [rng.randint(1, c) for c in ctx]
    else:
        case["hkv"] = rng.choice([1, 2, 4, 8])
        gq = rng.choice([g for g in (1, 2, 3, 4, 5, 7, 8, 16) if g * case["hkv"] <= 32])
        case["hq"] = gq * case["hkv"]
        most = max(1, 2048 // nseq)
        if rng.random() < 0.5:  # a decoding or verifying batch: the same few tokens each
            n = rng.randint(1, 8)
            new = [n] * nseq
        else:
            new = [_log_int(rng, 1, most) for _ in range(nseq)]
        room = min(14336, 160000 // nseq)
        ctx = [rng.choice([0, _log_int(rng, 1, room)]) if rng.random() < 0.3 else _log_int(rng, 1, room) for _ in range(nseq)]
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
        start = [(c - n) // 2 for c, n in zip(ctx, new)]
        return ctx, start, new
    return [c + n for c, n in zip(ctx, new)], ctx, new


# ---------------------------------------------------------------- inputs


def _gen(seed, k):
    return torch.Generator(device="cuda").manual_seed(seed * 7919 + k)


def _tok_pages(n_pages, hkv, seed):
    """A pool whose pages all hold quantized normal keys and values (unowned ones too: other sequences')."""
    pages = torch.empty((n_pages, hkv, PAGE_TOK), dtype=torch.uint8, device="cuda")
    for which in (0, 1):
        x = torch.randn((n_pages, hkv, GT, D), generator=_gen(seed, which), device="cuda")
        x[..., 5::37] *= 3.0  # a few channels stand out, as keys' and values' do
        scale = (x.abs().amax(-1) / 127.0).clamp_min(1e-8)
        codes = (x / scale[..., None]).round().clamp(-127, 127).to(torch.int8)
        pages[:, :, which * CODES:(which + 1) * CODES] = codes.reshape(n_pages, hkv, CODES).view(torch.uint8)
        at = 2 * CODES + which * 2 * GT
        pages[:, :, at:at + 2 * GT] = scale.to(torch.float16).view(torch.uint8)
    return pages


def _t64_pages(n_pages, hkv, seed):
    g = _gen(seed, 2)
    pages = torch.empty((n_pages, hkv, PAGE_T64), dtype=torch.uint8, device="cuda")
    pages[:, :, :2 * CODES] = torch.randint(0, 256, (n_pages, hkv, 2 * CODES), generator=g, device="cuda", dtype=torch.uint8)
    step = torch.rand((n_pages, hkv, 2, D), generator=g, device="cuda") * 0.02 + 0.005
    low = -step * (100 + 55 * torch.rand((n_pages, hkv, 2, D), generator=g, device="cuda"))
    rulers = torch.stack([step, low], dim=3).to(torch.float16)  # [.., K V, step min, D]
    pages[:, :, 2 * CODES:] = rulers.reshape(n_pages, hkv, 4 * D).view(torch.uint8)
    return pages


def prepare(case, seed):
    op, hkv = case["op"], case["hkv"]
    total, start, new = _spans(case)
    nseq, T = len(new), sum(new)
    tok = case.get("format", "tok") == "tok"
    need = [-(-t // GT) for t in total]
    n_pages, per_seq = sum(need) + 3, max(need) + 1
    order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).tolist()
    state = {"op": op, "hkv": hkv, "tok": tok, "T": T}
    pages = (_tok_pages if tok else _t64_pages)(n_pages, hkv, seed)
    rings = None if tok else (torch.randn((nseq, hkv, 2, GT, D), generator=_gen(seed, 3), device="cuda") * 0.7).half()

    table = torch.full((nseq, per_seq), -1, dtype=torch.int64)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(order[at:at + n])
        at += n
    if own:
        from nova_amd.paged import PagedKVInt8Cache, PagedKVInt8TokCache

        cache = (PagedKVInt8TokCache if tok else PagedKVInt8Cache)(1, hkv, D, case.get("hq", hkv), nseq, n_pages, per_seq)
        cache._free = order[::-1]  # pages are handed out from the end
        cache.pages[0].copy_(pages)
        if rings is not None:
            cache.rings[0].copy_(rings)
        held = start if op != "read" else total
        for b in range(nseq):
            cache.reserve(b, total[b])
            cache.pool.set_length(b, held[b])
        cache.pos[:nseq] = torch.tensor(held, device="cuda")
        state["cache"] = cache
        state["plan"] = cache.plan_chunks(new) if op != "read" else cache.plan_read(new, start)
        del pages
    else:
        state |= {"pages": pages, "rings": rings, "table": table.to("cuda"), "nseq": nseq, "most": max(total), "rows": max(new)}
        # packed token t: its sequence, its row among the sequence's new tokens, its position
        seq = torch.repeat_interleave(torch.arange(nseq), torch.tensor(new))
        row = torch.arange(T) - torch.tensor([sum(new[:b]) for b in range(nseq)])[seq]
        state["seq"], state["row"] = seq.to("cuda"), row.to("cuda")
        state["pos"] = (row + torch.tensor(start)[seq]).to("cuda")
        state["length"] = torch.tensor(total, device="cuda")
    if op == "append":
        hq, dt = case["hq"], DTYPES[case["dtype"]]
        state["hq"] = hq
        state["qkv"] = (torch.randn((T, (hq + 2 * hkv) * D), generator=_gen(seed, 4), device="cuda") * 0.9).to(dt)
        for k, name in ((5, "q_gamma"), (6, "k_gamma")):
            state[name] = (1.0 + 0.2 * torch.randn(D, generator=_gen(seed, k), device="cuda")).to(dt)
        inv = THETA ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
        state["inv_freq"] = inv.to(torch.float32).to("cuda")
    elif op == "attend":
        state["hq"] = case["hq"]
        state["q"] = (torch.randn((T, case["hq"], D), generator=_gen(seed, 7), device="cuda") * 1.5).half()
    else:
        state["dtype"] = DTYPES[case["dtype"]]
    return state


# ---------------------------------------------------------------- one pass


def run(state):
    if own:
        cache, plan = state["cache"], state["plan"]
        if state["op"] == "append":
            q = cache.append_chunks(plan, state["qkv"], 0, q_gamma=state["q_gamma"], k_gamma=state["k_gamma"], eps=EPS,
                                    inv_freq=state["inv_freq"])
            return (q, *cache.read(plan, 0))
        if state["op"] == "attend":
            return cache.attend_chunks(plan, state["q"], 0)
        return cache.read(plan, 0, state["dtype"])
    return {"append": _append, "attend": _attend, "read": _read}[state["op"]](state)


def _codes(pages, which):
    """The codes of one tensor as ``[pages, H_kv, 64, 128]``, a view."""
    return pages[:, :, which * CODES:(which + 1) * CODES].unflatten(2, (GT, D))


def _scales(pages, which):
    """The per-token scales of one tensor as ``[pages, H_kv, 64]``, a view."""
    return pages.view(torch.float16)[:, :, CODES + which * GT:CODES + (which + 1) * GT]


def _rms(x, gamma):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * gamma.float()


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
    _store(s["pages"], 0, page, slot, k)
    _store(s["pages"], 1, page, slot, x[:, hq + hkv:])
    return (q, _taken(s["pages"], 0, page, slot, torch.float16), _taken(s["pages"], 1, page, slot, torch.float16))


def _store(pages, which, page, slot, x):
    scale = (x.abs().amax(-1) / 127.0).clamp_min(1e-8)
    codes = (x / scale[..., None]).round().clamp(-127, 127).to(torch.int8)
    _codes(pages, which).view(torch.int8)[page, :, slot] = codes
    _scales(pages, which)[page, :, slot] = scale.to(torch.float16)


def _taken(pages, which, page, slot, dtype):
    codes = _codes(pages, which).view(torch.int8)[page, :, slot]
    return (codes.float() * _scales(pages, which)[page, :, slot].float()[..., None]).to(dtype)


def _attend(s):
    """Every sequence padded to the longest and to the most new tokens, in one product each way."""
    hq, hkv, nseq, most, rows = s["hq"], s["hkv"], s["nseq"], s["most"], s["rows"]
    gq, groups = hq // hkv, -(-most // GT)
    page = s["table"][:, :groups].clamp_min(0)
    q = torch.zeros((nseq, rows, hq, D), device="cuda")
    q[s["seq"], s["row"]] = s["q"].float()
    at = torch.full((nseq, rows), -1, dtype=torch.int64, device="cuda")
    at[s["seq"], s["row"]] = s["pos"]
    q = q.view(nseq, rows, hkv, gq, D).permute(0, 2, 3, 1, 4).reshape(nseq * hkv, gq * rows, D)
    k, v = (_whole(s["pages"], which, page) for which in (0, 1))
    scores = torch.bmm(q, k.transpose(1, 2).contiguous()).view(nseq, hkv, gq, rows, groups * GT)
    scores.mul_(1.0 / math.sqrt(D))
    scores.masked_fill_((torch.arange(groups * GT, device="cuda") > at[..., None])[:, None, None], -math.inf)
    scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = torch.bmm(scores.view(nseq * hkv, gq * rows, groups * GT), v).view(nseq, hkv, gq, rows, D) / total
    return out.permute(0, 3, 1, 2, 4).reshape(nseq, rows, hq, D)[s["seq"], s["row"]].half()


def _whole(pages, which, page):
    """``[sequences x H_kv, tokens, 128]`` of one tensor, dequantized."""
    x = _codes(pages, which).view(torch.int8)[page].float() * _scales(pages, which)[page].float()[..., None]
    nseq, groups, hkv = x.shape[:3]
    return x.transpose(1, 2).reshape(nseq * hkv, groups * GT, D)


def _read(s):
    pos, seq, dtype = s["pos"], s["seq"], s["dtype"]
    page, slot = s["table"][seq, pos // GT], pos % GT
    if s["tok"]:
        return tuple(_taken(s["pages"], which, page, slot, dtype) for which in (0, 1))
    newer = (pos // GT >= s["length"][seq] // GT)[:, None, None]  # still in the ring
    rulers = s["pages"].view(torch.float16)[:, :, CODES:].unflatten(2, (4, D))[page]  # kst kmn vst vmn
    out = []
    for which in (0, 1):
        x = _codes(s["pages"], which)[page, :, slot].float() * rulers[:, :, 2 * which].float() + rulers[:, :, 2 * which + 1].float()
        out.append(torch.where(newer, s["rings"][seq, :, which, slot].float(), x).to(dtype))
    return tuple(out)


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    total, start, new = _spans(case)
    hkv, T = case["hkv"], sum(new)
    if case["op"] == "append":
        hq, size = case["hq"], DTYPES[case["dtype"]].itemsize
        moved = T * ((hq + 2 * hkv) * D * size + hq * D * 2 + hkv * 2 * (D + 2))  # in, q out, pages
        moved += T * hkv * 2 * (D + 2 + D * 2)  # read back
        return {"bytes": moved, "flops": 12 * T * (hq + 2 * hkv) * D}
    if case["op"] == "attend":
        hq = case["hq"]
        pairs = sum(n * s + n * (n + 1) // 2 for s, n in zip(start, new))
        return {"bytes": 2 * T * hq * D * 2 + sum(total) * hkv * 2 * (D + 2), "flops": 4 * D * hq * pairs}
    size = DTYPES[case["dtype"]].itemsize
    if case["format"] == "tok":
        source = T * hkv * 2 * (D + 2)
    else:  # a span's groups bring their rulers whole
        paged = [max(0, min(s + n, t // GT * GT) - s) for t, s, n in zip(total, start, new)]
        groups = sum((s + p - 1) // GT - s // GT + 1 for s, p in zip(start, paged) if p)
        source = hkv * (sum(paged) * 2 * D + groups * 8 * D + (T - sum(paged)) * 4 * D)
    return {"bytes": source + T * hkv * 2 * D * size, "flops": 2 * T * hkv * 2 * D}


# ---------------------------------------------------------------- the definition in 64 bits


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    total, start, new = _spans(case)
    hkv, f64 = case["hkv"], torch.float64
    table, pages = s["table"], s["pages"]

    def cached(b, which):
        """Sequence b's keys or values as ``[H_kv, tokens, 128]`` in 64 bits, from the bytes of its pages."""
        rows = pages[table[b, :-(-total[b] // GT)]]
        codes = rows[:, :, which * CODES:(which + 1) * CODES].contiguous()
        if s["tok"]:
            sc = rows[:, :, 2 * CODES + which * 128:2 * CODES + (which + 1) * 128].contiguous().view(torch.float16)
            x = codes.view(torch.int8).to(f64).reshape(*codes.shape[:2], GT, D) * sc.to(f64).unsqueeze(-1)
        else:
            r = rows[:, :, 2 * CODES + which * 512:2 * CODES + (which + 1) * 512].contiguous().view(torch.float16).to(f64)
            x = codes.to(f64).reshape(*codes.shape[:2], GT, D) * r[:, :, None, :D] + r[:, :, None, D:]
        return x.permute(1, 0, 2, 3).reshape(hkv, -1, D)

    if case["op"] == "append":
        hq = case["hq"]
        x = s["qkv"].to(f64).reshape(-1, hq + 2 * hkv, D)

        def turned(h, gamma):
            h = h / (h.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt() * gamma.to(f64)
            z = torch.complex(h[..., :D // 2], h[..., D // 2:])
            a = s["pos"].to(f64)[:, None] * s["inv_freq"].to(f64)[None]
            z = z * torch.polar(torch.ones_like(a), a)[:, None]
            return torch.cat((z.real, z.imag), -1)

        def held(h):
            unit = torch.clamp(h.abs().max(-1, keepdim=True).values / 127, min=1e-8)
            return torch.clamp(torch.round(h / unit), -127, 127) * unit.half().to(f64)

        return (turned(x[:, :hq], s["q_gamma"]), held(turned(x[:, hq:hq + hkv], s["k_gamma"])), held(x[:, hq + hkv:]))
    if case["op"] == "read":
        outs = []
        for which in (0, 1):
            parts = []
            for b, (t, a, n) in enumerate(zip(total, start, new)):
                x = cached(b, which)[:, :t]
                if not s["tok"]:
                    whole = t // GT * GT
                    x = torch.cat((x[:, :whole], s["rings"][b, :, which, :t - whole].to(f64)), 1)
                parts.append(x[:, a:a + n].transpose(0, 1))
            outs.append(torch.cat(parts))
        return tuple(outs)
    hq, out, at = case["hq"], [], 0
    for b, n in enumerate(new):
        k, v = cached(b, 0)[:, :total[b]], cached(b, 1)[:, :total[b]]
        hidden = torch.ones((n, total[b]), dtype=torch.bool, device="cuda").triu(start[b] + 1)
        heads = []
        for i in range(hq):
            w = s["q"][at:at + n, i].to(f64) @ k[i // (hq // hkv)].T.contiguous() / D ** 0.5
            w = torch.softmax(w.masked_fill(hidden, -math.inf), -1)
            heads.append(w @ v[i // (hq // hkv)])
        out.append(torch.stack(heads, 1))
        at += n
    return torch.cat(out)
