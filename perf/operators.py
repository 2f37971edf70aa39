"""The operators between a layer's qkv projection and its output projection, for a key/value cache held in MXFP4: what is
measured of them, their plain forms in elementary torch operations, and their definitions in 64 bits.

Every case is a dict of plain values; ``op`` says what one pass is:

* ``rope``    norm of every query and key head and rotation by position (``qk_norm_rope``)
* ``append``  rotated (and normed) keys, and values, into a paged cache of E2M1 codes and E8M0 scales, the queries' norm and
              rotation in the same call where the case has them (``append_kv_mxfp4``), then the tokens' cached values read back
              (``gather_kv_mxfp4``)
* ``attend``  attention of a batch's new tokens over their sequences' cached keys and values (``attention_mxfp4``)

The cache is four tensors: codes ``[pages, kv_heads, page, D/2]`` and scale bytes ``[pages, kv_heads, page, D/32]`` of the keys,
and the same of the values.
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-6
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)      # E2M1 magnitudes by code
MAX_PAIRS = 2.1e9           # query-key pairs over all heads of a drawn prompt; the largest listed one has 2.15e9
MAX_CACHED = 2.6e8          # cached tokens * kv_heads * D of a drawn decode batch; the largest listed one has 2.7e8


# ---- cases -----------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one sequence, one token: latency
        {"name": "rope_decode_1", "op": "rope", "tokens": 1, "hq": 32, "hkv": 8, "d": 128, "rot": 128, "norm": True, "neighbours": False},
        # a prompt of 8192 tokens, strided heads of a packed projection
        {"name": "rope_prompt_8192", "op": "rope", "tokens": 8192, "hq": 32, "hkv": 8, "d": 128, "rot": 128, "norm": True, "neighbours": False},
        # one token of each of 64 sequences, queries in the same call
        {"name": "append_decode_64", "op": "append", "tokens": 64, "hq": 32, "hkv": 8, "d": 128, "rot": 128, "norm": True, "neighbours": False,
         "page": 64, "padding": 0},
        # a prompt of 8192 tokens, short heads
        {"name": "append_prompt_8192", "op": "append", "tokens": 8192, "hq": 64, "hkv": 8, "d": 64, "rot": 64, "norm": False, "neighbours": False,
         "page": 128, "padding": 0},
        # a ragged batch filled up with tokens that are not stored, keys and values alone, half of the channels rotated by neighbours
        {"name": "append_odd_777", "op": "append", "tokens": 777, "hq": 0, "hkv": 8, "d": 128, "rot": 64, "norm": False, "neighbours": True,
         "page": 16, "padding": 7},
        # one short sequence, one token: latency
        {"name": "attend_decode_1x300", "op": "attend", "batch": 1, "ctx": 300, "spread": 0.0, "new": 1, "mixed": False, "hq": 32, "hkv": 8,
         "d": 128, "page": 64, "window": 0, "sinks": False},
        # a decode batch whose sequences are between half and all of 4096 long: the cache read once
        {"name": "attend_decode_64x4096", "op": "attend", "batch": 64, "ctx": 4096, "spread": 0.5, "new": 1, "mixed": False, "hq": 32, "hkv": 8,
         "d": 128, "page": 64, "window": 0, "sinks": False},
        # one long context: the work of few rows split over the whole card
        {"name": "attend_decode_1x131072", "op": "attend", "batch": 1, "ctx": 131072, "spread": 0.0, "new": 1, "mixed": False, "hq": 32, "hkv": 8,
         "d": 128, "page": 256, "window": 0, "sinks": False},
        # four tokens at once (a draft being checked) over a window, with sinks, small pages, short heads
        {"name": "attend_draft_16x1500", "op": "attend", "batch": 16, "ctx": 1500, "spread": 0.9, "new": 4, "mixed": False, "hq": 64, "hkv": 8,
         "d": 64, "page": 16, "window": 128, "sinks": True},
        # a chunk of a prompt beside sequences that decode, on caches of up to 16000 tokens, five queries to a key head
        {"name": "attend_mixed_4x16000", "op": "attend", "batch": 4, "ctx": 16000, "spread": 0.7, "new": 600, "mixed": True, "hq": 40, "hkv": 8,
         "d": 128, "page": 64, "window": 0, "sinks": False},
        # prompts of about 1000 tokens
        {"name": "attend_prompt_6x1000", "op": "attend", "batch": 6, "ctx": 1000, "spread": 0.4, "new": 1000, "mixed": False, "hq": 64, "hkv": 8,
         "d": 64, "page": 32, "window": 0, "sinks": True},
        # one prompt of 8192 tokens
        {"name": "attend_prompt_8192", "op": "attend", "batch": 1, "ctx": 8192, "spread": 0.0, "new": 8192, "mixed": False, "hq": 32, "hkv": 8,
         "d": 128, "page": 128, "window": 0, "sinks": False},
    ]


HEADS = ((32, 8, 128), (32, 8, 128), (64, 8, 64), (40, 8, 128), (8, 1, 256), (16, 16, 64), (28, 4, 128), (48, 1, 128), (16, 4, 256))


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("rope", "append", "append", "decode", "decode", "decode", "prompt", "prompt"))
    hq, hkv, d = rng.choice(HEADS)
    page = rng.choice((16, 32, 64, 128, 256))
    if op in ("rope", "append"):
        case = {"op": op, "tokens": min(_log_int(rng, 1, 8192), 8192 * 5120 // ((hq + 2 * hkv) * d)), "hq": hq, "hkv": hkv, "d": d,
                "rot": rng.choice((d, d, d // 2)), "norm": rng.random() < 0.5, "neighbours": rng.random() < 0.3}
        if op == "append":
            case.update(hq=rng.choice((hq, hq, 0)), page=page, padding=rng.choice((0, 0, 5, 11)))
        return case
    case = {"op": "attend", "hq": hq, "hkv": hkv, "d": d, "page": page, "spread": rng.choice((0.0, 0.5, 0.9)), "mixed": False,
            "window": rng.choice((0, 0, 0, _log_int(rng, 16, 4096))), "sinks": rng.random() < 0.3}
    if op == "decode":
        case.update(batch=_log_int(rng, 1, 128), ctx=_log_int(rng, 1, 131072), new=rng.choice((1, 1, 1, 2, 5)))
        while case["batch"] * case["ctx"] * hkv * d > MAX_CACHED:
            case["batch"], case["ctx"] = max(1, case["batch"] * 3 // 4), case["ctx"] * 3 // 4
    else:
        case.update(batch=_log_int(rng, 1, 8), ctx=_log_int(rng, 64, 16384), mixed=rng.random() < 0.4)
        case["new"] = _log_int(rng, 16, case["ctx"])
        while case["batch"] * case["new"] * case["ctx"] * hq > MAX_PAIRS:
            case["batch"], case["ctx"] = max(1, case["batch"] * 3 // 4), max(64, case["ctx"] * 3 // 4)
            case["new"] = min(case["new"], case["ctx"])
    return case


def sequences(case):
    """``[(new tokens, keys)]`` of a batch: lengths spread below ``ctx``, in a mixed batch every other sequence decodes."""
    rows = []
    for b in range(case["batch"]):
        keys = max(1, case["ctx"] - int(case["ctx"] * case["spread"] * ((b * 0.618034) % 1.0)))
        new = min(case["new"], keys)
        rows.append((1 if case["mixed"] and b % 2 else new, keys))
    return rows


def _visible(new, keys, window):
    """Query-key pairs of one head: query i sees keys up to its position keys - new + i, at most the last `window` of them."""
    return sum(min(p, window) if window else p for p in range(keys - new + 1, keys + 1))


def work(case):
    d, hq, hkv = case["d"], case["hq"], case["hkv"]
    if case["op"] == "rope":
        return {"bytes": case["tokens"] * ((hq + hkv) * d * 4.0 + case["rot"] * 4.0), "flops": 8.0 * case["tokens"] * (hq + hkv) * d}
    if case["op"] == "append":   # codes and scales are written once; the pass also reads them and gives them out as bf16
        cached = 2 * hkv * d * 17 / 32
        return {"bytes": case["tokens"] * ((hq + 2 * hkv) * d * 2.0 + hq * d * 2.0 + case["rot"] * 4.0 + 2 * cached + 2 * hkv * d * 2.0),
                "flops": 8.0 * case["tokens"] * (hq + 2 * hkv) * d}
    rows = sequences(case)
    w = case["window"]
    seen = sum(min(k, w + n - 1) if w else k for n, k in rows)
    tokens = sum(n for n, _ in rows)
    pairs = sum(_visible(n, k, w) for n, k in rows)
    return {"bytes": seen * hkv * 2 * d * 17 / 32 + tokens * hq * d * 4.0, "flops": 4.0 * d * hq * pairs}


# ---- what a program has in hand ------------------------------------------------------------------------------------------------
def _tables(rot, length):
    angle = torch.arange(length, device="cuda", dtype=torch.float64)[:, None] * (10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot))
    return angle.cos().float(), angle.sin().float()


def _channel_gains(g, heads, d):
    """One channel in sixteen four times larger, as keys have."""
    return torch.where(torch.rand(heads, d, generator=g, device="cuda") < 1 / 16, 4.0, 1.0)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    s = dict(case)
    if case["op"] in ("rope", "append"):
        t = case["tokens"]
        qkv = torch.randn(t, hq + 2 * hkv, d, generator=g, device="cuda") * torch.cat(
            [_channel_gains(g, hq + hkv, d), torch.ones(hkv, d, device="cuda")])
        qkv = qkv.bfloat16()
        s["q"] = qkv[:, :hq] if hq else None
        s["k"], s["v"] = qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        s["cos"], s["sin"] = _tables(case["rot"], 16384)
        s["positions"] = torch.randint(0, 16384, (t,), generator=g, device="cuda", dtype=torch.int32)
        s["q_weight"] = (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).bfloat16() if case["norm"] and hq else None
        s["k_weight"] = (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).bfloat16() if case["norm"] else None
        if case["op"] == "append":
            page = case["page"]
            pages = -(-t // page) + 3
            s["cache"] = (torch.zeros(pages, hkv, page, d // 2, dtype=torch.uint8, device="cuda"), torch.zeros(pages, hkv, page, d // 32, dtype=torch.uint8, device="cuda"),
                          torch.zeros(pages, hkv, page, d // 2, dtype=torch.uint8, device="cuda"), torch.zeros(pages, hkv, page, d // 32, dtype=torch.uint8, device="cuda"))
            # runs of a page's slots, pages in any order; every padding-th token is not stored
            order = torch.randperm(pages, generator=g, device="cuda")
            slots = (order[:, None] * page + torch.arange(page, device="cuda")).reshape(-1)[:t].int()
            if case["padding"]:
                slots[case["padding"] - 1::case["padding"]] = -1
            s["slots"] = slots.contiguous()
        return s
    rows = sequences(case)
    page = case["page"]
    width = max(-(-k // page) for _, k in rows)
    pages = sum(-(-k // page) for _, k in rows)
    table = torch.zeros(len(rows), width, dtype=torch.int32, device="cuda")
    order, at = torch.randperm(pages, generator=g, device="cuda").int(), 0
    for b, (_, k) in enumerate(rows):
        n = -(-k // page)
        table[b, :n] = order[at:at + n]
        at += n
    keys = torch.randn(pages, hkv, page, d, generator=g, device="cuda") * _channel_gains(g, hkv, d)[:, None]
    k_codes, k_scale = _quantise(keys)
    del keys
    v_codes, v_scale = _quantise(torch.randn(pages, hkv, page, d, generator=g, device="cuda"))
    s["cache"] = (k_codes, k_scale, v_codes, v_scale)
    s["page_table"] = table
    s["seq_lens"] = torch.tensor([k for _, k in rows], dtype=torch.int32, device="cuda")
    new = [n for n, _ in rows]
    starts = [sum(new[:i]) for i in range(len(new) + 1)]
    s["cu_q"] = torch.tensor(starts, dtype=torch.int32, device="cuda") if case["new"] > 1 else None
    s["max_q"] = max(new)
    s["q"] = torch.randn(starts[-1], hq, d, generator=g, device="cuda").bfloat16()
    s["scale"] = 1.0 / math.sqrt(d)
    s["sink_logits"] = torch.randn(hq, generator=g, device="cuda") if case["sinks"] else None
    return s


# ---- the plain forms --------------------------------------------------------------------------------------------------------------
def _by_neighbours(x):
    """Sum over the last axis, neighbours first: the order is part of the operator, so that what is quantised behind it has
    the same bits wherever it is computed."""
    return x[..., 0] if x.shape[-1] == 1 else _by_neighbours(x[..., 0::2] + x[..., 1::2])


def _norm_rope(x, weight, cos, sin, neighbours):
    """fp32 ``[tokens, heads, D]`` of ``x``; ``cos``, ``sin`` are the tokens' rows."""
    x = x.float()
    if weight is not None:
        r = 1.0 / torch.sqrt(_by_neighbours(x * x) / x.shape[-1] + EPS)
        x = x * r[..., None] * weight.float()
    half = cos.shape[-1]
    c, s = cos[:, None], sin[:, None]
    if neighbours:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
        return torch.cat([turned, x[..., 2 * half:]], -1)
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * half:]], -1)


def _quantise(x):
    """``(codes [..., D/2], scale bytes [..., D/32])`` of fp32 ``[..., D]``: E8M0 of the largest magnitude's exponent minus 2, E2M1
    by round-to-nearest-even, the low nibble the even channel."""
    blocks = x.unflatten(-1, (-1, 32))
    field = blocks.abs().amax(-1).view(torch.int32) >> 23
    byte = torch.where(field == 0, 127, (field - 2).clamp(min=0))
    a = blocks.abs() / (byte << 23).view(torch.float32)[..., None]
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75).to(torch.uint8) + (a > 1.25).to(torch.uint8) + (a >= 1.75).to(torch.uint8)
            + (a > 2.5).to(torch.uint8) + (a >= 3.5).to(torch.uint8) + (a > 5.0).to(torch.uint8) + (blocks < 0).to(torch.uint8) * 8)
    code = code.flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), byte.to(torch.uint8)


def _values(codes, scale):
    """fp32 ``[..., D]`` of packed codes and scale bytes."""
    grid = torch.tensor(GRID + tuple(-v for v in GRID), device=codes.device)
    x = torch.stack([grid[(codes & 15).int()], grid[(codes >> 4).int()]], -1).flatten(-2)
    power = (scale.int() << 23).view(torch.float32)
    return (x.unflatten(-1, (-1, 32)) * power[..., None]).flatten(-2)


def _plain_append(s):
    c, sn = s["cos"][s["positions"]], s["sin"][s["positions"]]
    k = _quantise(_norm_rope(s["k"], s["k_weight"], c, sn, s["neighbours"]))
    v = _quantise(s["v"].float())
    page = s["page"]
    stored = s["slots"] >= 0
    at = s["slots"][stored].long()
    for cache, new in zip(s["cache"], (*k, *v)):
        cache[at // page, :, at % page] = new[stored]
    at = s["slots"].clamp(min=0).long()
    kc, ks, vc, vs = (cache[at // page, :, at % page] for cache in s["cache"])
    out = {"k": torch.where(stored[:, None, None], _values(kc, ks), 0.0).bfloat16(), "v": torch.where(stored[:, None, None], _values(vc, vs), 0.0).bfloat16()}
    if s["q"] is not None:
        out["q"] = _norm_rope(s["q"], s["q_weight"], c, sn, s["neighbours"]).bfloat16()
    return out


def _plain_attend(s):
    hq, hkv, d, page = s["hq"], s["hkv"], s["d"], s["page"]
    batch, width = s["page_table"].shape
    group, length, most = hq // hkv, width * page, s["max_q"]

    def cached(codes, scale):   # [batch, kv heads, keys, D]
        at = s["page_table"].long()
        return _values(codes[at].transpose(1, 2).reshape(batch, hkv, length, -1), scale[at].transpose(1, 2).reshape(batch, hkv, length, -1))

    keys, values = cached(*s["cache"][:2]), cached(*s["cache"][2:])
    if s["cu_q"] is None:
        first, new = torch.arange(batch, device="cuda"), torch.ones(batch, dtype=torch.int64, device="cuda")
    else:
        first, new = s["cu_q"][:-1].long(), (s["cu_q"][1:] - s["cu_q"][:-1]).long()
    i = torch.arange(most, device="cuda")
    real = i < new[:, None]                                             # [batch, most]
    at = torch.where(real, first[:, None] + i, 0)
    q = s["q"][at].float().unflatten(2, (hkv, group)).permute(0, 2, 3, 1, 4).reshape(batch, hkv, group * most, d)
    scores = torch.matmul(q, keys.transpose(2, 3).contiguous()).view(batch, hkv, group, most, length) * s["scale"]
    lens = s["seq_lens"].long()
    position = (lens[:, None] - new[:, None] + i)[..., None]              # [batch, most, 1]
    j = torch.arange(length, device="cuda")
    seen = (j <= position) & (j < lens[:, None, None])
    if s["window"]:
        seen = seen & (j > position - s["window"])
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    m = scores.amax(-1, keepdim=True)
    if s["sink_logits"] is not None:
        sink = s["sink_logits"].view(1, hkv, group, 1, 1)
        m = torch.maximum(m, sink)
    m = torch.where(m == -math.inf, 0.0, m)
    p = torch.exp(scores.sub_(m))
    total = p.sum(-1, keepdim=True)
    if s["sink_logits"] is not None:
        total = total + torch.exp(sink - m)
    out = torch.matmul(p.view(batch, hkv, group * most, length), values).view(batch, hkv, group, most, d)
    out = torch.where(total > 0, out / total, 0.0)
    return out.permute(0, 3, 1, 2, 4).reshape(batch, most, hq, d)[real].bfloat16()


def run(state):
    s = state
    if own:
        import avelang_amd as ave

        if s["op"] == "rope":
            return ave.qk_norm_rope(s["q"], s["k"], s["cos"], s["sin"], s["positions"], s["q_weight"], s["k_weight"], eps=EPS, neighbours=s["neighbours"])
        if s["op"] == "append":
            q = ave.append_kv_mxfp4(s["k"], s["v"], s["cache"], s["slots"], s["cos"], s["sin"], s["positions"], s["k_weight"], q=s["q"],
                                    q_weight=s["q_weight"], eps=EPS, neighbours=s["neighbours"])
            k, v = ave.gather_kv_mxfp4(s["cache"], s["slots"])
            return {"k": k, "v": v} if q is None else {"k": k, "v": v, "q": q}
        return ave.attention_mxfp4(s["q"], s["cache"], s["page_table"], s["seq_lens"], s["cu_q"], max_q=s["max_q"], scale=s["scale"],
                                   window=s["window"], sinks=s["sink_logits"])
    if s["op"] == "rope":
        c, sn = s["cos"][s["positions"]], s["sin"][s["positions"]]
        return tuple(_norm_rope(s[n], s[n + "_weight"], c, sn, s["neighbours"]).bfloat16() for n in ("q", "k"))
    return _plain_append(s) if s["op"] == "append" else _plain_attend(s)


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------------------
def _exact_turn(x, weight, angle_cos, angle_sin, neighbours):
    """Norm and rotation as a product of every pair, seen as a complex number, with a point of the unit circle."""
    x = x.double()
    if weight is not None:
        x = x * weight.double() * (x.pow(2).mean(-1, keepdim=True) + EPS).rsqrt()
    half = angle_cos.shape[-1]
    pairs = x[..., :2 * half]
    pairs = pairs.unflatten(-1, (half, 2)) if neighbours else pairs.unflatten(-1, (2, half)).transpose(-1, -2)
    turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * torch.complex(angle_cos.double(), angle_sin.double())[:, None])
    turned = turned if neighbours else turned.transpose(-1, -2)
    return torch.cat([turned.flatten(-2), x[..., 2 * half:]], -1)


def _exact_rounded(x):
    """fp64 ``[..., D]`` rounded to E2M1 times a power of two per 32 channels."""
    b = x.double().unflatten(-1, (-1, 32))
    power = torch.ldexp(torch.ones_like(b[..., :1]), torch.frexp(b.abs().amax(-1, keepdim=True))[1] - 3)
    a = b / power
    step = torch.where(a.abs() < 2, 0.5, torch.where(a.abs() < 4, 1.0, 2.0))
    return ((a / step).round() * step).clamp(-6, 6).mul(power).flatten(-2)


def _exact_cached(codes, scale):
    both = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).double()
    sign, mag = 1 - 2 * (both >= 8).double(), both % 8
    exponent = torch.div(mag, 2, rounding_mode="floor")
    value = torch.where(mag < 2, mag / 2, (1 + (mag % 2) / 2) * torch.exp2(exponent - 1))
    return sign * value * torch.exp2(scale.double() - 127).repeat_interleave(32, -1)


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] in ("rope", "append"):
        at = s["positions"].long()
        turn = {n: _exact_turn(s[n], s[n + "_weight"], s["cos"][at], s["sin"][at], s["neighbours"]) for n in ("q", "k") if s[n] is not None}
        if s["op"] == "rope":
            return turn["q"], turn["k"]
        stored = (s["slots"] >= 0)[:, None, None]
        return {"k": _exact_rounded(turn["k"]) * stored, "v": _exact_rounded(s["v"]) * stored, **({"q": turn["q"]} if "q" in turn else {})}
    hq, hkv = s["hq"], s["hkv"]
    group, out, first = hq // hkv, [], 0
    for b, (new, keys) in enumerate(sequences(case)):
        pages = s["page_table"][b, : -(-keys // s["page"])].long()
        position = torch.arange(keys - new, keys, device="cuda")[:, None]
        j = torch.arange(keys, device="cuda")
        hidden = (j > position) | ((j <= position - s["window"]) if s["window"] else (j < 0))
        rows = torch.empty(new, hq, s["d"], dtype=torch.float64, device="cuda")
        for h in range(hkv):
            k, v = (_exact_cached(c[pages, h].flatten(0, 1)[:keys], f[pages, h].flatten(0, 1)[:keys]) for c, f in (s["cache"][:2], s["cache"][2:]))
            for n in range(h * group, (h + 1) * group):
                logits = (s["q"][first:first + new, n].double() @ k.t() * s["scale"]).masked_fill(hidden, -math.inf)
                if s["sink_logits"] is not None:
                    logits = torch.cat([logits, s["sink_logits"][n].double().expand(new, 1)], 1)
                rows[:, n] = torch.softmax(logits, 1)[:, :keys] @ v
        out.append(rows)
        first += new
    return torch.cat(out)
