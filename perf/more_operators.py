"""The operators of a decoding step that checks a tree of drafted tokens over an MXFP4 key/value cache: what is measured of them,
their plain forms in elementary torch operations, and their definitions in 64 bits.

Every case is a dict of plain values; ``op`` says what one pass is:

* ``tree``    which nodes of its sequence each node descends from, as bits, and its position, from the nodes' parents (``draft_tree``)
* ``attend``  attention of the nodes over their sequences' cached tokens and over their own ancestors (``tree_attention_mxfp4``)
* ``verify``  which drafted tokens the target's distributions accept for given random numbers, and the token behind them (``verify_draft``)
* ``keep``    the kept ones of each sequence's last tokens moved together, in the caches of all layers (``keep_kv_mxfp4``)

A sequence's nodes are its last ``n`` tokens, in an order that has parents before children; node 0 is the last token that was
already decided on.
"""
from __future__ import annotations

import math
import random

import torch

own = False

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)      # E2M1 magnitudes by code
MAX_CACHED = 131072 * 8 * 128        # cached tokens * kv_heads * D of a drawn batch; the largest listed one has as many
MAX_SCORES = 64 * 131072 * 32 * 128  # nodes * keys * heads * D
MAX_LOGITS = 1024 * 131072
MAX_NODES = 256 * 64
MAX_MOVED = 16 * 4096 * 8 * 128      # layers * tokens * kv_heads * D


# ---- cases -----------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one sequence with a small tree: latency
        {"name": "tree_1x8", "op": "tree", "batch": 1, "nodes": 8, "spread": 0.0, "chain": False},
        # a large batch of trees of 64
        {"name": "tree_256x64", "op": "tree", "batch": 256, "nodes": 64, "spread": 0.3, "chain": False},
        # one short sequence, eight nodes: latency
        {"name": "attend_1x700_8", "op": "attend", "batch": 1, "ctx": 700, "spread": 0.0, "nodes": 8, "chain": False, "hq": 32, "hkv": 8, "d": 128,
         "page": 64, "window": 0, "sinks": False},
        # a batch whose sequences are between half and all of 4096 long, trees of up to 16
        {"name": "attend_16x4096_16", "op": "attend", "batch": 16, "ctx": 4096, "spread": 0.5, "nodes": 16, "chain": False, "hq": 32, "hkv": 8, "d": 128,
         "page": 64, "window": 0, "sinks": False},
        # large ragged trees, short heads, small pages, a window and sinks
        {"name": "attend_8x3000_64", "op": "attend", "batch": 8, "ctx": 3000, "spread": 0.9, "nodes": 64, "chain": False, "hq": 64, "hkv": 8, "d": 64,
         "page": 16, "window": 1000, "sinks": True},
        # one long context, a tree of 64
        {"name": "attend_1x131072_64", "op": "attend", "batch": 1, "ctx": 131072, "spread": 0.0, "nodes": 64, "chain": False, "hq": 32, "hkv": 8, "d": 128,
         "page": 256, "window": 0, "sinks": False},
        # one sequence, a chain of five drafts, greedy
        {"name": "verify_greedy_1x6", "op": "verify", "batch": 1, "nodes": 6, "spread": 0.0, "chain": True, "vocab": 32768, "f32": True, "probs": False,
         "temperature": 0.0},
        # chains of five sampled drafts with the distributions that they were drawn from, an odd vocabulary
        {"name": "verify_probs_8x6", "op": "verify", "batch": 8, "nodes": 6, "spread": 0.4, "chain": True, "vocab": 50001, "f32": False, "probs": True,
         "temperature": 1.0},
        # a batch of trees, sampled from, a large vocabulary
        {"name": "verify_tree_64x16", "op": "verify", "batch": 64, "nodes": 16, "spread": 0.0, "chain": False, "vocab": 131072, "f32": False, "probs": False,
         "temperature": 0.8},
        # one sequence's accepted nodes in the caches of 32 layers: latency
        {"name": "keep_1x16_32_layers", "op": "keep", "batch": 1, "ctx": 512, "spread": 0.0, "nodes": 16, "evict": False, "layers": 32, "hkv": 8, "d": 128,
         "page": 64},
        # a batch of 64 of them
        {"name": "keep_64x16_32_layers", "op": "keep", "batch": 64, "ctx": 512, "spread": 0.5, "nodes": 16, "evict": False, "layers": 32, "hkv": 8, "d": 128,
         "page": 64},
        # the first tokens and the later half of long sequences stay in one layer's cache
        {"name": "keep_half_of_16x4099", "op": "keep", "batch": 16, "ctx": 4099, "spread": 0.0, "nodes": 4099, "evict": True, "layers": 1, "hkv": 8, "d": 128,
         "page": 64},
    ]


HEADS = ((32, 8, 128), (32, 8, 128), (64, 8, 64), (40, 8, 128), (8, 1, 256), (16, 16, 64), (28, 4, 128), (48, 1, 128), (16, 4, 256))


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("tree", "attend", "attend", "attend", "attend", "verify", "verify", "verify", "keep", "keep"))
    hq, hkv, d = rng.choice(HEADS)
    page = rng.choice((16, 32, 64, 128, 256))
    case = {"op": op, "batch": _log_int(rng, 1, 128), "nodes": _log_int(rng, 1, 64), "spread": rng.choice((0.0, 0.4, 0.9)), "chain": rng.random() < 0.25}
    if op == "tree":
        while case["batch"] * case["nodes"] > MAX_NODES:
            case["batch"] = max(1, case["batch"] * 3 // 4)
    elif op == "attend":
        case.update(ctx=max(case["nodes"], _log_int(rng, 1, 131072)), hq=hq, hkv=hkv, d=d, page=page, window=rng.choice((0, 0, 0, _log_int(rng, 64, 4096))),
                    sinks=rng.random() < 0.3)
        while case["batch"] * case["ctx"] * hkv * d > MAX_CACHED or case["batch"] * case["ctx"] * case["nodes"] * hq * d > MAX_SCORES:
            case["batch"], case["ctx"] = max(1, case["batch"] * 3 // 4), max(case["nodes"], case["ctx"] * 3 // 4)
    elif op == "verify":
        probs = rng.random() < 0.35
        case.update(vocab=_log_int(rng, 1000, 262144), f32=rng.random() < 0.3, probs=probs, temperature=rng.choice((0.0, 0.6, 1.0, 1.3)))
        # logits of 32 bits and the drafts' distributions beside them cost two and four times as much
        while case["batch"] * case["nodes"] * case["vocab"] * (2 if case["f32"] else 1) * (4 if probs else 1) > MAX_LOGITS:
            case["batch"], case["nodes"] = max(1, case["batch"] * 3 // 4), max(1, case["nodes"] * 3 // 4)
    else:
        evict = rng.random() < 0.4
        layers = _log_int(rng, 1, 4 if evict else 48)
        case.update(layers=layers, evict=evict, hkv=hkv, d=d, page=page)
        case["nodes"] = _log_int(rng, 300, 8192) if evict else case["nodes"]
        del case["chain"]
        while layers * case["batch"] * case["nodes"] * hkv * d > MAX_MOVED:
            case["batch"], case["nodes"] = max(1, case["batch"] * 3 // 4), max(1, case["nodes"] * 3 // 4)
        case["ctx"] = case["nodes"] if evict else 256 + case["nodes"]
    return case


def _spread(case, what, b):
    return max(1, case[what] - int(case[what] * case["spread"] * ((b * 0.618034) % 1.0)))


def sequences(case):
    """``[(nodes, tokens)]`` of a batch: both spread below the case's numbers, the nodes the last of the tokens."""
    rows = []
    for b in range(case["batch"]):
        nodes = _spread(case, "nodes", b)
        rows.append((nodes, max(nodes, _spread(case, "ctx", b + 1)) if "ctx" in case else nodes))
    return rows


def kept_of(case):
    """How many of its last tokens a sequence of the case keeps."""
    if case["evict"]:
        return [n // 2 for n, _ in sequences(case)]
    return [min(1 + (b * 7 + 3) % 5, (n + 1) // 2) for b, (n, _) in enumerate(sequences(case))]


def work(case):
    rows = sequences(case)
    nodes = sum(n for n, _ in rows)
    if case["op"] == "tree":      # parents in; a word of bits and a position out
        return {"bytes": nodes * 16.0 + 8.0 * case["batch"], "flops": 2.0 * sum(n * n for n, _ in rows)}
    if case["op"] == "attend":
        d, hq, hkv, w = case["d"], case["hq"], case["hkv"], case["window"]
        seen = sum(min(k, w + n) if w else k for n, k in rows)
        pairs = sum(n * (min(k - n, w) if w else k - n) + n * (n + 1) // 2 for n, k in rows)
        return {"bytes": seen * hkv * 2 * d * 17 / 32 + nodes * (hq * d * 4.0 + 8.0), "flops": 4.0 * d * hq * pairs}
    if case["op"] == "verify":
        inner = (nodes - case["batch"]) if case["probs"] else 0      # at most so many nodes have children
        return {"bytes": case["vocab"] * (nodes * (4.0 if case["f32"] else 2.0) + inner * 4.0), "flops": 4.0 * case["vocab"] * (nodes + inner)}
    moved = sum(max(0, n - 1) for n in kept_of(case))     # the first one stays where it is
    return {"bytes": moved * case["layers"] * case["hkv"] * 2 * case["d"] * 17 / 32 * 2 + 16.0 * case["batch"], "flops": 1.0 * moved}


# ---- what a program has in hand ------------------------------------------------------------------------------------------------
def _quantise(x):
    """``(codes [..., D/2], scale bytes [..., D/32])`` of fp32 ``[..., D]``, values that a cache holds."""
    blocks = x.unflatten(-1, (-1, 32))
    field = blocks.abs().amax(-1).view(torch.int32) >> 23
    byte = torch.where(field == 0, 127, (field - 2).clamp(min=0))
    a = blocks.abs() / (byte << 23).view(torch.float32)[..., None]
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75).to(torch.uint8) + (a > 1.25).to(torch.uint8) + (a >= 1.75).to(torch.uint8)
            + (a > 2.5).to(torch.uint8) + (a >= 3.5).to(torch.uint8) + (a > 5.0).to(torch.uint8) + (blocks < 0).to(torch.uint8) * 8)
    code = code.flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), byte.to(torch.uint8)


def _channel_gains(g, heads, d):
    """One channel in sixteen four times larger, as keys have."""
    return torch.where(torch.rand(heads, d, generator=g, device="cuda") < 1 / 16, 4.0, 1.0)


def _parents(seed, case, counts):
    """int32, the nodes of all sequences in a row: a chain, or trees of up to four children a node, level by level; -1 for the first node."""
    rng, parents = random.Random(seed), []
    for n in counts:
        up, children = -1, 0
        for j in range(n):
            if case.get("chain") or j < 2:
                up, children = j - 1, 0
            elif children == 4 or rng.random() < 0.45:
                up, children = min(up + rng.choice((1, 1, 2)), j - 1), 0
            children += 1
            parents.append(up)
    return torch.tensor(parents, dtype=torch.int32).cuda()


def _paged(g, rows, page):
    """``(page table, pages)``: every sequence's pages anywhere among them."""
    width = max(-(-k // page) for _, k in rows)
    pages = sum(-(-k // page) for _, k in rows)
    table = torch.zeros(len(rows), width, dtype=torch.int32)
    order, at = torch.randperm(pages, generator=torch.Generator().manual_seed(g.initial_seed() % 2 ** 31)).int(), 0
    for b, (_, k) in enumerate(rows):
        n = -(-k // page)
        table[b, :n] = order[at:at + n]
        at += n
    return table.cuda(), pages


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    rows = sequences(case)
    counts = [n for n, _ in rows]
    starts = [sum(counts[:i]) for i in range(len(counts) + 1)]
    s["cu_q"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    s["seq_lens"] = torch.tensor([k for _, k in rows], dtype=torch.int32, device="cuda")
    s["max_q"] = max(counts)
    if case["op"] != "keep":
        s["parents"] = _parents(seed, case, counts)
    if case["op"] == "attend":
        hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
        s["seen"], _ = _plain_tree(s)
        s["page_table"], pages = _paged(g, rows, page)
        keys = torch.randn(pages, hkv, page, d, generator=g, device="cuda") * _channel_gains(g, hkv, d)[:, None]
        k_codes, k_scale = _quantise(keys)
        del keys
        s["cache"] = (k_codes, k_scale, *_quantise(torch.randn(pages, hkv, page, d, generator=g, device="cuda")))
        s["q"] = torch.randn(starts[-1], hq, d, generator=g, device="cuda").bfloat16()
        s["scale"] = 1.0 / math.sqrt(d)
        s["sink_logits"] = torch.randn(hq, generator=g, device="cuda") if case["sinks"] else None
    elif case["op"] == "verify":
        _prepare_verify(s, g, case)
    elif case["op"] == "keep":
        hkv, d, page, layers = case["hkv"], case["d"], case["page"], case["layers"]
        s["page_table"], pages = _paged(g, rows, page)
        # every layer's cache is a part of four large tensors, as a program allocates them
        s["all"] = tuple(torch.randint(0, 256, (layers, pages, hkv, page, n), generator=g, device="cuda", dtype=torch.uint8)
                         for n in (d // 2, d // 32, d // 2, d // 32))
        s["caches"] = [tuple(t[layer] for t in s["all"]) for layer in range(layers)]
        kept = kept_of(case)
        s["accepted"] = torch.tensor(kept, dtype=torch.int32, device="cuda")
        # Kept tokens: the first, and later ones none of whose places another one takes (so that a pass over what a pass has left does
        # the same moves again).  Evicted: the first few and the latest stay.
        paths = []
        for n, count in zip(counts, kept):
            path = torch.full((n,), -1, dtype=torch.int32)
            if count:
                if case["evict"]:
                    path[:count] = torch.arange(n - count, n)
                    path[0] = 0
                else:
                    others = torch.randperm(n - count, generator=torch.Generator().manual_seed(seed % 2 ** 31 + n))[:count - 1].sort().values + count
                    path[:count] = torch.cat([torch.zeros(1, dtype=torch.int64), others])
            paths.append(path)
        s["path"] = torch.cat(paths).cuda()
    return s


def _prepare_verify(s, g, case):
    """Logits as a trained model's: a wide spread, and one token that stands out, more or less; drafted tokens are that one, and for the
    siblings the next ones; with ``probs`` they are drawn from a distribution near the target's."""
    t, v = s["parents"].shape[0], case["vocab"]
    x = torch.randn(t, v, generator=g, device="cuda") * 2.5
    stars = torch.randint(0, v, (t, 4), generator=g, device="cuda")
    level = math.log(v) + 3.0 + torch.randn(t, 1, generator=g, device="cuda") - torch.tensor([0.0, 1.0, 2.0, 3.0], device="cuda")
    x.scatter_(1, stars, level)
    s["logits"] = x if case["f32"] else x.bfloat16()
    row = torch.arange(t, device="cuda")
    first = torch.repeat_interleave(s["cu_q"][:-1].long(), (s["cu_q"][1:] - s["cu_q"][:-1]).long())
    parent = first + s["parents"].clamp(min=0)
    if case["probs"]:
        q = torch.softmax(x / max(case["temperature"], 0.5) + 0.5 * torch.randn(t, v, generator=g, device="cuda"), 1)
        s["draft_probs"] = q
        noise = torch.empty(t, v, device="cuda").exponential_(generator=g)
        token = torch.empty(t, dtype=torch.int64, device="cuda")
        for part in torch.arange(t, device="cuda").split(256):
            token[part] = (q[parent[part]] / noise[part]).argmax(1)
    else:
        s["draft_probs"] = None
        rank = ((parent[None] == parent[:, None]) & (row[None] < row[:, None]) & (s["parents"] >= 0)[None]).sum(1)
        below = (torch.rand(t, generator=g, device="cuda") < 0.25).long()[parent]      # sometimes the drafts are not the likeliest
        token = stars[parent, (rank + below).clamp(max=3)]
    s["tokens"] = token.int()
    s["uniform"] = torch.rand(t, generator=g, device="cuda")
    s["temps"] = torch.full((case["batch"],), case["temperature"], device="cuda")


# ---- the plain forms --------------------------------------------------------------------------------------------------------------
def _padded(s):
    """Rows of the nodes as ``[batch, most]`` (row 0 where there is none), which of them are real, and the numbers of nodes."""
    first, n = s["cu_q"][:-1].long(), (s["cu_q"][1:] - s["cu_q"][:-1]).long()
    i = torch.arange(s["max_q"], device="cuda")
    real = i < n[:, None]
    return torch.where(real, first[:, None] + i, 0), real, n


def _flat(s, padded):
    """Rows of the nodes out of ``[batch, most, ...]``."""
    row = torch.arange(s["parents"].shape[0] if "parents" in s else s["path"].shape[0], device="cuda")
    b = torch.searchsorted(s["cu_q"][1:].long(), row, right=True)
    return padded[b, row - s["cu_q"].long()[b]]


def _ancestors(s):
    """``[batch, most, most]``: does node i descend from node j, or is it j?  The powers of "is its parent"."""
    at, real, _ = _padded(s)
    j = torch.arange(s["max_q"], device="cuda")
    up = (torch.where(real, s["parents"][at].long(), -1)[..., None] == j).float() + torch.eye(s["max_q"], device="cuda")
    return (torch.linalg.matrix_power(up, s["max_q"]) > 0) & real[..., None]


def _plain_tree(s):
    above = _ancestors(s)
    words = -(-s["max_q"] // 64)
    bits = torch.nn.functional.pad(above, (0, 64 * words - s["max_q"])).unflatten(-1, (words, 64)).long() << torch.arange(64, device="cuda")
    lens, n = s["seq_lens"].long(), (s["cu_q"][1:] - s["cu_q"][:-1]).long()
    return _flat(s, bits.sum(-1)), _flat(s, (lens - n)[:, None] + above.sum(-1) - 1).int()


def _values(codes, scale):
    """fp32 ``[..., D]`` of packed codes and scale bytes."""
    grid = torch.tensor(GRID + tuple(-v for v in GRID), device=codes.device)
    x = torch.stack([grid[(codes & 15).int()], grid[(codes >> 4).int()]], -1).flatten(-2)
    power = (scale.int() << 23).view(torch.float32)
    return (x.unflatten(-1, (-1, 32)) * power[..., None]).flatten(-2)


def _plain_attend(s):
    hq, hkv, d, page, most = s["hq"], s["hkv"], s["d"], s["page"], s["max_q"]
    batch, width = s["page_table"].shape
    group, length = hq // hkv, width * page

    def cached(codes, scale):   # [batch, kv heads, keys, D]
        at = s["page_table"].long()
        return _values(codes[at].transpose(1, 2).reshape(batch, hkv, length, -1), scale[at].transpose(1, 2).reshape(batch, hkv, length, -1))

    keys, values = cached(*s["cache"][:2]), cached(*s["cache"][2:])
    at, real, n = _padded(s)
    q = s["q"][at].float().unflatten(2, (hkv, group)).permute(0, 2, 3, 1, 4).reshape(batch, hkv, group * most, d)
    scores = torch.matmul(q, keys.transpose(2, 3).contiguous()).view(batch, hkv, group, most, length) * s["scale"]
    lens = s["seq_lens"].long()
    base = (lens - n)[:, None, None]
    j = torch.arange(length, device="cuda")
    node = j - base                                                   # [batch, 1, keys]
    bits = s["seen"][at].view(batch, most, -1)
    word = torch.gather(bits, 2, (node.clamp(0, 64 * bits.shape[-1] - 1) // 64).expand(batch, most, length))
    seen = (node >= 0) & (j < lens[:, None, None]) & ((word >> (node.clamp(min=0) % 64)) & 1).bool()
    before = (node < 0).expand(batch, most, length)
    if s["window"]:      # the last `window` of what a row sees
        before = before & (j >= base + seen.sum(-1, keepdim=True) - s["window"])
    seen = seen | before
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
    return _flat(s, out.permute(0, 3, 1, 2, 4).reshape(batch, most, hq, d)).bfloat16()


def _plain_verify(s):
    """In 64 bits: a token is chosen by where a number lies among sums of very many probabilities.

    Whether a node is accepted, once its parent is and its elder siblings are not, does not depend on where else the walk
    went; so all nodes are decided on at once, and the path is those whose ancestors all were the first accepted child."""
    at, real, n = _padded(s)
    most, v = s["max_q"], s["vocab"]
    j = torch.arange(most, device="cuda")
    parent = torch.where(real, s["parents"][at].long(), -1)
    token = s["tokens"][at].long()
    up = parent.clamp(min=0)
    greedy = ~(s["temps"] > 0)
    x = s["logits"].double()
    top, best = x.max(1)
    per = torch.where(greedy, 1.0, s["temps"].double())[:, None].expand(at.shape)
    weight = torch.exp((x - top[:, None]) / _flat(s, per)[:, None])
    p = weight / weight.sum(1, keepdim=True)
    row = at.gather(1, up)                                   # the parents' rows
    mine = p[row, token]
    sibling = (parent[:, None] == parent[..., None]) & (parent >= 0)[..., None]      # [batch, node, its sibling]
    elder = sibling & (j < j[:, None])
    u = s["uniform"].double()[at]
    if s["draft_probs"] is None:      # a rejected token's probability goes to the others
        again = (elder & (token[:, None] == token[..., None])).any(-1)
        mine = torch.where(again, 0.0, mine)
        taken = (elder * mine[:, None]).sum(-1)
        accept = u * (1 - taken) < mine
    else:                             # rejected k times: max(p - times[k] q, 0), over its sum
        q = s["draft_probs"].double()
        rank = elder.sum(-1)
        times, left = torch.zeros_like(p[:, 0]), torch.ones_like(p[:, 0])
        steps = [(times, left)]
        for _ in range(1 if s["chain"] else 4):
            times = times + left
            left = (p - times[:, None] * q).clamp(min=0).sum(1)
            steps.append((times, left))
        times, left = (torch.stack(t) for t in zip(*steps))
        drafted, by = q[row, token], rank.clamp(max=len(steps) - 1)
        accept = u * drafted * left[by, row] < (mine - times[by, row] * drafted).clamp(min=0)
    accept = torch.where(greedy[:, None], token == best[row], accept)
    chosen = (j == 0) | (accept & (parent >= 0) & ~(elder & accept[:, None]).any(-1))
    on = real & ~(_ancestors(s) & ~chosen[:, None]).any(-1)
    on = on & (_ancestors(s)[..., 0])
    path = torch.where(on, j, most).sort(1).values
    accepted = on.sum(1)
    last = torch.where(on, j, 0).amax(1)
    row = at.gather(1, last[:, None])[:, 0]
    tried = (parent == last[:, None]) & real
    if s["draft_probs"] is None:
        gone = torch.zeros(at.shape[0], v, device="cuda").scatter_reduce_(1, token, tried.float(), "amax")
        rest = torch.where(gone > 0, 0.0, p[row])
    else:
        rest = (p[row] - times[tried.sum(1), row][:, None] * q[row]).clamp(min=0)
    rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, p[row])
    sums = rest.cumsum(1)
    drawn = (sums <= s["uniform"].double()[at[:, 0]][:, None] * sums[:, -1:]).sum(1)
    drawn = torch.where(greedy, best[row], drawn)
    kept = j < accepted[:, None]
    path = torch.where(kept, path, -1)
    following = torch.cat([path[:, 1:], torch.full_like(path[:, :1], -1)], 1)
    emitted = torch.where(j == accepted[:, None] - 1, drawn[:, None], token.gather(1, following.clamp(min=0)))
    return accepted.int(), _flat(s, path).int(), _flat(s, torch.where(kept, emitted, -1)).int()


def _plain_keep(s):
    at, real, n = _padded(s)
    page, lens = s["page"], s["seq_lens"].long()
    i = torch.arange(s["max_q"], device="cuda")
    b = torch.arange(len(n), device="cuda")[:, None].expand(at.shape)
    stays = i < s["accepted"].long()[:, None]
    base = (lens - n)[:, None]
    row = torch.arange(s["path"].shape[0], device="cuda")
    to = base + i
    come = base + torch.where(stays & real, s["path"][at].long(), i)      # the others stay as they are

    def place(position):      # page and offset of every row
        which = s["page_table"][b, (position // page).clamp(max=s["page_table"].shape[1] - 1)].long()
        return _of_rows(s, which, row), _of_rows(s, position % page, row)

    (p0, o0), (p1, o1) = place(come), place(to)
    for cache in s["all"]:
        cache[:, p1, :, o1] = cache[:, p0, :, o0]
    return (*s["all"], (lens - n + s["accepted"].long()).int())


def _of_rows(s, padded, row):
    b = torch.searchsorted(s["cu_q"][1:].long(), row, right=True)
    return padded[b, row - s["cu_q"].long()[b]]


def run(state):
    s = state
    if own:
        import avelang_amd as ave

        if s["op"] == "tree":
            return ave.draft_tree(s["parents"], s["cu_q"], s["seq_lens"], max_q=s["max_q"])
        if s["op"] == "attend":
            return ave.tree_attention_mxfp4(s["q"], s["cache"], s["page_table"], s["seq_lens"], s["cu_q"], s["seen"], max_q=s["max_q"],
                                            scale=s["scale"], window=s["window"], sinks=s["sink_logits"])
        if s["op"] == "verify":
            return ave.verify_draft(s["logits"], s["tokens"], s["parents"], s["cu_q"], s["uniform"], s["temps"], s["draft_probs"])
        return (*s["all"], ave.keep_kv_mxfp4(s["caches"], s["page_table"], s["seq_lens"], s["cu_q"], s["path"], s["accepted"]))
    return {"tree": _plain_tree, "attend": _plain_attend, "verify": _plain_verify, "keep": _plain_keep}[s["op"]](s)


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------------------
def _exact_cached(codes, scale):
    both = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).double()
    sign, mag = 1 - 2 * (both >= 8).double(), both % 8
    exponent = torch.div(mag, 2, rounding_mode="floor")
    value = torch.where(mag < 2, mag / 2, (1 + (mag % 2) / 2) * torch.exp2(exponent - 1))
    return sign * value * torch.exp2(scale.double() - 127).repeat_interleave(32, -1)


def _lines(parents):
    """For each node of one sequence, the nodes from the first one down to it."""
    lines = []
    for i, p in enumerate(parents):
        lines.append((lines[p] if p >= 0 else []) + [i])
    return lines


def _exact_attend(s, case):
    hq, hkv = s["hq"], s["hkv"]
    group, out, first = hq // hkv, [], 0
    for b, (new, keys) in enumerate(sequences(case)):
        pages = s["page_table"][b, : -(-keys // s["page"])].long()
        hidden = torch.ones(new, keys, dtype=torch.bool)
        for i, line in enumerate(_lines(s["parents"][first:first + new].tolist())):
            sees = list(range(max(0, keys - new - max(0, s["window"] - len(line))) if s["window"] else 0, keys - new)) + [keys - new + a for a in line]
            hidden[i, sees] = False
        hidden = hidden.cuda()
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


def _exact_verify(s, case):
    """The walk as it is described: one distribution at a time, renewed after each rejection."""
    accepted, paths, emitted, first = [], [], [], 0
    for b, (n, _) in enumerate(sequences(case)):
        parents, tokens = s["parents"][first:first + n].tolist(), s["tokens"][first:first + n].tolist()
        u = s["uniform"][first:first + n].double().tolist()
        path, words = [0], []
        while True:
            node = path[-1]
            x = s["logits"][first + node].double()
            if case["temperature"] == 0:
                final = int((x == x.max()).nonzero()[0])
                child = next((c for c in range(node + 1, n) if parents[c] == node and tokens[c] == final), None)
            else:
                target = torch.softmax(x / s["temps"][b].double(), 0)
                p, child = target, None
                for c in (c for c in range(node + 1, n) if parents[c] == node):
                    q = torch.zeros_like(p).index_fill_(0, torch.tensor([tokens[c]], device="cuda"), 1.0) if s["draft_probs"] is None \
                        else s["draft_probs"][first + node].double()
                    if u[c] * float(q[tokens[c]]) < float(p[tokens[c]]):
                        child = c
                        break
                    rest = (p - q).clamp(min=0) if s["draft_probs"] is not None else p * (1 - q)
                    p = rest / rest.sum() if float(rest.sum()) > 0 else target
                if child is None:
                    sums = p.cumsum(0)
                    final = int(torch.searchsorted(sums, (u[0] * sums[-1]).view(1), right=True))
            if child is None:
                break
            path.append(child)
            words.append(tokens[child])
        accepted.append(len(path))
        paths += path + [-1] * (n - len(path))
        emitted += words + [final] + [-1] * (n - len(path))
        first += n
    return tuple(torch.tensor(t, dtype=torch.int32) for t in (accepted, paths, emitted))


def _exact_keep(s, case):
    """Token by token, as in a list."""
    kept, out = kept_of(case), [t.clone() for t in s["all"]]
    for new, old in zip(out, s["all"]):
        flat_new, flat_old = (t.transpose(2, 3).flatten(1, 2).clone() for t in (new, old))      # [layers, slots, heads, bytes]
        first = 0
        for b, (n, tokens) in enumerate(sequences(case)):
            table = s["page_table"][b].tolist()
            slot = lambda position: table[position // s["page"]] * s["page"] + position % s["page"]   # noqa: E731
            come = [slot(tokens - n + i) for i in s["path"][first:first + kept[b]].tolist()]
            to = [slot(tokens - n + i) for i in range(kept[b])]
            flat_new[:, to] = flat_old[:, come]
            first += n
        new.copy_(flat_new.unflatten(1, (new.shape[1], new.shape[3])).transpose(2, 3))
    return (*out, torch.tensor([tokens - n + kept[b] for b, (n, tokens) in enumerate(sequences(case))], dtype=torch.int32))


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "attend":
        return _exact_attend(s, case)
    if s["op"] == "verify":
        return _exact_verify(s, case)
    if s["op"] == "keep":
        return _exact_keep(s, case)
    seen, positions, first = [], [], 0
    for n, keys in sequences(case):
        for line in _lines(s["parents"][first:first + n].tolist()):
            words = [0] * (-(-s["max_q"] // 64))
            for a in line:
                words[a // 64] |= 1 << a % 64
            seen.append([w - (1 << 64) if w >> 63 else w for w in words])
            positions.append(keys - n + len(line) - 1)
        first += n
    return torch.tensor(seen, dtype=torch.int64), torch.tensor(positions, dtype=torch.int32)
