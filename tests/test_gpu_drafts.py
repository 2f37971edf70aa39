"""Checking a tree of drafted tokens -- ancestors, attention under their bits, acceptance, the move of what is kept -- against plain implementations in 64 bits,
where each can go wrong."""
import numpy as np
import pytest
import torch

import avelang_amd as ave
from avelang_amd import _lib, attention as attention_module, drafts as drafts_module
from tests import attention_helpers as A
from tests import draft_helpers as D

pytestmark = pytest.mark.gpu

HEADS = {"gqa64": (8, 2, 64), "gqa128": (8, 2, 128), "gqa256": (6, 2, 256), "mha128": (3, 3, 128), "group5": (10, 2, 128), "mqa64": (24, 1, 64),
         "group40": (40, 1, 128)}
#: (nodes, keys): few rows, the kernel for prompts, more nodes than a word has bits, no keys before the nodes, nodes only, tiles' edges
ROWS = [[(1, 1), (8, 8), (3, 100)], [(7, 700)], [(16, 257), (1, 30), (16, 16)], [(64, 300), (5, 1000)], [(64, 64), (63, 127), (64, 128)], [(65, 200), (130, 130)],
        [(12, 1037), (0, 40), (33, 64)]]


def _parents(batch, seed, chain=False):
    rng = np.random.default_rng(seed)
    return [D.random_parents(rng, n, chain) for n, _ in batch.rows]


def _attend(gpu, batch, above, *, words=None, window=0, sinks=None, scale=None, max_q=None, wide=False):
    """The call, and its comparison; `above`: bool [nodes, nodes] of each sequence.  wide: a page table for 2^17 tokens, by which other kernels are chosen
    (blocks of 128 rows; no items kept whole)."""
    t = batch.tensors(gpu)
    if wide:
        t["page_table"] = torch.nn.functional.pad(t["page_table"], (0, 2 ** 17 // batch.page), value=-7)
    most = max(1, max(n for n, _ in batch.rows))
    words = -(-most // 64) if words is None else words
    seen = D.tensor(np.concatenate([D.words_of(a, words) for a in above]), gpu)
    lse = torch.full((batch.q.shape[0], batch.hq), float("nan"), device=gpu)
    out = torch.full(batch.q.shape, float("nan"), dtype=torch.bfloat16, device=gpu)
    got = ave.tree_attention_mxfp4(t["q"], t["cache"], t["page_table"], t["seq_lens"], t["cu_q"], seen, out, lse, max_q=most if max_q is None else max_q,
                                   window=window, sinks=D.tensor(sinks, gpu) if sinks is not None else None, scale=scale)
    assert got is out
    cut = [np.where(np.arange(a.shape[1]) < 64 * words, a, False) for a in above]
    want, want_lse, tol, lse_tol = D.masked_reference(batch, [D.visible(a, k, window) for a, (_, k) in zip(cut, batch.rows)], scale=scale, sinks=sinks)
    err = np.abs(out.float().cpu().numpy() - want)
    assert (err <= tol).all(), (float((err / tol).max()), np.argwhere(~(err <= tol))[:5].tolist())
    le, some = lse.cpu().numpy(), np.isfinite(want_lse)
    assert np.array_equal(le[~some], want_lse[~some])
    assert (np.abs(le[some] - want_lse[some]) <= lse_tol[some]).all()
    return t, seen, out


@pytest.mark.parametrize("rows", ROWS, ids=str)
@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("heads", HEADS)
def test_attention_over_trees(gpu, heads, page, rows):
    batch = A.Batch(rows, *HEADS[heads], page, seed=page + rows[0][1])
    above = [D.ancestors(p) for p in _parents(batch, rows[0][0])]
    _attend(gpu, batch, above)
    _attend(gpu, batch, above, wide=True)


@pytest.mark.parametrize("heads", ["gqa64", "gqa128", "gqa256", "mha128", "mqa64"])
@pytest.mark.parametrize("count,nodes,keys", [(70, 3, 40), (150, 9, 60), (300, 20, 50), (9, 64, 700)])
def test_many_sequences(gpu, heads, count, nodes, keys):
    """More sequences than a wave has lanes, more items than workgroups, items whole and in parts, some sequences empty."""
    rng = np.random.default_rng(count)
    rows = [(int(n), int(n) + int(k)) if n else (0, int(k)) for n, k in zip(rng.integers(0, nodes + 1, count), rng.integers(0, keys + 1, count))]
    batch = A.Batch(rows, *HEADS[heads], 16, seed=count)
    above = [D.ancestors(p) for p in _parents(batch, 3)]
    _attend(gpu, batch, above)
    _attend(gpu, batch, above, wide=True, window=33)


def test_a_bound_that_is_wrong(gpu):
    """max_q below and far above the nodes that there are chooses other kernels and costs time only."""
    batch = A.Batch([(40, 300), (3, 90), (64, 64)], *HEADS["gqa128"], 16, seed=9)
    above = [D.ancestors(p) for p in _parents(batch, 4)]
    for bound in (0, 1, 3, 9, 5000):
        _attend(gpu, batch, above, max_q=bound)
        _attend(gpu, batch, above, max_q=bound, wide=True)


@pytest.mark.parametrize("rows", [[(6, 400), (3, 30)], [(40, 300), (20, 21), (64, 130)]], ids=str)
@pytest.mark.parametrize("how", [{"window": 1}, {"window": 7}, {"window": 64}, {"window": 100, "sinks": True}, {"sinks": True}, {"scale": -0.25}, {"scale": 0.0},
                                 {"window": (1 << 31) - 1}], ids=str)
@pytest.mark.parametrize("heads", ["gqa64", "gqa128", "gqa256", "group5"])
def test_windows_sinks_scales(gpu, heads, how, rows):
    batch = A.Batch(rows, *HEADS[heads], 32, seed=3)
    how = {k: batch.sinks if k == "sinks" else v for k, v in how.items()}
    for wide in (False, True):
        _attend(gpu, batch, [D.ancestors(p) for p in _parents(batch, 5)], wide=wide, **how)


@pytest.mark.parametrize("heads", ["gqa64", "gqa128", "gqa256", "group40"])
def test_any_bits(gpu, heads):
    """Bits that are no tree: later nodes, not the node itself, none at all (rows that see nothing where no key is before the nodes), bits behind the
    last node, and rows with fewer words than nodes."""
    rng = np.random.default_rng(1)
    batch = A.Batch([(5, 5), (20, 20), (70, 70), (70, 200), (130, 400)], *HEADS[heads], 16, seed=9)
    above = [rng.random((n, n)) < 0.3 for n, _ in batch.rows]
    for a in above:
        a[::3] = False
    _, _, out = _attend(gpu, batch, above)
    assert out[0].eq(0).all() and out[5].eq(0).all()
    for wide in (False, True):
        _attend(gpu, batch, above, words=1, wide=wide)
        _attend(gpu, batch, above, window=40, sinks=batch.sinks, wide=wide)
    wide = [np.concatenate([a, np.ones((a.shape[0], 300), bool)], 1) for a in above]      # bits of nodes that are not there
    t = batch.tensors(gpu)
    a, b = (ave.tree_attention_mxfp4(t["q"], t["cache"], t["page_table"], t["seq_lens"], t["cu_q"], D.tensor(np.concatenate([D.words_of(x, 4) for x in m]), gpu), max_q=130,
                                     window=w) for m, w in ((above, 0), (wide, 0)))
    assert torch.equal(a, b)


@pytest.mark.parametrize("heads", ["gqa64", "gqa128", "gqa256"])
@pytest.mark.parametrize("window", [0, 50])
def test_a_chain_is_causal_attention(gpu, heads, window):
    """The same kernels with another way to say what is seen: the bits of a chain give the causal call's result where both take the same parts."""
    batch = A.Batch([(5, 300), (4, 4), (8, 1025)], *HEADS[heads], 16, seed=2)
    t, seen, out = _attend(gpu, batch, [np.tril(np.ones((n, n), bool)) for n, _ in batch.rows], window=window)
    want, _, tol, _ = batch.reference(window=window)
    causal = ave.attention_mxfp4(t["q"], t["cache"], t["page_table"], t["seq_lens"], t["cu_q"], max_q=8, window=window)
    assert (np.abs(causal.float().cpu().numpy() - out.float().cpu().numpy()) <= 2 * tol).all()


def test_more_nodes_than_keys(gpu):
    """The first nodes stand before the sequence's start; their keys do not exist."""
    batch = A.Batch([(5, 3), (90, 20), (2, 0)], *HEADS["gqa128"], 16, seed=4)
    above = [np.tril(np.ones((n, n), bool)) for n, _ in batch.rows]
    t = batch.tensors(gpu)
    seen = D.tensor(np.concatenate([D.words_of(a, 2) for a in above]), gpu)
    out = ave.tree_attention_mxfp4(t["q"], t["cache"], t["page_table"], t["seq_lens"], t["cu_q"], seen, max_q=90)
    want, _, tol, _ = batch.reference()
    assert (np.abs(out.float().cpu().numpy() - want) <= tol).all()


def test_strides_other_rows_and_streams(gpu):
    """Rows of `seen` apart from each other and one row for all; rows behind the last sequence stay as they were; another stream; no `cu_q`."""
    batch = A.Batch([(9, 60), (4, 200)], *HEADS["gqa128"], 16, seed=6)
    t, seen, out = _attend(gpu, batch, [D.ancestors(p) for p in _parents(batch, 8)])
    call = lambda seen, **kw: ave.tree_attention_mxfp4(t["q"], t["cache"], t["page_table"], t["seq_lens"], t["cu_q"], seen, max_q=9, **kw)   # noqa: E731
    wide = torch.full((13, 5), -1, dtype=torch.int64, device=gpu)
    wide[:, :1] = seen
    assert torch.equal(call(wide[:, :1]), out)
    same = torch.full((13, 1), 0b1011, dtype=torch.int64, device=gpu)
    assert torch.equal(call(same), call(same[:1].expand(13, 1)))
    q = torch.cat([t["q"], t["q"][:3]])
    more = torch.full((16, 8, 128), 3.0, dtype=torch.bfloat16, device=gpu)
    got = ave.tree_attention_mxfp4(q, t["cache"], t["page_table"], t["seq_lens"], t["cu_q"], torch.cat([seen, seen[:3]]), more, max_q=9)
    assert torch.equal(got[:13], out) and got[13:].eq(3).all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call(seen)
    side.synchronize()
    assert torch.equal(other, out)
    one = ave.tree_attention_mxfp4(t["q"][:2], t["cache"], t["page_table"], t["seq_lens"], None, torch.ones(2, 1, dtype=torch.int64, device=gpu))
    assert torch.equal(one, ave.attention_mxfp4(t["q"][:2], t["cache"], t["page_table"], t["seq_lens"]))


@pytest.mark.parametrize("nodes", [2, 6, 40])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("heads", ["gqa64", "gqa128", "gqa256"])
def test_hidden_nodes_do_not_matter(gpu, heads, wide, nodes):
    """NaN scales of keys and values in nodes that a row does not see leave it alone; those that it sees make it NaN."""
    batch = A.Batch([(nodes, nodes + 70)], *HEADS[heads], 16, seed=7)
    above = np.eye(nodes, dtype=bool)
    above[:, 0] = True
    t, seen, out = _attend(gpu, batch, [above], wide=wide)
    for part in (1, 3):
        cache = [c.clone() for c in t["cache"]]
        hidden = min(3, nodes - 1)
        p, o = batch.place(0, 70 + hidden)
        cache[part][int(p), :, int(o)] = 0xFF
        got = ave.tree_attention_mxfp4(t["q"], tuple(cache), t["page_table"], t["seq_lens"], t["cu_q"], seen, max_q=nodes)
        others = [i for i in range(nodes) if i != hidden]
        assert torch.equal(got[others], out[others]) and got[hidden].isnan().all()


def test_workspaces_that_do_not_do(gpu):
    """(Their size depends on the device.)"""
    lib = _lib.load()
    batch = A.Batch([(40, 60)], *HEADS["gqa128"], 16, seed=6)
    t = batch.tensors(gpu)
    seen = torch.ones(40, 1, dtype=torch.int64, device=gpu)
    out = torch.empty_like(t["q"])
    table = torch.zeros(1, 4096, dtype=torch.int32, device=gpu)
    c, _ = attention_module._cache(t["cache"])
    a = _lib.Attention(q=t["q"].data_ptr(), q_token_stride=1024, q_head_stride=128, out=out.data_ptr(), page_table=table.data_ptr(), page_table_stride=4096,
                       seq_lens=t["seq_lens"].data_ptr(), cu_q=t["cu_q"].data_ptr(), tokens=40, batch=1, heads=8, table_pages=4096, max_q=40, scale=1)
    tree = _lib.Tree(seen.data_ptr(), 1, 1)
    need = lib.ave_fp4_tree_attention_mxfp4_workspace_bytes(a, tree, c)
    assert need > 0
    for ws, size in ((None, need), (1 << 20, need - 1), ((1 << 20) + 8, need)):
        assert lib.ave_fp4_tree_attention_mxfp4(a, tree, c, ws, size, None) == -1 and "workspace" in _lib.last_error()


# ---- ancestors and positions ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("counts", [[1], [0, 3, 0], [64, 65, 1, 130], [7] * 300, [500, 2]], ids=lambda c: str(c)[:20])
@pytest.mark.parametrize("chain", [False, True])
def test_tree_of_parents(gpu, counts, chain):
    rng = np.random.default_rng(len(counts))
    parents = [D.random_parents(rng, n, chain) for n in counts]
    for p in parents:
        if len(p) > 2:
            p[len(p) // 2] = rng.choice([-5, len(p) // 2, 1 << 30])   # hangs at nothing
    cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    lens = (np.array(counts) + rng.integers(0, 5000, len(counts))).astype(np.int32)
    t, most = int(cu[-1]), max(counts)
    seen = torch.full((t + 2, -(-most // 64)), 77, dtype=torch.int64, device=gpu)
    positions = torch.full((t + 2,), 77, dtype=torch.int32, device=gpu)
    flat = np.concatenate(parents + [[0, 0]]).astype(np.int32)
    got = ave.draft_tree(D.tensor(flat, gpu), D.tensor(cu, gpu), D.tensor(lens, gpu), seen, positions, max_q=most)
    assert got[0] is seen and got[1] is positions
    want = np.concatenate([D.words_of(D.ancestors(p), seen.shape[1]) for p in parents])
    at = np.concatenate([k - len(p) + D.ancestors(p).sum(1) - 1 for p, k in zip(parents, lens)])
    assert np.array_equal(seen.cpu().numpy()[:t], want) and np.array_equal(positions.cpu().numpy()[:t], at)
    assert seen[t:].eq(77).all() and positions[t:].eq(77).all()
    if 64 < most < 1000:      # fewer bits than nodes
        narrow, same = ave.draft_tree(D.tensor(flat, gpu), D.tensor(cu, gpu), D.tensor(lens, gpu), max_q=64)
        assert np.array_equal(narrow.cpu().numpy()[:t, 0], want[:, 0]) and torch.equal(same[:t], positions[:t])


def test_more_trees_than_workgroups(gpu):
    """Chains of 0 to 2 nodes for 70000 sequences: a workgroup takes a second one."""
    count = 70000
    n = np.arange(count) % 3
    cu = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
    place = np.arange(cu[-1]) - np.repeat(cu[:-1], n)
    lens = (n + np.arange(count) % 7).astype(np.int32)
    seen, positions = ave.draft_tree(D.tensor((place - 1).astype(np.int32), gpu), D.tensor(cu, gpu), D.tensor(lens, gpu), max_q=2)
    assert np.array_equal(seen.cpu().numpy()[:, 0], 2 ** (place + 1) - 1)
    assert np.array_equal(positions.cpu().numpy(), np.repeat(lens - n, n) + place)


def test_trees_beyond_what_lds_holds(gpu):
    rng = np.random.default_rng(5)
    n = 9001
    parents = np.array([-1] + [int(rng.integers(0, j)) for j in range(1, n)], np.int32)
    cu, lens = np.array([0, 5, 5 + n], np.int32), np.array([5, n + 10], np.int32)
    seen, positions = ave.draft_tree(D.tensor(np.concatenate([[-1, 0, 1, 2, 3], parents]).astype(np.int32), gpu), D.tensor(cu, gpu), D.tensor(lens, gpu), max_q=n)
    seen, positions, lines = seen.cpu().numpy(), positions.cpu().numpy(), D.lines_of(parents)
    for i in range(0, n, 7):
        bits = np.flatnonzero(np.unpackbits(seen[5 + i].view(np.uint8), bitorder="little"))
        assert bits.tolist() == lines[i] and positions[5 + i] == 10 + len(lines[i]) - 1


# ---- acceptance -----------------------------------------------------------------------------------------------------------------------------
def _draft(seed, counts, vocab, *, chain=False, f32=False, probs=False, sharp=3.0):
    """Logits with a few likely tokens, drafts among those (or drawn from distributions near the target's)."""
    rng = np.random.default_rng(seed)
    cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    t = int(cu[-1])
    logits = rng.standard_normal((t, vocab)).astype(np.float32) * sharp
    if not f32:
        logits = A.bf16(logits)
    parents = np.concatenate([D.random_parents(rng, n, chain) for n in counts] + [np.zeros(0, np.int32)]).astype(np.int32)
    tokens, q = np.zeros(t, np.int32), None
    if probs:
        q = np.stack([D.softmax(x + rng.standard_normal(vocab), 1.0) for x in logits]).astype(np.float32) if t else np.zeros((0, vocab), np.float32)
    for b, n in enumerate(counts):
        for j in range(1, n):
            row = cu[b] + parents[cu[b] + j]
            if probs:
                tokens[cu[b] + j] = rng.choice(vocab, p=q[row].astype(np.float64) / q[row].sum(dtype=np.float64))
            else:
                order = np.argsort(-logits[row], kind="stable")
                tokens[cu[b] + j] = order[min(int(rng.integers(0, 3)), vocab - 1)]
    return {"logits": logits, "tokens": tokens, "parents": parents, "cu": cu, "uniform": rng.random(t).astype(np.float32), "probs": q, "f32": f32}


def _verify(gpu, d, temps, extra=0):
    """The call with `extra` rows of nobody behind the last, against the walk."""
    grow = lambda x, fill: np.concatenate([x, np.full((extra, *x.shape[1:]), fill, x.dtype)])   # noqa: E731
    temps = np.asarray(temps, np.float32)
    logits = D.tensor(grow(d["logits"], 0), gpu)
    t = d["logits"].shape[0] + extra
    path, emitted = (torch.full((t,), -7, dtype=torch.int32, device=gpu) for _ in range(2))
    got = ave.verify_draft(logits if d["f32"] else logits.bfloat16(), D.tensor(grow(d["tokens"], 0), gpu), D.tensor(grow(d["parents"], 0), gpu), D.tensor(d["cu"], gpu),
                           D.tensor(grow(d["uniform"], 0), gpu), D.tensor(temps, gpu), None if d["probs"] is None else D.tensor(grow(d["probs"], 0), gpu),
                           path=path, emitted=emitted)
    assert got[1] is path and got[2] is emitted
    with np.errstate(all="ignore"):
        want = D.verify_all(d["logits"], d["tokens"], d["parents"], d["cu"], d["uniform"], temps, d["probs"])
    for g, w in zip(got, want):
        g = g.cpu().numpy()
        assert np.array_equal(g[:len(w)], w), (g[:40], w[:40])
        assert (g[len(w):] == -7).all()
    return want


@pytest.mark.parametrize("vocab", [1, 2, 63, 1000, 8191, 8192, 8193, 50001])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("counts", [[1], [6], [0, 5, 1, 16, 3]], ids=str)
def test_accepted_nodes(gpu, counts, probs, f32, vocab):
    for seed, chain in ((1, True), (2, False), (3, False)):
        d = _draft(seed, counts, vocab, chain=chain, f32=f32, probs=probs)
        _verify(gpu, d, np.resize([1.0, 0.0, 0.7, 1.5], len(counts)), extra=2)


@pytest.mark.parametrize("probs", [False, True])
def test_many_nodes_many_siblings(gpu, probs):
    """More nodes than a wave has lanes, nodes with dozens of children, the same token among siblings, children far behind their parents."""
    longest = 0
    for seed in range(12):
        d = _draft(seed, [200, 70, 130], 300, probs=probs, sharp=1.0)
        rng = np.random.default_rng(seed + 50)
        for b in range(3):
            n = d["cu"][b + 1] - d["cu"][b]
            d["parents"][d["cu"][b] + 1:d["cu"][b + 1]] = [int(rng.integers(0, max(1, j // 40))) for j in range(1, n)]
        if seed < 6:
            d["uniform"] = np.sqrt(d["uniform"])      # many rejections
        longest = max(longest, _verify(gpu, d, [1.0, 2.0, 0.5])[0].max())
    assert longest >= 2


def test_numbers_at_the_ends(gpu):
    """uniform 0 takes the first token that has a weight, the largest number below 1 and those outside [0, 1) the last; NaN is 0."""
    for seed, u in ((1, 0.0), (2, np.nextafter(np.float32(1), np.float32(0))), (3, 1.0), (4, 7.0), (5, -1.0), (6, np.nan), (7, np.inf)):
        for probs in (False, True):
            d = _draft(seed, [5, 4], 9000, probs=probs)
            d["logits"][:, :5] = d["logits"][:, -5:] = -np.inf
            d["uniform"][:] = u
            _verify(gpu, d, [1.0, 0.8])


@pytest.mark.parametrize("f32", [False, True])
def test_odd_logits(gpu, f32):
    """-inf, +inf, NaN, rows without any number, ties, tiny and huge temperatures, tokens and parents that are none."""
    d = _draft(11, [8, 6, 5, 4, 3, 3], 700, f32=f32)
    x, cu = d["logits"], d["cu"]
    x[::2, 3:600] = -np.inf
    x[1, 10], x[2, 5], x[2, 7], x[3, 4] = np.nan, np.inf, np.inf, np.nan
    x[cu[2]] = -np.inf
    x[cu[3]] = np.nan
    x[cu[4]] = 2.5                       # all equal
    d["tokens"][cu[1] + 1], d["tokens"][cu[1] + 2] = -3, 700
    d["parents"][cu[1] + 3], d["parents"][cu[1] + 4] = 5, -1
    d["parents"][cu[0]] = 2
    for temps in ([1.0] * 6, [0.0] * 6, [-1.0, float("nan"), 0.0, -2.0, 0.0, 1.0], [1e-30, 1e30, 1.0, 1.0, float("inf"), 1e-45]):
        _verify(gpu, d, [t if t == t else 0.0 for t in temps])


@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("vocab", [140001, 600011])
def test_many_pieces(gpu, vocab, probs):
    """More pieces of a row than are looked at together; at temperature 0 equal largest logits far apart, the lowest of which counts; pieces without a number."""
    d = _draft(12, [5, 1, 4], vocab, f32=True, probs=probs)
    for row, at in ((0, (vocab - 1, vocab // 2, 8192 * 3 + 5)), (5, (vocab - 2, 8192 * 16)), (6, (7, vocab - 9))):
        d["logits"][row, list(at)] = 30.0
    d["logits"][2, :8192 * 16] = -np.inf
    d["logits"][7, 8192:] = np.nan
    for temps in ([0.0, 0.0, 0.0], [1.0, 0.6, 2.0]):
        _verify(gpu, d, temps, extra=1)


def test_rejected_with_nothing_left(gpu):
    """Draft distributions above the target's everywhere (no sum of 1), and all of the target's tokens among rejected children."""
    d = _draft(5, [4, 4], 50, probs=True, chain=True)
    d["probs"] = np.full_like(d["probs"], 2.0)
    d["uniform"][[1, 5]] = 0.999
    _verify(gpu, d, [1.0, 1.0])
    d = _draft(6, [4], 3, f32=True)
    d["logits"][:], d["parents"][:], d["tokens"][:] = 0.0, [-1, 0, 0, 0], [0, 0, 1, 2]
    for u in (0.1, 0.5, 0.9, 0.99):
        d["uniform"][:] = u
        _verify(gpu, d, [1.0])
    d = _draft(7, [3], 40, probs=True, chain=True)
    d["probs"][0, ::2], d["probs"][0, 1::2] = np.nan, -1.0       # both count as 0
    _verify(gpu, d, [1.0])


def test_numbers_next_to_a_border(gpu):
    """Random numbers as near as fp32 has them to where the choice changes, on both sides: what 64 bits tell apart, 32 do not."""
    rng = np.random.default_rng(3)
    d = _draft(21, [1] * 64, 30011, f32=True, sharp=2.0)
    hits = 0
    for b in range(64):
        sums = D.softmax(d["logits"][b], 1.0).cumsum()
        at = int(np.searchsorted(sums, rng.random()))
        u = np.float32(sums[at])
        d["uniform"][b] = u
        hits += abs(float(u) - sums[at]) < 2.0 ** -26
    assert hits > 5
    _verify(gpu, d, [1.0] * 64)


@pytest.mark.parametrize("f32", [False, True])
def test_acceptance_next_to_a_border(gpu, f32):
    """The number of a child is the fp32 one nearest to the probability that it is compared with: of a first child, and of a second one behind a rejected one."""
    d = _draft(22, [4] * 48, 20011, f32=f32, sharp=2.0)
    hits = 0
    for b in range(48):
        r = slice(4 * b, 4 * b + 4)
        d["parents"][r] = [-1, 0, 0, 1 + b % 2]
        d["tokens"][r] = np.argsort(-d["logits"][4 * b], kind="stable")[:4]
        p = D.softmax(d["logits"][4 * b], 1.0)[d["tokens"][r]]
        exact = [0, p[1], p[2] / (1 - p[1]), 0]
        d["uniform"][r] = [0.5, p[1] if b % 2 else 1.0, exact[2], 0.5]
        at = 1 if b % 2 else 2
        hits += abs(float(d["uniform"][4 * b + at]) - exact[at]) < 2.0 ** -24 * exact[at]
    assert hits == 48
    want = _verify(gpu, d, [1.0] * 48)
    assert 5 < (want[0] > 1).sum() < 43


@pytest.mark.parametrize("f32", [False, True])
def test_much_to_read(gpu, f32):
    """Rows of more than 64 MB: node 0's first, then those behind the accepted child."""
    d = _draft(31, [14, 1, 20, 12, 17, 0, 9], 270003 if f32 else 500009, f32=f32)
    _verify(gpu, d, [1.0, 0.9, 0.0, 1.0, 0.7, 1.0, 1.0], extra=3)


def test_strided_rows_and_no_temperature(gpu):
    d = _draft(4, [6, 5], 1001, probs=True)
    logits, probs = D.tensor(d["logits"], gpu).bfloat16(), D.tensor(d["probs"], gpu)
    rest = [D.tensor(d[k], gpu) for k in ("tokens", "parents", "cu", "uniform")]
    want = ave.verify_draft(logits, *rest, None, probs)
    wide, wide_probs = torch.zeros(11, 1100, dtype=torch.bfloat16, device=gpu), torch.zeros(11, 1003, device=gpu)
    wide[:, 3:1004], wide_probs[:, 1:1002] = logits, probs
    for x, y in ((wide[:, 3:1004], wide_probs[:, 1:1002]), (logits, wide_probs[:, 1:1002])):
        assert all(torch.equal(a, b) for a, b in zip(ave.verify_draft(x, *rest, torch.ones(2, device=gpu), y), want))


def test_draws_follow_the_target(gpu):
    """What a step emits first is distributed as the target's row, drafts or not: 20000 sequences, a vocabulary of 12.  A frequency f of N draws deviates by
    sqrt(f (1 - f) / N) = 0.0036 at most; five times that for each of 12 tokens and 3 ways goes wrong once in 5e4 runs (and the seed is fixed)."""
    n, v = 20000, 12
    rng = np.random.default_rng(17)
    x = rng.standard_normal(v).astype(np.float32) * 1.5
    p = D.softmax(x, 1.0)
    q = D.softmax(x + rng.standard_normal(v), 1.0).astype(np.float32)
    cu = torch.arange(0, 3 * n + 1, 3, dtype=torch.int32, device=gpu)
    parents = torch.tensor([-1, 0, 0], dtype=torch.int32, device=gpu).repeat(n)
    logits = D.tensor(np.tile(x, (3 * n, 1)), gpu)
    uniform = D.tensor(rng.random(3 * n).astype(np.float32), gpu)
    given = np.tile(np.array([0, 4, 7], np.int32), n)
    drawn = given.copy()
    drawn.reshape(n, 3)[:, 1:] = rng.choice(v, (n, 2), p=q.astype(np.float64) / q.sum(dtype=np.float64))
    for tokens, probs in ((given, None), (drawn, D.tensor(np.tile(q, (3 * n, 1)), gpu))):
        accepted, _, emitted = ave.verify_draft(logits, D.tensor(tokens, gpu), parents, cu, uniform, None, probs)
        assert accepted.min() >= 1 and accepted.max() == 2
        f = np.bincount(emitted.cpu().numpy()[::3], minlength=v) / n
        assert (np.abs(f - p) <= 5 * np.sqrt(p * (1 - p) / n)).all(), (f, p)


# ---- the move of the kept tokens ----------------------------------------------------------------------------------------------------------------
def _kept(rng, n, evict=False):
    many = int(rng.integers(0, n + 1))
    return np.sort(rng.choice(n, many, replace=False)).astype(np.int32)


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("rows", [[(1, 1)], [(8, 8), (16, 100), (5, 33)], [(64, 64), (0, 20), (33, 500)], [(300, 300), (1000, 1500), (7, 90)]], ids=str)
def test_kept_tokens(gpu, rows, d, page):
    """Everything else in the cache stays as it was; tokens move into places that other kept ones leave."""
    rng = np.random.default_rng(d + page)
    batch = A.Batch([(n, k) for n, k in rows], 2, 2, d, page, seed=page)
    layers = [[rng.integers(0, 256, c.shape).astype(np.uint8) for c in batch.cache] for _ in range(3)]
    t = batch.tensors(gpu)
    for case in range(3):
        path, accepted = np.full(int(batch.cu[-1]) + 2, -1, np.int32), []
        for b, (n, _) in enumerate(batch.rows):
            keep = _kept(rng, n) if case < 2 else np.arange(n // 2, n, dtype=np.int32)
            path[batch.cu[b]:batch.cu[b] + len(keep)] = keep
            accepted.append(len(keep))
        lens = np.array([k for _, k in batch.rows], np.int32)
        caches = [tuple(D.tensor(c, gpu) for c in layer) for layer in layers]
        for max_q in (None, 1, 16):
            now = [tuple(c.clone() for c in cache) for cache in caches]
            kept = ave.keep_kv_mxfp4(now if max_q is None or max_q > 1 else list(now), t["page_table"], t["seq_lens"], t["cu_q"], D.tensor(path, gpu),
                                     D.tensor(np.array(accepted, np.int32), gpu), max_q=max_q)
            for got, layer in zip(now, layers):
                want, want_lens = D.keep_tokens(layer, batch.table, lens, batch.cu, path, accepted)
                assert all(np.array_equal(g.cpu().numpy(), w) for g, w in zip(got, want))
            assert np.array_equal(kept.cpu().numpy(), want_lens)


def test_moves_that_name_nothing(gpu):
    """Indices and pages that are none, counts beyond the nodes, lengths below and beyond what there is: nothing moves, and nothing else changes."""
    batch = A.Batch([(6, 40), (6, 40), (6, 3), (6, 100), (6, 40)], 2, 2, 128, 16, seed=1)
    t = batch.tensors(gpu)
    table = batch.table.copy()
    table[1, 2] = -1                      # the page of tokens 32 .. 47
    table[4, 2] = 1 << 20
    lens = np.array([40, 40, 3, 4000, 40], np.int32)
    path = np.tile(np.array([0, 2, 7, -4, 5, 5], np.int32), 5)
    accepted = np.array([9, 6, 6, 6, -2], np.int32)
    for cap in (6, 100000):
        cache = tuple(c.clone() for c in t["cache"])
        kept = ave.keep_kv_mxfp4(cache, D.tensor(table, gpu), D.tensor(lens, gpu), t["cu_q"], D.tensor(path, gpu), D.tensor(accepted, gpu), max_q=cap)
        want, _ = D.keep_tokens([c.copy() for c in batch.cache], table, np.array([40, 40, 3, 4000, 40]), batch.cu, path, accepted)
        places = {i: [batch.place(0, 34 + i)] for i in range(6)}
        for g, w in zip(cache, want):
            assert np.array_equal(g.cpu().numpy(), w), places
        assert kept.tolist() == [40, 40, 3, 4000, 34]


def test_many_layers(gpu):
    """More layers than one launch takes; each layer moves by itself."""
    rng = np.random.default_rng(2)
    batch = A.Batch([(5, 30), (4, 4)], 1, 1, 64, 16, seed=3)
    t = batch.tensors(gpu)
    layers = [[rng.integers(0, 256, c.shape).astype(np.uint8) for c in batch.cache] for _ in range(101)]
    caches = [tuple(D.tensor(c, gpu) for c in layer) for layer in layers]
    path, accepted = np.array([0, 2, 4, -1, -1, 0, 3, -1, -1], np.int32), np.array([3, 2], np.int32)
    kept = ave.keep_kv_mxfp4(caches, t["page_table"], t["seq_lens"], t["cu_q"], D.tensor(path, gpu), D.tensor(accepted, gpu))
    for got, layer in zip(caches, layers):
        want, lens = D.keep_tokens(layer, batch.table, np.array([30, 4]), batch.cu, path, accepted)
        assert all(np.array_equal(g.cpu().numpy(), w) for g, w in zip(got, want))
    assert np.array_equal(kept.cpu().numpy(), lens)


# ---- together ---------------------------------------------------------------------------------------------------------------------------------
def test_a_step_replayed(gpu):
    """Append, attention, acceptance and move as a step uses them, captured once and replayed on other drafts, each against the same calls outside
    a graph; the caches end up equal, too."""
    hq, hkv, d, page, nodes, vocab, b = 8, 2, 128, 16, 12, 3000, 3
    rng = np.random.default_rng(8)
    starts = np.array([40, 7, 100], np.int32)
    g = torch.Generator(device=gpu).manual_seed(1)
    pages = 3 * 12
    table = torch.randperm(pages, generator=g, device=gpu).int().view(3, 12)
    cu = torch.arange(0, b * nodes + 1, nodes, dtype=torch.int32, device=gpu)
    of_row = torch.arange(b, device=gpu).repeat_interleave(nodes)
    state = {"parents": torch.zeros(b * nodes, dtype=torch.int32, device=gpu), "tokens": torch.zeros(b * nodes, dtype=torch.int32, device=gpu),
             "uniform": torch.zeros(b * nodes, device=gpu), "logits": torch.zeros(b * nodes, vocab, dtype=torch.bfloat16, device=gpu),
             "qkv": torch.zeros(b * nodes, hq + 2 * hkv, d, dtype=torch.bfloat16, device=gpu)}
    cos, sin = (D.tensor(x, gpu) for x in A.tables(300, d))

    def step(cache, lens):
        full = lens + nodes
        seen, positions = ave.draft_tree(state["parents"], cu, full, max_q=nodes)
        at = lens[of_row] + torch.arange(nodes, dtype=torch.int32, device=gpu).repeat(b)
        slots = table[of_row].gather(1, (at // page).long()[:, None])[:, 0] * page + at % page
        q, k, v = state["qkv"].split([hq, hkv, hkv], 1)
        q = ave.append_kv_mxfp4(k, v, cache, slots.int(), cos, sin, positions, q=q)
        out = ave.tree_attention_mxfp4(q, cache, table, full, cu, seen, max_q=nodes)
        accepted, path, emitted = ave.verify_draft(state["logits"], state["tokens"], state["parents"], cu, state["uniform"])
        kept = ave.keep_kv_mxfp4(cache, table, full, cu, path, accepted, max_q=nodes)
        lens.copy_(kept)
        return seen, positions, out, accepted, path, emitted

    def draft(i):
        x = _draft(i, [nodes] * b, vocab)
        for k in ("parents", "tokens", "uniform", "logits"):
            state[k].copy_(D.tensor(x[k], gpu))
        state["qkv"].copy_(D.tensor(rng.standard_normal((b * nodes, hq + 2 * hkv, d)).astype(np.float32), gpu))

    caches = [tuple(c.clone() for c in ave.kv_cache_mxfp4(pages, hkv, page, d)) for _ in range(2)]
    lens = [D.tensor(starts, gpu) for _ in range(2)]
    draft(0)
    warm = tuple(c.clone() for c in caches[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(warm, D.tensor(starts, gpu))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        replayed = step(caches[1], lens[1])
    total = 0
    for i in range(5):
        draft(i)
        eager = step(caches[0], lens[0])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(eager, replayed)), i
        assert torch.equal(lens[0], lens[1]) and all(torch.equal(x, y) for x, y in zip(*caches))
        total += int(eager[3].sum())
    assert total > 5 * b and int(lens[0].sum()) == total + int(starts.sum())


def _acceptance(gpu, seed, counts, vocab, probs):
    d = _draft(seed, counts, vocab, probs=probs)
    args = [D.tensor(d["logits"], gpu).bfloat16()] + [D.tensor(d[k], gpu) for k in ("tokens", "parents", "cu", "uniform")]
    return args + [torch.ones(len(counts), device=gpu), D.tensor(d["probs"], gpu) if probs else None]


@pytest.mark.parametrize("counts,vocab,probs", [([6], 9000, False), ([6], 9000, True), ([6] * 70, 20000, False), ([5] * 40, 20000, True), ([14, 1, 20, 12, 17, 0, 9], 500009, False)],
                         ids=["one", "one-probs", "many", "many-probs", "two-steps"])
def test_acceptance_replayed(gpu, counts, vocab, probs):
    """Every order of launches in a graph, on inputs that change between replays."""
    inputs = [_acceptance(gpu, seed, counts, vocab, probs) for seed in (1, 2)]
    held = [None if x is None else x.clone() for x in inputs[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ave.verify_draft(*held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        replayed = ave.verify_draft(*held)
    for i in (1, 0, 1, 1):
        for to, x in zip(held, inputs[i]):
            if x is not None:
                to.copy_(x)
        graph.replay()
        eager = ave.verify_draft(*inputs[i])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(replayed, eager)), i


def test_calls_at_once(gpu):
    """Two streams, each with calls of its own that share nothing, give what the calls give alone."""
    batches = [A.Batch([(40, 300), (9, 2000), (64, 64)], *HEADS["gqa128"], 16, seed=1), A.Batch([(3, 5000), (6, 70)], *HEADS["gqa64"], 64, seed=2)]
    work = []
    for i, batch in enumerate(batches):
        t = batch.tensors(gpu)
        seen, _ = ave.draft_tree(D.tensor(np.concatenate(_parents(batch, 7 + i)), gpu), t["cu_q"], t["seq_lens"], max_q=64)
        work.append((t, seen, _acceptance(gpu, 3 + i, [6] * (70 if i else 2), 20000, bool(i))))

    def calls(t, seen, accept):
        return ave.tree_attention_mxfp4(t["q"], t["cache"], t["page_table"], t["seq_lens"], t["cu_q"], seen, max_q=64), *ave.verify_draft(*accept)

    alone = [[x.clone() for x in calls(*w)] for w in work]
    streams = [torch.cuda.Stream() for _ in work]
    torch.cuda.synchronize()
    results = [[], []]
    for _ in range(10):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                results[i].append(calls(*work[i]))
    torch.cuda.synchronize()
    for got, want in zip(results, alone):
        for run in got:
            live = [torch.equal(a, b) for a, b in zip(run, want)]
            assert all(live), live


def test_both_bindings_agree(gpu, monkeypatch):
    """The entry points in C++ and through ctypes."""
    batch = A.Batch([(9, 60), (20, 200)], *HEADS["gqa128"], 16, seed=6)
    parents = _parents(batch, 8)
    t = batch.tensors(gpu)
    flat = D.tensor(np.concatenate(parents), gpu)
    d = _draft(3, [9, 20], 500, probs=True)
    rest = [D.tensor(d[k], gpu) for k in ("logits", "tokens", "parents", "cu", "uniform")]

    def all_of_them():
        seen, positions = ave.draft_tree(flat, t["cu_q"], t["seq_lens"], max_q=20)
        out = ave.tree_attention_mxfp4(t["q"], t["cache"], t["page_table"], t["seq_lens"], t["cu_q"], seen, max_q=20, window=50)
        accepted, path, emitted = ave.verify_draft(*rest, torch.ones(2, device=gpu), D.tensor(d["probs"], gpu))
        cache = tuple(c.clone() for c in t["cache"])
        kept = ave.keep_kv_mxfp4([cache], t["page_table"], t["seq_lens"], t["cu_q"], path, accepted)
        return seen, positions, out, accepted, path, emitted, kept, *cache

    native = all_of_them()
    none = _lib._NotBuilt("switched off")
    monkeypatch.setattr(attention_module, "_native", none)
    monkeypatch.setattr(drafts_module, "_native", none)
    assert all(torch.equal(x, y) for x, y in zip(native, all_of_them()))
