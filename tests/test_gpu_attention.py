"""Attention over an MXFP4 cache against fp64, at the lengths, shapes and masks where it can go wrong."""
import numpy as np
import pytest
import torch

import avelang_amd as ave
from avelang_amd import _lib, attention as mod
from tests import attention_helpers as A

pytestmark = pytest.mark.gpu

HEADS = {"gqa64": (8, 2, 64), "gqa128": (8, 2, 128), "gqa256": (6, 2, 256), "mha128": (3, 3, 128), "group5": (10, 2, 128), "mqa64": (24, 1, 64),
         "group40": (40, 1, 128), "mha64": (2, 2, 64), "mqa256": (8, 1, 256)}


def _check(gpu, batch, **how):
    t = batch.tensors(gpu)
    sinks = how.get("sinks")
    lse = torch.full((batch.q.shape[0], batch.hq), float("nan"), device=gpu)
    out = torch.full(batch.q.shape, float("nan"), dtype=torch.bfloat16, device=gpu)
    kw = {k: v for k, v in how.items() if k != "sinks"}
    got = ave.attention_mxfp4(t["q"], t["cache"], t["page_table"], t["seq_lens"], t["cu_q"], out, lse,
                              max_q=max([n for n, _ in batch.rows]), sinks=torch.from_numpy(sinks).to(gpu) if sinks is not None else None, **kw)
    assert got is out
    want, want_lse, tol, lse_tol = batch.reference(**how)
    err = np.abs(out.float().cpu().numpy() - want)
    assert (err <= tol).all(), (float((err / tol).max()), np.argwhere(~(err <= tol))[:5].tolist())
    le = lse.cpu().numpy()
    some = np.isfinite(want_lse)
    assert np.array_equal(le[~some], want_lse[~some])
    assert (np.abs(le[some] - want_lse[some]) <= lse_tol[some]).all(), float((np.abs(le[some] - want_lse[some]) - lse_tol[some]).max())
    return t, out


DECODE = [[(1, 1)], [(1, 2), (1, 15), (1, 16), (1, 17)], [(1, 63), (1, 64), (1, 65), (1, 127), (1, 128), (1, 129)], [(1, 300)], [(1, 1000), (1, 1), (1, 511)]]


@pytest.mark.parametrize("rows", DECODE, ids=str)
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("heads", HEADS)
def test_single_tokens(gpu, heads, page, rows):
    batch = A.Batch(rows, *HEADS[heads], page, seed=page + len(rows))
    t, out = _check(gpu, batch)
    same = ave.attention_mxfp4(t["q"], t["cache"], t["page_table"], t["seq_lens"])   # without cu_q: one token each
    assert torch.equal(same, out)


SEVERAL = [[(4, 4), (3, 100), (1, 1)], [(2, 1000), (5, 64), (8, 8)], [(70, 70), (1, 257), (33, 130)], [(200, 200)], [(130, 300), (0, 50), (2, 50)],
           [(1, 700), (257, 257)]]


@pytest.mark.parametrize("rows", SEVERAL, ids=str)
@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("heads", HEADS)
def test_several_tokens_and_prompts(gpu, heads, page, rows):
    _check(gpu, A.Batch(rows, *HEADS[heads], page, seed=page + rows[0][1]))


@pytest.mark.parametrize("rows", [[(1, 400), (1, 30)], [(5, 300), (2, 3)], [(150, 200), (40, 500), (1, 90)]], ids=str)
@pytest.mark.parametrize("how", [{"window": 1}, {"window": 7}, {"window": 64}, {"window": 100, "sinks": True}, {"sinks": True}, {"causal": False},
                                 {"scale": 0.5}, {"scale": -0.25, "sinks": True}, {"scale": 0.0}, {"window": 1 << 30}], ids=str)
@pytest.mark.parametrize("heads", ["gqa64", "gqa128", "gqa256", "group5"])
def test_windows_sinks_scales(gpu, heads, how, rows):
    batch = A.Batch(rows, *HEADS[heads], 32, seed=3)
    _check(gpu, batch, **{k: batch.sinks if k == "sinks" else v for k, v in how.items()})


@pytest.mark.parametrize("heads", ["gqa64", "gqa128", "mqa256"])
def test_rows_that_see_nothing(gpu, heads):
    """More new tokens than keys (the first stand before the sequence's start), and sequences without keys."""
    batch = A.Batch([(1, 0), (5, 3), (90, 20), (2, 0), (1, 5)], *HEADS[heads], 16, seed=4)
    _, out = _check(gpu, batch)
    assert out[0].eq(0).all() and out[1:3].eq(0).all() and not out[3].eq(0).all()
    _check(gpu, batch, sinks=batch.sinks)
    _check(gpu, batch, window=2)


@pytest.mark.parametrize("heads", ["gqa64", "gqa128", "gqa256"])
def test_sharp_distributions(gpu, heads):
    """Scores of tens and hundreds: the running maximum moves, and almost all of the weight is on few keys."""
    _check(gpu, A.Batch([(1, 900), (1, 33), (3, 500)], *HEADS[heads], 64, seed=5, q_std=4.0))
    _check(gpu, A.Batch([(100, 300)], *HEADS[heads], 64, seed=6, q_std=12.0))


def test_long_sequences_split_over_workgroups(gpu):
    for rows, heads in (([(1, 20000)], (8, 2, 128)), ([(1, 9000), (1, 100), (1, 5000)], (16, 2, 64)), ([(3, 6000)], (4, 1, 256)), ([(64, 5000)], (4, 1, 128))):
        _check(gpu, A.Batch(rows, *heads, 64, seed=7))


def test_results_do_not_depend_on_the_workspace_or_the_run(gpu):
    """The same bits twice, whatever the workspace held."""
    for rows, heads in (([(1, 5000), (1, 70)], (8, 2, 128)), ([(100, 3000), (1, 900)], (8, 2, 128)), ([(1, 3000)], (8, 1, 64))):
        t = A.Batch(rows, *heads, 64, seed=8).tensors(gpu)
        c, _ = mod._cache(t["cache"])
        lib = _lib.load()
        outs = []
        for fill in (0x00, 0xFF, 0x7F):
            out = torch.empty(t["q"].shape, dtype=torch.bfloat16, device=gpu)
            a = _lib.Attention(q=t["q"].data_ptr(), q_token_stride=t["q"].stride(0), q_head_stride=t["q"].stride(1), out=out.data_ptr(),
                               page_table=t["page_table"].data_ptr(), page_table_stride=t["page_table"].stride(0), seq_lens=t["seq_lens"].data_ptr(),
                               cu_q=t["cu_q"].data_ptr(), tokens=out.shape[0], batch=len(rows), heads=heads[0], table_pages=t["page_table"].shape[1],
                               max_q=max(n for n, _ in rows), causal=1, scale=heads[2] ** -0.5)
            need = lib.ave_fp4_attention_mxfp4_workspace_bytes(mod._ref(a), mod._ref(c))
            ws = torch.full((max(need, 16),), fill, dtype=torch.uint8, device=gpu)
            _lib.check(lib.ave_fp4_attention_mxfp4(mod._ref(a), mod._ref(c), ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream))
            outs.append(out)
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
        assert torch.equal(outs[0], ave.attention_mxfp4(t["q"], t["cache"], t["page_table"], t["seq_lens"], t["cu_q"], max_q=max(n for n, _ in rows)))


def test_strided_queries_tables_and_caches(gpu):
    batch = A.Batch([(1, 200), (3, 90), (40, 64)], 8, 2, 128, 16, seed=9)
    t, out = _check(gpu, batch)
    n = out.shape[0]
    wide = torch.zeros(n, 8 + 5, 128 + 1, dtype=torch.bfloat16, device=gpu)       # odd strides: no row is aligned
    wide[:, 2:10, 1:].copy_(t["q"])
    table = torch.full((3, t["page_table"].shape[1] + 9), -7, dtype=torch.int32, device=gpu)
    table[:, 3:3 + t["page_table"].shape[1]] = t["page_table"]
    pages = t["cache"][0].shape[0]
    layers = tuple(torch.zeros(pages, 3, *c.shape[1:], dtype=torch.uint8, device=gpu) for c in t["cache"])   # pages of three layers side by side
    for big, c in zip(layers, t["cache"]):
        big[:, 1].copy_(c)
    got = ave.attention_mxfp4(wide[:, 2:10, 1:], tuple(b[:, 1] for b in layers), table[:, 3:3 + t["page_table"].shape[1]], t["seq_lens"], t["cu_q"], max_q=40)
    assert torch.equal(got, out)
    # without a bound on the new tokens the result may come from another kernel: the same within the tolerance
    got = ave.attention_mxfp4(t["q"], t["cache"], t["page_table"], t["seq_lens"], t["cu_q"])
    want, _, tol, _ = batch.reference()
    assert (np.abs(got.float().cpu().numpy() - want) <= tol).all()


@pytest.mark.parametrize("rows", [[(1, 100), (1, 60)], [(50, 100), (70, 70)]], ids=str)
def test_nan_and_infinity(gpu, rows):
    """A NaN scale of a key makes every row that sees it NaN, of a value its 32 channels; a NaN or infinity in a query its row.  What a row
    does not see has no effect."""
    new, keys = rows[0]
    for part in (1, 3):
        batch = A.Batch(rows, 4, 2, 128, 16, seed=10)
        clean = A.Batch(rows, 4, 2, 128, 16, seed=10)
        page, at = batch.place(0, keys - 20)
        batch.cache[part][page, 1, at, 2] = 0xFF
        t, c = batch.tensors(gpu), clean.tensors(gpu)
        call = lambda x: ave.attention_mxfp4(x["q"], x["cache"], x["page_table"], x["seq_lens"], x["cu_q"], max_q=new)   # noqa: E731
        got, want = call(t), call(c)
        sees = torch.zeros(got.shape, dtype=torch.bool, device=gpu)
        first = max(0, new - 20)                       # the first row that stands at or behind the key
        if part == 1:
            sees[first:new, 2:] = True
        else:
            sees[first:new, 2:, 64:96] = True
        if new > 1:
            sees[:new - 20] = False
            sees[new - 20:new, 2:, (slice(None) if part == 1 else slice(64, 96))] = True
        assert got[sees].isnan().all() and torch.equal(got[~sees], want[~sees])
    batch = A.Batch(rows, 4, 2, 128, 16, seed=11)
    t = batch.tensors(gpu)
    want = ave.attention_mxfp4(t["q"], t["cache"], t["page_table"], t["seq_lens"], t["cu_q"], max_q=new)
    t["q"][0, 1, 5], t["q"][new, 3, 100] = float("inf"), float("nan")
    got = ave.attention_mxfp4(t["q"], t["cache"], t["page_table"], t["seq_lens"], t["cu_q"], max_q=new)
    assert got[0, 1].isnan().all() and got[new, 3].isnan().all()
    keep = torch.ones(got.shape[:2], dtype=torch.bool, device=gpu)
    keep[0, 1] = keep[new, 3] = False
    assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("rows", [[(1, 150), (1, 40)], [(60, 150)]], ids=str)
def test_extreme_scales(gpu, rows):
    """Values between 2^-100 and 2^100 beside each other, keys of 2^-60: probabilities and scales multiply without leaving their range."""
    batch = A.Batch(rows, 4, 2, 64, 16, seed=12)
    rng = np.random.default_rng(13)
    for b, (_, keys) in enumerate(rows):
        for j in range(keys):
            page, at = batch.place(b, j)
            up = rng.integers(-100, 101, (2, 2))
            batch.cache[3][page, :, at] = (batch.cache[3][page, :, at].astype(int) + up).astype(np.uint8)
            batch.v[b][j] *= np.repeat(np.exp2(up.astype(float)), 32, axis=-1).reshape(2, 64)
            if j % 3 == 0:
                batch.cache[1][page, :, at] -= 60
                batch.k[b][j] *= 2.0 ** -60
    _check(gpu, batch)


def test_hidden_values_of_the_largest_scale_have_no_effect(gpu):
    """Keys behind a row's position hold values of 2^125 and more: an exact zero is what they count."""
    rows = [(30, 100)]
    batch = A.Batch(rows, 4, 2, 128, 16, seed=14)
    t, out = _check(gpu, batch)
    for j in range(71, 100):
        page, at = batch.place(0, j)
        batch.cache[3][page, :, at] = 254
    t = batch.tensors(gpu)
    got = ave.attention_mxfp4(t["q"], t["cache"], t["page_table"], t["seq_lens"], t["cu_q"], max_q=30)
    assert torch.equal(got[0], out[0])
    one = ave.attention_mxfp4(t["q"][:1], t["cache"], t["page_table"], t["seq_lens"] - 29, max_q=1)
    want, _, tol, _ = A.Batch(rows, 4, 2, 128, 16, seed=14).reference()
    assert (np.abs(one.float().cpu().numpy() - want[:1]) <= tol[:1]).all()


def test_offsets_beyond_32_bits(gpu):
    """Three pages a little over 2 GiB apart."""
    batch = A.Batch([(1, 170), (20, 20)], 4, 2, 128, 64, seed=15, spare=0)
    t, out = _check(gpu, batch)
    pages = t["cache"][0].shape[0]
    gap = (1 << 31) + 4096
    buf = torch.zeros((pages - 1) * gap + (1 << 20), dtype=torch.uint8, device=gpu)
    cache, at = [], 0
    for c in t["cache"]:
        view = buf[at:].as_strided(tuple(c.shape), (gap, *c.stride()[1:]))
        view.copy_(c)
        cache.append(view)
        at += c[0].numel()
    got = ave.attention_mxfp4(t["q"], tuple(cache), t["page_table"], t["seq_lens"], t["cu_q"], max_q=20)
    assert torch.equal(got, out)


def test_untrusted_tables_stay_inside_the_cache(gpu):
    """Lengths beyond the table, pages outside the cache, rows outside q: nothing faults, and the other sequences are untouched."""
    batch = A.Batch([(1, 90), (1, 60), (1, 40)], 4, 2, 64, 16, seed=16)
    t, out = _check(gpu, batch)
    lens = t["seq_lens"].clone()
    lens[0], lens[2] = 2 ** 31 - 1, -5
    table = t["page_table"].clone()
    table[0, 2], table[0, 3] = -1, 2 ** 31 - 1
    got = ave.attention_mxfp4(t["q"], t["cache"], table, lens)
    assert torch.equal(got[1], out[1]) and got[2].eq(0).all()
    cu = torch.tensor([0, 1, 2, 2 ** 31 - 1], dtype=torch.int32, device=gpu)
    got = ave.attention_mxfp4(t["q"], t["cache"], t["page_table"], t["seq_lens"], cu, max_q=1)
    assert torch.equal(got[1], out[1])
    cu = torch.tensor([-3, 1, 0, 3], dtype=torch.int32, device=gpu)
    ave.attention_mxfp4(t["q"], t["cache"], t["page_table"], t["seq_lens"], cu, max_q=1)
    torch.cuda.synchronize()


def test_another_stream_and_graph_replays(gpu):
    """A decode step (append, attention) captured once and replayed while lengths, slots and positions move on."""
    hq, hkv, d, page, steps = 8, 2, 128, 16, 5
    batch = A.Batch([(1, 30), (1, 47)], hq, hkv, d, page, seed=17, spare=4)
    t = batch.tensors(gpu)
    table = t["page_table"].clone()
    table[0, 2], table[1, 3] = 100, 100                     # room for growth: set below
    free = sorted(set(range(t["cache"][0].shape[0])) - set(table[table < (1 << 30)].cpu().tolist()))
    table[0, 2], table[1, 3] = free[0], free[1]
    rng = torch.Generator(device="cpu").manual_seed(1)
    qkv = torch.randn(steps, 2, hq + 2 * hkv, d, generator=rng).bfloat16().to(gpu)
    cos, sin = (torch.from_numpy(x).to(gpu) for x in A.tables(100, d))

    def step(x, cache, lens):
        pos = lens - 1
        slots = table.gather(1, (pos // page).long()[:, None])[:, 0] * page + pos % page
        q = ave.append_kv_mxfp4(x[:, hq:hq + hkv], x[:, hq + hkv:], cache, slots, cos, sin, pos, q=x[:, :hq])
        return ave.attention_mxfp4(q, cache, table, lens)

    eager = tuple(c.clone() for c in t["cache"])
    want = []
    for i in range(steps):
        want.append(step(qkv[i], eager, t["seq_lens"] + i + 1))
    cache, x, lens = tuple(c.clone() for c in t["cache"]), qkv[0].clone(), t["seq_lens"] + 1
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, tuple(c.clone() for c in cache), lens)      # first launches outside the capture
        other = step(x, tuple(c.clone() for c in cache), lens)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x, cache, lens)
    for i in range(steps):
        x.copy_(qkv[i])
        lens.copy_(t["seq_lens"] + i + 1)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i]), i
        torch.randn(1000, device=gpu).sum().item()          # the program's own work between replays
    assert all(torch.equal(a, b) for a, b in zip(cache, eager))


def test_the_wrapper_and_the_extension_agree(gpu, monkeypatch):
    batch = A.Batch([(1, 100), (30, 30)], 8, 2, 128, 16, seed=18)
    t = batch.tensors(gpu)
    cache = ave.kv_cache_mxfp4(4, 2, 16, 128, gpu)
    slots = torch.arange(31, dtype=torch.int32, device=gpu)
    cos, sin = (torch.from_numpy(x).to(gpu) for x in A.tables(100, 64))
    w = torch.rand(128, device=gpu)
    kv = t["q"][:, :2]
    lse = torch.empty(31, 8, device=gpu)

    def calls():
        c = tuple(x.clone() for x in cache)
        return [ave.qk_norm_rope(t["q"], kv, cos, sin, slots, w, w, eps=1e-5, neighbours=True),
                (ave.append_kv_mxfp4(kv, kv, c, slots, cos, sin, slots, w, q=t["q"], q_weight=w), *c), ave.gather_kv_mxfp4(c, slots),
                (ave.attention_mxfp4(t["q"], t["cache"], t["page_table"], t["seq_lens"], t["cu_q"], None, lse, max_q=30, window=9, sinks=w[:8].contiguous()), lse.clone())]

    native = calls()
    monkeypatch.setattr(mod, "_native", type("Slow", (), {"__getattr__": lambda self, name: lambda *args: None})())
    for a, b in zip(native, calls()):
        assert len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


def test_nothing_to_do(gpu):
    cache = ave.kv_cache_mxfp4(1, 2, 16, 64, gpu)
    q = torch.empty(0, 4, 64, dtype=torch.bfloat16, device=gpu)
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device=gpu)   # noqa: E731
    assert ave.attention_mxfp4(q, cache, i(0, 1), i(0)).shape == (0, 4, 64)
    assert ave.attention_mxfp4(q, cache, i(3, 1), i(3), i(4), max_q=2).shape == (0, 4, 64)
    q = torch.ones(2, 4, 64, dtype=torch.bfloat16, device=gpu)
    assert ave.attention_mxfp4(q, cache, i(2, 0), i(2) + 5).eq(0).all()      # a table without pages: no keys


@pytest.mark.parametrize("heads", ["gqa64", "gqa128"])
@pytest.mark.parametrize("count", [17, 65, 150])
def test_many_sequences(gpu, heads, count):
    """More sequences than a wave has lanes, empty ones among them; single tokens, then several each."""
    rng = np.random.default_rng(count)
    keys = rng.integers(0, 90, count)
    keys[[0, count // 2, count - 1]] = 0, 89, 1
    _check(gpu, A.Batch([(1, int(k)) for k in keys], *HEADS[heads], 16, seed=20))
    _check(gpu, A.Batch([(int(rng.integers(0, 20)), int(k)) for k in keys], *HEADS[heads], 16, seed=21))


@pytest.mark.parametrize("heads", ["gqa64", "gqa128", "gqa256"])
@pytest.mark.parametrize("rows", [[(1, 2500)], [(9, 2500), (1, 10)], [(40, 2500)]], ids=str)
def test_maxima_that_climb(gpu, heads, rows):
    """Keys that grow towards the sequence's end: what is subtracted from the scores has to follow, again and again."""
    hq, hkv, d = HEADS[heads]
    batch = A.Batch(rows, hq, hkv, d, 32, seed=22)
    for b, (_, keys) in enumerate(rows):
        for j in range(keys):
            page, at = batch.place(b, j)
            up = j // 250
            batch.cache[1][page, :, at] += up
            batch.k[b][j] *= 2.0 ** up
    _check(gpu, batch, scale=d ** -0.5 / 16)


@pytest.mark.parametrize("heads", ["gqa64", "gqa128", "gqa256"])
def test_few_blocks_of_many_parts(gpu, heads):
    """One block of rows over a long cache: its keys are shared by many workgroups; one row, a few, more than a block."""
    for new in (1, 6, 40):
        _check(gpu, A.Batch([(new, 6000)], *HEADS[heads], 256, seed=23 + new))
    batch = A.Batch([(33, 3001)], *HEADS[heads], 64, seed=24)
    _check(gpu, batch, window=2200, sinks=batch.sinks)


def test_prompts_beyond_32_bit_offsets(gpu):
    batch = A.Batch([(60, 170), (1, 20)], 4, 2, 128, 64, seed=25, spare=0)
    t, out = _check(gpu, batch)
    gap = (1 << 31) + 4096
    buf = torch.zeros((t["cache"][0].shape[0] - 1) * gap + (1 << 20), dtype=torch.uint8, device=gpu)
    cache, at = [], 0
    for c in t["cache"]:
        view = buf[at:].as_strided(tuple(c.shape), (gap, *c.stride()[1:]))
        view.copy_(c)
        cache.append(view)
        at += c[0].numel()
    got = ave.attention_mxfp4(t["q"], tuple(cache), t["page_table"], t["seq_lens"], t["cu_q"], max_q=60)
    assert torch.equal(got, out)


def test_untrusted_prompts_stay_inside_the_cache(gpu):
    """The same as for single tokens: lengths, pages and row ranges that do not fit; the sequence that does is untouched."""
    batch = A.Batch([(40, 90), (50, 60), (20, 40)], 4, 2, 64, 16, seed=26)
    t, out = _check(gpu, batch)
    lens, table = t["seq_lens"].clone(), t["page_table"].clone()
    lens[0], lens[2] = 2 ** 31 - 1, -5
    table[0, 2], table[0, 3] = -1, 2 ** 31 - 1
    got = ave.attention_mxfp4(t["q"], t["cache"], table, lens, t["cu_q"], max_q=50)
    assert torch.equal(got[40:90], out[40:90]) and got[90:].eq(0).all()
