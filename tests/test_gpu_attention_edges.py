"""Attention over an MXFP4 cache and the kernels around it at the edges of what they accept."""
import numpy as np
import pytest
import torch

import avelang_amd as ave
from tests import attention_helpers as A

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("rows", [[(1, 300), (1, 90)], [(5, 300), (3, 90)], [(150, 300), (70, 90)], [(1, 5000)], [(70, 5000)]], ids=str)
def test_a_seen_value_with_a_nan_scale_counts_however_small_its_probability(gpu, d, rows):
    """Scores of hundreds: almost every probability is zero as a number, and still 0 * NaN is NaN.  Rows that do not see the key, and the
    other blocks of channels, keep their bits."""
    hq, hkv, window = 4, 2, 40
    new, keys = rows[0]
    for at_key in (keys - 60, keys - 30, keys - 1):
        for how in ({}, {"window": window}):
            batch, clean = (A.Batch(rows, hq, hkv, d, 32, seed=31, q_std=60.0) for _ in range(2))
            page, at = batch.place(0, at_key)
            batch.cache[3][page, 1, at, d // 32 - 1] = 253
            got, want = (ave.attention_mxfp4(t["q"], t["cache"], t["page_table"], t["seq_lens"], t["cu_q"], max_q=max(n for n, _ in rows), **how)
                         for t in (batch.tensors(gpu), clean.tensors(gpu)))
            position = keys - new + torch.arange(new, device=gpu)
            sees = position >= at_key
            if how:
                sees = sees & (position - window < at_key)
            nan = torch.zeros(got.shape, dtype=torch.bool, device=gpu)
            block = torch.zeros(hq, d, dtype=torch.bool, device=gpu)
            block[2:, d - 32:] = True
            nan[:new] = sees[:, None, None] & block
            assert torch.equal(got.isnan(), nan), (at_key, how)
            assert torch.equal(got[~nan], want[~nan])


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("rows", [[(1, 200)], [(20, 200)], [(150, 200)], [(1, 4000)], [(70, 4000)]], ids=str)
@pytest.mark.parametrize("power", [10, 28, -100])
def test_large_and_small_scores(gpu, d, rows, power):
    """Every key is the same and every product -2^power: the mean of the values that a row sees.  (Beyond 2^30 fp32 has no bits left for what
    a score differs by.)"""
    hq, hkv = 4, 2
    batch = A.Batch(rows, hq, hkv, d, 32, seed=32)
    batch.cache[0][:] = 0x22                      # ones
    batch.cache[1][:] = 127
    batch.q[:] = -(2.0 ** power / d)
    new, keys = rows[0]
    n = keys - new + 1 + np.arange(new)
    for scale in (0.125, 1.0, float(np.log(2.0))):
        t = batch.tensors(gpu)
        lse = torch.full(batch.q.shape[:2], float("nan"), device=gpu)
        got = ave.attention_mxfp4(t["q"], t["cache"], t["page_table"], t["seq_lens"], t["cu_q"], None, lse, max_q=new, scale=scale)
        got = got.double().cpu().numpy().reshape(new, hkv, -1, d)
        for i in range(new):
            v, size = (x[:n[i]].mean(0)[:, None] for x in (batch.v[0], np.abs(batch.v[0])))       # [hkv, 1, d]
            # all probabilities are equal, one rounding (2^-9 of the numerator at most) apart from the sum's; fp32 sums of at most 128 steps
            # a lane and the result's rounding
            assert (np.abs(got[i] - v) <= 2.0 ** -8 * np.abs(v) + (2.0 ** -8 + 2.0 ** -16) * size).all(), (i, scale)
        want = -scale * 2.0 ** power + np.log(n)
        assert np.allclose(lse.double().cpu().numpy(), want[:, None], rtol=2.0 ** -20, atol=2.0 ** -16)


def test_windows_beyond_31_bits(gpu):
    batch = A.Batch([(1, 300), (40, 90)], 4, 2, 64, 16, seed=33)
    t = batch.tensors(gpu)
    call = lambda **kw: ave.attention_mxfp4(t["q"], t["cache"], t["page_table"], t["seq_lens"], t["cu_q"], **{"max_q": 40, **kw})   # noqa: E731
    want = call()
    for window in (2 ** 31 - 1, 2 ** 31, 2 ** 32 + 5, 2 ** 40 + 1, 2 ** 70):
        assert torch.equal(call(window=window), want), window
    assert torch.equal(call(max_q=2 ** 32 + 40), want)
    for window in (-1, -2 ** 31 - 1, -2 ** 32, 1 - 2 ** 32):
        with pytest.raises(ValueError, match="window must be non-negative"):
            call(window=window)
    with pytest.raises(ValueError, match="max_q"):
        call(max_q=-2 ** 32 + 1)


def test_more_than_2_to_the_24_tokens(gpu):
    """Head kernels take a workgroup a token: more workgroups than one launch may have threads for."""
    t, d, rows = (1 << 24) + 37, 64, 64
    x = torch.randn(rows, 1, d, generator=torch.Generator().manual_seed(1)).bfloat16().to(gpu)
    cos, sin = (torch.from_numpy(c).to(gpu) for c in A.tables(rows, d))
    pos = (torch.arange(t, device=gpu) % rows).int()
    many = x.repeat(t // rows + 1, 1, 1)[:t]
    out, _ = ave.qk_norm_rope(many, None, cos, sin, pos)
    want, _ = ave.qk_norm_rope(x, None, cos, sin, pos[:rows].contiguous())
    whole = t // rows * rows
    assert (out[:whole].view(-1, rows, 1, d) == want).all() and torch.equal(out[whole:], want[:t - whole])
    del out
    # appended: the last tokens alone are stored
    cache = ave.kv_cache_mxfp4(4, 1, 16, d, gpu)
    slots = torch.full((t,), -1, dtype=torch.int32, device=gpu)
    slots[-rows:] = torch.arange(rows, dtype=torch.int32, device=gpu)
    ave.append_kv_mxfp4(many, many, cache, slots, cos, sin, pos)
    last = many[-rows:].contiguous()
    small = ave.kv_cache_mxfp4(4, 1, 16, d, gpu)
    ave.append_kv_mxfp4(last, last, small, torch.arange(rows, dtype=torch.int32, device=gpu), cos, sin, pos[-rows:].contiguous())
    assert all(torch.equal(a, b) for a, b in zip(cache, small))


def test_more_than_2_to_the_32_units(gpu):
    """257 single tokens of 1024 heads over 2^20 keys, which are the same 64 keys again and again (one page): units of 64 keys."""
    heads, d, page, batch, keys = 1024, 64, 64, 257, 1 << 20
    g = torch.Generator().manual_seed(34)
    cache = ave.kv_cache_mxfp4(1, heads, page, d, gpu)
    kv = torch.randn(2, page, heads, d, generator=g).to(gpu)
    ave.append_kv_mxfp4(kv[0], kv[1], cache, torch.arange(page, dtype=torch.int32, device=gpu))
    q = torch.randn(1, heads, d, generator=g).bfloat16().to(gpu)
    lens = torch.full((batch,), keys, dtype=torch.int32, device=gpu)
    lens[::7] += 1 - page                                      # not every one of them a whole number of pages
    table = torch.zeros(1, keys // page, dtype=torch.int32, device=gpu).expand(batch, -1)
    out = torch.full((batch, heads, d), float("nan"), dtype=torch.bfloat16, device=gpu)
    ave.attention_mxfp4(q.expand(batch, -1, -1), cache, table, lens, out=out)
    k, v = (x.double().cpu() for x in ave.gather_kv_mxfp4(cache, torch.arange(page, dtype=torch.int32, device=gpu)))
    p = torch.softmax((k * q.double().cpu()).sum(-1) * d ** -0.5, 0)[..., None]
    want, weight = (p * v).sum(0), (p * v.abs()).sum(0)
    # the result's rounding and a probability's; two fp32 sums of 2^16 steps a lane; the last page counting in part, one of 2^14
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2 * 2.0 ** -24 * 2 ** 16) * weight + 2.0 ** -13 * (weight + v.abs().amax(0))
    err = (out.double().cpu() - want).abs()
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 2, 40])
def test_tables_wide_enough_for_units_beyond_32_bits(gpu, d, new):
    """The width of the page table alone decides how units are numbered, so that short sequences reach the 64-bit forms, too."""
    hq, hkv, page = 16, 8, 4096
    rows = [(new, (2400 if new > 2 else 600) - 7 * i) for i in range(12)] + [(new, 3000), (0, 9), (new, 3), (new, 64)]
    batch = A.Batch(rows, hq, hkv, d, page, seed=35)
    t = batch.tensors(gpu)
    wide = torch.full((len(rows), (1 << 31) // page - 1), 1 << 30, dtype=torch.int32, device=gpu)
    wide[:, :t["page_table"].shape[1]] = t["page_table"]
    want, want_lse, tol, lse_tol = batch.reference()
    outs = []
    for table in (t["page_table"], wide):
        lse = torch.full(batch.q.shape[:2], float("nan"), device=gpu)
        out = torch.full(batch.q.shape, float("nan"), dtype=torch.bfloat16, device=gpu)
        ave.attention_mxfp4(t["q"], t["cache"], table, t["seq_lens"], t["cu_q"], out, lse, max_q=new)
        assert (np.abs(out.float().cpu().numpy() - want) <= tol).all()
        some = np.isfinite(want_lse)
        assert np.array_equal(lse.cpu().numpy()[~some], want_lse[~some])
        assert (np.abs(lse.cpu().numpy()[some] - want_lse[some]) <= lse_tol[some]).all()
        outs.append(out)
    if new == 40:
        assert torch.equal(*outs)      # the kernel for prompts: the same parts either way


def test_tokens_that_share_a_slot_leave_the_others_alone(gpu):
    """Padding that is all sent to one slot: that one's contents are undefined, every other token is in its place."""
    heads, d, page, t = 3, 128, 16, 1500
    g = torch.Generator().manual_seed(36)
    k, v = (torch.randn(t, heads, d, generator=g).bfloat16().to(gpu) for _ in range(2))
    slots = torch.randperm(2000, generator=g)[:t].int().to(gpu)
    shared = int(slots[0])
    slots[::3] = shared
    one, other = (ave.kv_cache_mxfp4(125, heads, page, d, gpu) for _ in range(2))
    ave.append_kv_mxfp4(k, v, one, slots)
    keep = slots != shared
    ave.append_kv_mxfp4(k[keep].contiguous(), v[keep].contiguous(), other, slots[keep].contiguous())
    for a, b in zip(one, other):
        a, b = (x.transpose(1, 2).flatten(0, 1) for x in (a, b))
        a, b = (torch.cat([x[:shared], x[shared + 1:]]) for x in (a, b))
        assert torch.equal(a, b)
