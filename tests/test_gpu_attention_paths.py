"""How attention's work is divided: each way through the division, at numbers of sequences and items that the other tests do not reach, against fp64;
and norm and rotation against fp64 at every shape."""
import numpy as np
import pytest
import torch

import avelang_amd as ave
from tests import attention_helpers as A
from tests.test_gpu_attention import _check
from tests.test_gpu_kv_cache import SHAPES, _case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("count", [250, 256])
def test_whole_items_in_several_rounds(gpu, d, count):
    """Short prompts, about 2600 blocks of rows for 1024, 768 or 512 workgroups: to and fro, the last round not full, LDS used again by the next item."""
    rng = np.random.default_rng(count + d)
    new = rng.integers(1, 46, count)
    new[[0, 5, count - 1]] = 45, 0, 33
    rows = [(int(n), int(n + k)) for n, k in zip(new, rng.integers(0, 30, count))]
    _check(gpu, A.Batch(rows, 32, 8, d, 16, seed=41), **({"window": 20} if count == 256 else {}))


@pytest.mark.parametrize("rows,heads", [
    ([(40, 2300 - 5 * i) for i in range(12)], (8, 2, 64)), ([(40, 2300 - 5 * i) for i in range(12)], (8, 2, 128)), ([(40, 2300 - 5 * i) for i in range(12)], (8, 2, 256)),
    ([(40 - i % 3, 2300 - 11 * i) if i % 10 else (i % 4, 64 * i) for i in range(70)], (8, 2, 64)), ([(300, 2000), (0, 100)] + [(17, 2100)] * 8 + [(1, 3)], (10, 2, 128))],
    ids=["12x64", "12x128", "12x256", "70x64", "mixed"])
def test_prompts_of_more_than_eight_sequences_in_parts(gpu, rows, heads):
    batch = A.Batch(rows, *heads, 32, seed=42)
    _check(gpu, batch)
    if heads[2] == 64:
        _check(gpu, batch, window=1900, sinks=batch.sinks)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("count", [257, 300, 513])
def test_more_sequences_than_whole_items_are_taken_for(gpu, d, count):
    rng = np.random.default_rng(count)
    keys = rng.integers(0, 90, count)
    keys[[0, 64, 255, 256, count - 1]] = 0, 89, 64, 1, 70
    rows = [(int(rng.integers(0, 20)), int(k)) for k in keys]
    rows[count // 3:count // 3 + 66] = [(0, k) for _, k in rows[count // 3:count // 3 + 66]]     # 64 in a row without work
    _check(gpu, A.Batch(rows, 8, 2, d, 16, seed=43))


@pytest.mark.parametrize("heads", [(8, 2, 64), (8, 2, 128), (6, 2, 256), (40, 1, 128)], ids=str)
@pytest.mark.parametrize("count", [64, 70, 140])
def test_single_tokens_of_many_sequences_in_parts(gpu, heads, count):
    """Tables of more than 2048 tokens, so that items are split, for more sequences than a wave has lanes."""
    rng = np.random.default_rng(count)
    keys = rng.integers(1, 700, count)
    keys[[1, count // 2, count - 1]] = 2200, 0, 1300
    _check(gpu, A.Batch([(1, int(k)) for k in keys], *heads, 64, seed=44))
    if heads[0] == 8:
        _check(gpu, A.Batch([(3 if i % 5 else 0, int(k)) for i, k in enumerate(keys)], *heads, 32, seed=45))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t,hq,hkv,d,rot,norm,neighbours", SHAPES)
def test_norm_and_rotation_of_every_shape_against_fp64(gpu, t, hq, hkv, d, rot, norm, neighbours, dtype):
    dev, _, _, _ = _case(gpu, t, hq, hkv, d, rot, norm, neighbours, dtype, seed=t + d)
    got = ave.qk_norm_rope(dev["q"], dev["k"], dev["cos"], dev["sin"], dev["positions"], dev["q_weight"], dev["k_weight"], eps=A.EPS, neighbours=neighbours)
    for out, name in zip(got, ("q", "k")):
        y = dev[name].double().cpu()
        if norm:
            y = y / (y.pow(2).mean(-1, keepdim=True) + A.EPS).sqrt() * dev[name + "_weight"].double().cpu()
        want, size = y.clone(), y.abs()
        if rot:
            c, s = (dev[n].double().cpu()[dev["positions"].long().cpu()][:, None] for n in ("cos", "sin"))
            a, b = (slice(0, rot, 2), slice(1, rot, 2)) if neighbours else (slice(0, rot // 2), slice(rot // 2, rot))
            want[..., a], want[..., b] = y[..., a] * c - y[..., b] * s, y[..., b] * c + y[..., a] * s
            size[..., a] = size[..., b] = y[..., a].abs() + y[..., b].abs()
        # squares, a tree of at most 8 additions, division, eps, root, division, two products, the rotation's three operations: under 32 roundings
        # of 2^-24; one to bf16
        bound = 2.0 ** -8 * want.abs() + 32 * 2.0 ** -24 * 1.01 * size
        assert ((out.double().cpu() - want).abs() <= bound).all()


@pytest.mark.parametrize("heads", [(8, 2, 64), (10, 2, 128), (6, 2, 256), (40, 1, 128)], ids=str)
def test_a_wrong_bound_on_new_tokens_costs_time_only(gpu, heads):
    for rows in ([(150, 300), (1, 40), (20, 2500)], [(1, 70), (1, 3000)], [(0, 50), (2, 0), (9, 9)]):
        batch = A.Batch(rows, *heads, 32, seed=46)
        t = batch.tensors(gpu)
        for how in ({}, {"window": 70}):
            want, _, tol, _ = batch.reference(**how)
            for max_q in (0, 1, 2, 9, 1000, 2 ** 31 - 1):
                got = ave.attention_mxfp4(t["q"], t["cache"], t["page_table"], t["seq_lens"], t["cu_q"], max_q=max_q, **how)
                assert (np.abs(got.float().cpu().numpy() - want) <= tol).all(), (rows, how, max_q)
