"""Norm and rotation of query and key heads, appending to an MXFP4 cache and reading it back: codes and scales bit for bit against
single fp32 operations in numpy and the oracle's quantiser; bf16 results within one rounding of fp64."""
import numpy as np
import pytest
import torch

import avelang_amd as ave
from oracle import fp4_oracle as orc
from tests import attention_helpers as A

pytestmark = pytest.mark.gpu


def _dev(x, gpu):
    return torch.from_numpy(np.ascontiguousarray(x)).to(gpu)


def _case(gpu, t, hq, hkv, d, rot, norm, neighbours, dtype, seed, rows=600):
    """A packed projection ``[T, hq + 2 hkv, d]``, its tables and weights; numpy and device side."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((t, hq + 2 * hkv, d)).astype(np.float32) * np.exp2(rng.integers(-6, 7, (t, hq + 2 * hkv, 1))).astype(np.float32)
    if dtype == torch.bfloat16:
        x = A.bf16(x)
    cos, sin = A.tables(rows, rot) if rot else (None, None)
    pos = rng.integers(0, rows, t).astype(np.int32)
    wq, wk = (A.bf16(1 + 0.3 * rng.standard_normal(d)) if norm else None for _ in range(2))
    packed = _dev(x, gpu).to(dtype)
    dev = {"q": packed[:, :hq], "k": packed[:, hq:hq + hkv], "v": packed[:, hq + hkv:],
           "cos": _dev(cos, gpu) if rot else None, "sin": _dev(sin, gpu) if rot else None, "positions": _dev(pos, gpu) if rot else None,
           "q_weight": _dev(wq, gpu).bfloat16() if norm else None, "k_weight": _dev(wk, gpu).bfloat16() if norm else None}
    q = A.norm_rope_f32(x[:, :hq], wq, cos, sin, pos, neighbours)
    k = A.norm_rope_f32(x[:, hq:hq + hkv], wk, cos, sin, pos, neighbours)
    return dev, q, k, x[:, hq + hkv:]


def _bits(t):
    return t.contiguous().view(torch.int16).cpu().numpy().view(np.uint16)


SHAPES = [(1, 32, 8, 128, 128, True, False), (7, 3, 1, 64, 64, True, False), (130, 8, 8, 128, 64, True, True), (33, 4, 2, 256, 256, False, False),
          (5, 5, 5, 256, 96, True, False), (64, 16, 2, 64, 16, False, True), (2000, 4, 1, 128, 128, True, False), (9, 2, 2, 128, 0, True, False)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t,hq,hkv,d,rot,norm,neighbours", SHAPES)
def test_norm_and_rotation(gpu, t, hq, hkv, d, rot, norm, neighbours, dtype):
    dev, q, k, _ = _case(gpu, t, hq, hkv, d, rot, norm, neighbours, dtype, seed=t + d)
    args = (dev["cos"], dev["sin"], dev["positions"], dev["q_weight"], dev["k_weight"])
    q_out, k_out = ave.qk_norm_rope(dev["q"], dev["k"], *args, eps=A.EPS, neighbours=neighbours)
    assert np.array_equal(_bits(q_out), orc.f32_to_bf16_bits(q)) and np.array_equal(_bits(k_out), orc.f32_to_bf16_bits(k))
    # fp64: the products and sums of fp32 (2^-23 of the pair's magnitude, norm included a few of them) and one rounding
    # one side alone, through a strided output
    wide = torch.full((t, hq + 3, d), float("nan"), dtype=torch.bfloat16, device=gpu)
    q_only, none = ave.qk_norm_rope(dev["q"], None, *args[:4], q_out=wide[:, 1:hq + 1], eps=A.EPS, neighbours=neighbours)
    assert none is None and torch.equal(q_only, q_out) and q_only.data_ptr() == wide[:, 1:].data_ptr()
    assert wide[:, 0].isnan().all() and wide[:, hq + 1:].isnan().all()
    none, k_only = ave.qk_norm_rope(None, dev["k"], *args[:3], None, args[4], eps=A.EPS, neighbours=neighbours)
    assert none is None and torch.equal(k_only, k_out)
    if dtype == torch.bfloat16:   # in place
        again = ave.qk_norm_rope(dev["q"], dev["k"], *args, dev["q"], dev["k"], eps=A.EPS, neighbours=neighbours)
        assert torch.equal(again[0], q_out) and torch.equal(again[1], k_out) and again[0].data_ptr() == dev["q"].data_ptr()


@pytest.mark.parametrize("neighbours", [False, True])
def test_norm_and_rotation_against_fp64(gpu, neighbours):
    t, h, d, rot = 50, 6, 128, 96
    rng = np.random.default_rng(5)
    x = A.bf16(rng.standard_normal((t, h, d)) * 3)
    w = rng.standard_normal(d).astype(np.float32)
    cos, sin = A.tables(4000, rot)
    pos = rng.integers(0, 4000, t).astype(np.int32)
    got, _ = ave.qk_norm_rope(_dev(x, gpu).bfloat16(), None, _dev(cos, gpu), _dev(sin, gpu), _dev(pos, gpu), _dev(w, gpu), eps=1e-5, neighbours=neighbours)
    y = x.astype(np.float64)
    y = y / np.sqrt((y * y).mean(-1, keepdims=True) + 1e-5) * w
    z = y[..., :rot].reshape(t, h, rot // 2, 2) if neighbours else np.stack([y[..., :rot // 2], y[..., rot // 2:rot]], -1)
    turn = (z[..., 0] + 1j * z[..., 1]) * (cos[pos] + 1j * sin[pos].astype(np.float64))[:, None]
    size = np.abs(z[..., 0]) + np.abs(z[..., 1])
    if neighbours:
        turned, size = np.stack([turn.real, turn.imag], -1).reshape(t, h, rot), np.stack([size, size], -1).reshape(t, h, rot)
    else:
        turned, size = np.concatenate([turn.real, turn.imag], -1), np.concatenate([size, size], -1)
    want = np.concatenate([turned, y[..., rot:]], -1)
    size = np.concatenate([size, np.abs(y[..., rot:])], -1)
    # sum of 128 squares by a tree of 7 additions, division, root, division, two products, rotation: under 32 roundings of 2^-24
    bound = 2.0 ** -8 * np.abs(want) + 32 * 2.0 ** -24 * 1.01 * size
    assert (np.abs(got.float().cpu().numpy() - want) <= bound).all()


@pytest.mark.parametrize("offset", [1, 3, 8])
def test_unaligned_heads_and_odd_strides(gpu, offset):
    t, h, d = 21, 3, 64
    rng = np.random.default_rng(offset)
    x = A.bf16(rng.standard_normal((t, h, d)))
    cos, sin = A.tables(64, d)
    pos = np.arange(t, dtype=np.int32)
    flat = torch.zeros(t * (h * (d + 5) + 7) + 64, dtype=torch.bfloat16, device=gpu)
    view = flat.as_strided((t, h, d), (h * (d + 5) + 7, d + 5, 1), offset)
    view.copy_(_dev(x, gpu))
    want = orc.f32_to_bf16_bits(A.norm_rope_f32(x, None, cos, sin, pos, False))
    got, _ = ave.qk_norm_rope(view, None, _dev(cos, gpu), _dev(sin, gpu), _dev(pos, gpu))
    assert np.array_equal(_bits(got), want)
    # tables that start at no 16-byte boundary
    odd = [torch.cat([torch.zeros(offset), torch.from_numpy(c).reshape(-1)]).to(gpu)[offset:].view(c.shape) for c in (cos, sin)]
    got, _ = ave.qk_norm_rope(view, None, *odd, _dev(pos, gpu))
    assert np.array_equal(_bits(got), want)


def test_positions_outside_the_table_give_nan(gpu):
    dev, _, _, _ = _case(gpu, 4, 2, 2, 64, 32, False, False, torch.bfloat16, seed=1, rows=10)
    pos = torch.tensor([-1, 0, 9, 10], dtype=torch.int32, device=gpu)
    q, k = ave.qk_norm_rope(dev["q"], dev["k"], dev["cos"], dev["sin"], pos)
    for out, x in ((q, dev["q"]), (k, dev["k"])):
        assert out[[0, 3], :, :32].isnan().all() and not out[1:3].isnan().any() and torch.equal(out[:, :, 32:], x[:, :, 32:])
    cache = ave.kv_cache_mxfp4(1, 2, 16, 64, gpu)
    ave.append_kv_mxfp4(dev["k"], dev["v"], cache, torch.arange(4, dtype=torch.int32, device=gpu), dev["cos"], dev["sin"], pos)
    assert cache[1][0, :, [0, 3], 0].eq(0xFF).all() and not cache[1][0, :, 1:3].eq(0xFF).any()


@pytest.mark.parametrize("page", [16, 64, 512])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t,hq,hkv,d,rot,norm,neighbours", SHAPES)
def test_append_and_gather(gpu, t, hq, hkv, d, rot, norm, neighbours, dtype, page):
    dev, q, k, v = _case(gpu, t, hq, hkv, d, rot, norm, neighbours, dtype, seed=t + d + page)
    rng = np.random.default_rng(page)
    pages = -(-t // page) + 2
    slots = rng.permutation(pages * page)[:t].astype(np.int32)
    slots[3::5] = np.resize(np.array([-1, pages * page, 2 ** 31 - 1, -2 ** 31], np.int32), slots[3::5].shape)   # not stored
    cache = ave.kv_cache_mxfp4(pages, hkv, page, d, gpu)
    for c in cache:
        c.fill_(0xA5)
    want = [np.full(tuple(c.shape), 0xA5, np.uint8) for c in cache]
    stored = (slots >= 0) & (slots < pages * page)
    for i, x in enumerate((k, v)):
        codes, scale = orc.quantize_mxfp4(x.reshape(t * hkv, d))
        want[2 * i][slots[stored] // page, :, slots[stored] % page] = codes.reshape(t, hkv, -1)[stored]
        want[2 * i + 1][slots[stored] // page, :, slots[stored] % page] = scale.reshape(t, hkv, -1)[stored]
    args = (dev["cos"], dev["sin"], dev["positions"], dev["k_weight"])
    q_out = ave.append_kv_mxfp4(dev["k"], dev["v"], cache, _dev(slots, gpu), *args, q=dev["q"], q_weight=dev["q_weight"], eps=A.EPS, neighbours=neighbours)
    for got, w, name in zip(cache, want, ("keys", "key scales", "values", "value scales")):
        assert np.array_equal(got.cpu().numpy(), w), name
    assert np.array_equal(_bits(q_out), orc.f32_to_bf16_bits(q))
    # without queries: the same cache
    other = tuple(torch.full_like(c, 0xA5) for c in cache)
    assert ave.append_kv_mxfp4(dev["k"], dev["v"], other, _dev(slots, gpu), *args, eps=A.EPS, neighbours=neighbours) is None
    assert all(torch.equal(a, b) for a, b in zip(cache, other))
    got = ave.gather_kv_mxfp4(cache, _dev(slots, gpu))
    at = np.where(stored, slots, 0)
    for i in range(2):
        codes, scale = (want[2 * i + n][at // page, :, at % page] for n in range(2))
        x = orc.dequantize_mxfp4(codes.reshape(t * hkv, -1), scale.reshape(t * hkv, -1)).reshape(t, hkv, d)
        assert np.array_equal(_bits(got[i]), orc.f32_to_bf16_bits(np.where(stored[:, None, None], x, np.float32(0))))


def test_special_values(gpu):
    """Infinities and NaN make their block's scale 0xFF, zeros a zero block, and come back as NaN and zeros; every code and a range of scale
    bytes come back exactly."""
    d, page = 64, 16
    x = np.ones((4, 1, d), np.float32)
    x[0, 0, 3], x[1, 0, 40], x[2] = np.inf, np.nan, 0
    t = _dev(x, gpu)
    cache = ave.kv_cache_mxfp4(1, 1, page, d, gpu)
    slots = torch.arange(4, dtype=torch.int32, device=gpu)
    ave.append_kv_mxfp4(t, t, cache, slots)
    for codes, scale in (cache[:2], cache[2:]):
        assert scale[0, 0, :4].cpu().tolist() == [[255, 125], [125, 255], [127, 127], [125, 125]]
        assert codes[0, 0, 0, :16].eq(0).all() and codes[0, 0, 2].eq(0).all()
    k, v = ave.gather_kv_mxfp4(cache, slots)
    for y in (k, v):
        assert y[0, 0, :32].isnan().all() and y[1, 0, 32:].isnan().all() and y[0, 0, 32:].eq(1).all() and y[2].eq(0).all()
    rng = np.random.default_rng(0)
    for c in cache[0], cache[2]:
        c.copy_(_dev(rng.integers(0, 256, tuple(c.shape), dtype=np.uint8), gpu))
    scale = np.arange(0, 252, 252 / 32).astype(np.uint8).reshape(1, 1, page, 2)
    for c in cache[1], cache[3]:
        c.copy_(_dev(scale, gpu))
    k, v = ave.gather_kv_mxfp4(cache, torch.arange(page, dtype=torch.int32, device=gpu))
    for y, codes in ((k, cache[0]), (v, cache[2])):
        want = orc.dequantize_mxfp4(codes.cpu().numpy().reshape(page, -1), scale.reshape(page, -1), np.float64)
        assert np.array_equal(y.double().cpu().numpy().reshape(page, d), want)


def test_pages_beyond_32_bit_offsets_and_inside_a_larger_buffer(gpu):
    """Three pages a little over 2 GiB apart, codes and scales."""
    d, page, hkv, t = 128, 64, 2, 3 * 64
    gap = (1 << 31) + 4096
    buf = torch.zeros(2 * gap + (1 << 20), dtype=torch.uint8, device=gpu)
    size = hkv * page * d // 2
    view = lambda at, last: buf[at:].as_strided((3, hkv, page, last), (gap, page * last, last, 1))   # noqa: E731
    cache = (view(0, d // 2), view(2 * size, d // 32), view(size, d // 2), view(3 * size, d // 32))
    rng = np.random.default_rng(2)
    k, v = (A.bf16(rng.standard_normal((t, hkv, d))) for _ in range(2))
    slots = rng.permutation(t).astype(np.int32)
    ave.append_kv_mxfp4(_dev(k, gpu).bfloat16(), _dev(v, gpu).bfloat16(), cache, _dev(slots, gpu))
    got = ave.gather_kv_mxfp4(cache, _dev(slots, gpu))
    for x, y in zip((k, v), got):
        codes, scale = orc.quantize_mxfp4(x.reshape(-1, d))
        assert np.array_equal(_bits(y), orc.f32_to_bf16_bits(orc.dequantize_mxfp4(codes, scale)).reshape(t, hkv, d))


def test_no_tokens(gpu):
    cache = ave.kv_cache_mxfp4(1, 2, 16, 64, gpu)
    none = torch.empty(0, 2, 64, dtype=torch.bfloat16, device=gpu)
    slots = torch.empty(0, dtype=torch.int32, device=gpu)
    assert ave.append_kv_mxfp4(none, none, cache, slots, q=none).shape == (0, 2, 64)
    assert ave.gather_kv_mxfp4(cache, slots)[0].shape == (0, 2, 64)
    assert ave.qk_norm_rope(none, none)[1].shape == (0, 2, 64)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hq,hkv,d,rot", [(70, 9, 128, 96), (131, 3, 64, 64), (20, 3, 256, 256), (33, 8, 256, 32)])
def test_many_heads_of_many_tokens(gpu, hq, hkv, d, rot, dtype):
    """Several groups of heads in a workgroup, the last one not full; a token count that no eight divides; then from an odd address."""
    t = 1029
    dev, q, k, v = _case(gpu, t, hq, hkv, d, rot, True, False, dtype, seed=d + hq)
    slots = torch.randperm(1040, generator=torch.Generator().manual_seed(1))[:t].int().to(gpu)
    args = (dev["cos"], dev["sin"], dev["positions"], dev["k_weight"])
    caches = []
    for shift in (0, 1):
        wide = torch.zeros(t * (hq + 2 * hkv) * d + 8, dtype=dtype, device=gpu)
        x = wide[shift:shift + t * (hq + 2 * hkv) * d].view(t, hq + 2 * hkv, d)
        x.copy_(torch.cat([dev["q"], dev["k"], dev["v"]], 1))
        cache = ave.kv_cache_mxfp4(65, hkv, 16, d, gpu)
        q_out = ave.append_kv_mxfp4(x[:, hq:hq + hkv], x[:, hq + hkv:], cache, slots, *args, q=x[:, :hq], q_weight=dev["q_weight"], eps=A.EPS)
        assert np.array_equal(_bits(q_out), orc.f32_to_bf16_bits(q))
        caches.append(cache)
    assert all(torch.equal(a, b) for a, b in zip(*caches))
    at = slots.cpu().numpy()
    for i, x in enumerate((k, v)):
        codes, scale = orc.quantize_mxfp4(x.reshape(t * hkv, d))
        assert np.array_equal(caches[0][2 * i].cpu().numpy()[at // 16, :, at % 16], codes.reshape(t, hkv, -1))
        assert np.array_equal(caches[0][2 * i + 1].cpu().numpy()[at // 16, :, at % 16], scale.reshape(t, hkv, -1))
