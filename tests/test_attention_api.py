"""Refusals of the attention entry points, without a GPU: the C ABI's checks, the wrappers' messages, the structures' layout."""
import ctypes

import pytest
import torch

import avelang_amd as ave
from avelang_amd import _lib

P = 1 << 20   # any aligned address: nothing is launched


def _cache(**kw):
    c = dict(k=P, k_scale=P, v=P, v_scale=P, k_page_stride=2 * 16 * 64, k_scale_page_stride=2 * 16 * 4, v_page_stride=2 * 16 * 64,
             v_scale_page_stride=2 * 16 * 4, pages=3, kv_heads=2, page_size=16, head_dim=128)
    return _lib.KVCache(**{**c, **kw})


def _heads(**kw):
    return _lib.Heads(**{**dict(data=P, token_stride=1024, head_stride=128, heads=2, is_f32=0), **kw})


def _ref(x):
    return ctypes.byref(x) if x is not None else None


def _refused(rc, text):
    assert rc == -1 and text in _lib.last_error(), _lib.last_error()


BAD_CACHES = [(dict(head_dim=96), "head_dim must be 64, 128 or 256, got 96"), (dict(kv_heads=0), "kv_heads must be positive"),
              (dict(page_size=24), "power of two"), (dict(page_size=8), "from 16 to 4096"), (dict(page_size=8192), "from 16 to 4096"),
              (dict(pages=0), "slots"), (dict(pages=1 << 28), "slots"), (dict(k=0), "null device pointer"), (dict(v=P + 8), "16-byte aligned"),
              (dict(k_page_stride=2056), "16-byte aligned"), (dict(k_scale=P + 2), "4-byte aligned"), (dict(v_scale_page_stride=130), "4-byte aligned"),
              (dict(v_page_stride=1024), "overlap")]


@pytest.mark.parametrize("bad,text", BAD_CACHES, ids=str)
def test_caches_that_are_refused(bad, text):
    lib = _lib.load()
    c, h = _cache(**bad), _heads()
    _refused(lib.ave_fp4_gather_kv_mxfp4(_ref(c), P, 4, P, P, None), text)
    _refused(lib.ave_fp4_append_kv_mxfp4(_ref(h), _ref(h), 4, P, None, _ref(c), None, None, None), text)
    a = _lib.Attention(q=P, out=P, page_table=P, seq_lens=P, tokens=1, batch=1, heads=4, table_pages=1, max_q=1, causal=1, scale=1)
    _refused(lib.ave_fp4_attention_mxfp4(_ref(a), _ref(c), None, 0, None), text)
    assert lib.ave_fp4_attention_mxfp4_workspace_bytes(_ref(a), _ref(c)) == 0


def test_heads_norms_and_rotations_that_are_refused():
    lib = _lib.load()
    h, c = _heads(), _cache()
    how = lambda **kw: _lib.NormRope(**{**dict(cos=P, sin=P, positions=P, table_rows=10, rotary_dim=64), **kw})   # noqa: E731
    call = lambda q, k, qo, ko, w=None, d=128, t=4: lib.ave_fp4_qk_norm_rope(_ref(q), _ref(k), t, d, _ref(w), _ref(qo), _ref(ko), None)   # noqa: E731
    _refused(call(h, None, h, None, d=80), "head_dim")
    _refused(call(h, None, h, None, t=-1), "tokens must be non-negative")
    _refused(call(None, None, None, None), "queries, keys or both")
    _refused(call(h, h, h, None), "each with its output")
    _refused(call(h, None, _heads(heads=3), None), "q has 2 heads and q_out 3")
    _refused(call(h, None, _heads(is_f32=1), None), "q_out must be bf16")
    _refused(call(h, _heads(is_f32=1), h, h), "one type")
    _refused(call(_heads(data=0), None, h, None), "null device pointer")
    _refused(call(_heads(data=P + 1), None, h, None), "aligned to its elements")
    for bad, text in ((dict(sin=0), "come together"), (dict(rotary_dim=24), "multiple of 16"), (dict(rotary_dim=144), "up to head_dim"),
                      (dict(table_rows=0), "rows"), (dict(positions=0), "positions"), (dict(cos=P + 2), "4-byte"), (dict(q_weight=P + 1), "norm weights")):
        _refused(call(h, None, h, None, how(**bad)), text)
    assert call(h, None, h, None, how(), t=0) == 0
    append = lambda k, v, q=None, qo=None, slots=P: lib.ave_fp4_append_kv_mxfp4(_ref(k), _ref(v), 4, slots, None, _ref(c), _ref(q), _ref(qo), None)   # noqa: E731
    _refused(append(None, h), "keys and values are required")
    _refused(append(h, _heads(heads=3)), "the cache has 2 heads, k 2 and v 3")
    _refused(append(h, _heads(is_f32=1)), "one type")
    _refused(append(h, h, h), "queries come with their output")
    _refused(append(h, h, slots=None), "slots")
    _refused(lib.ave_fp4_gather_kv_mxfp4(_ref(c), P, 4, P + 8, P, None), "16-byte aligned")


@pytest.mark.parametrize("bad,text", [
    (dict(heads=3), "multiple of the cache's 2"), (dict(heads=0), "multiple"), (dict(heads=4096), "at most 1024"), (dict(tokens=-1), "non-negative"),
    (dict(tokens=1 << 30, batch=1 << 30), "31 bits"), (dict(table_pages=1 << 28), "2^31"), (dict(max_q=-1), "max_q"), (dict(window=-1), "window must"),
    (dict(window=5, causal=0), "window needs causal"), (dict(tokens=2), "without cu_q"), (dict(q=0), "null device pointer"),
    (dict(out=P + 2), "4-byte aligned"), (dict(q=P + 1), "2-byte")], ids=str)
def test_attention_calls_that_are_refused(bad, text):
    lib = _lib.load()
    a = _lib.Attention(**{**dict(q=P, out=P, page_table=P, seq_lens=P, tokens=1, batch=1, heads=4, table_pages=1, max_q=1, causal=1, scale=1), **bad})
    _refused(lib.ave_fp4_attention_mxfp4(_ref(a), _ref(_cache()), None, 0, None), text)


def test_wrappers_say_what_is_wrong():
    x = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    cache = ave.kv_cache_mxfp4(1, 2, 16, 64, "cpu")
    assert [tuple(c.shape) for c in cache] == [(1, 2, 16, 32), (1, 2, 16, 2)] * 2
    with pytest.raises(ValueError, match="head_dim must be 64, 128 or 256"):
        ave.kv_cache_mxfp4(1, 1, 16, 80, "cpu")
    with pytest.raises(ValueError, match="power of two"):
        ave.kv_cache_mxfp4(1, 1, 48, 64, "cpu")
    with pytest.raises(ValueError, match="pages and kv_heads"):
        ave.kv_cache_mxfp4(0, 1, 16, 64, "cpu")
    with pytest.raises(ValueError, match="ROCm GPU"):
        ave.append_kv_mxfp4(x, x, cache, i)
    with pytest.raises(TypeError, match="kv_cache_mxfp4"):
        ave.gather_kv_mxfp4(cache[:3], i)
    with pytest.raises(ValueError, match="4-D"):
        ave.gather_kv_mxfp4((x.byte(), *cache[1:]), i)
    with pytest.raises(ValueError, match="ROCm GPU"):
        ave.attention_mxfp4(x, cache, i[:, None], i)
    with pytest.raises(ValueError, match="q, k or both"):
        ave.qk_norm_rope(None, None)
    with pytest.raises(ValueError, match="head_dim must be"):
        ave.qk_norm_rope(x[..., :48], None)
    with pytest.raises(ValueError, match="a ROCm GPU"):
        ave.qk_norm_rope(x, None)


def test_structures_match_the_header():
    """Sizes as a C compiler lays them out: eight-byte members first, then four-byte ones."""
    assert ctypes.sizeof(_lib.KVCache) == 80 and ctypes.sizeof(_lib.Heads) == 32
    assert ctypes.sizeof(_lib.NormRope) == 64 and ctypes.sizeof(_lib.Attention) == 112
