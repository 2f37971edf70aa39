"""Refusals of the entry points for drafted trees, without a GPU: the C ABI's checks, the wrappers' messages, the structures' layout; and the plain
implementations that the GPU tests compare with, by hand."""
import ctypes

import numpy as np
import pytest
import torch

import avelang_amd as ave
from avelang_amd import _lib
from tests import draft_helpers as D
from tests.test_attention_api import BAD_CACHES, P, _cache, _ref, _refused


def _attention(**kw):
    return _lib.Attention(**{**dict(q=P, out=P, page_table=P, seq_lens=P, cu_q=P, tokens=8, batch=2, heads=4, table_pages=1, max_q=4, causal=1, scale=1), **kw})


def _tree(**kw):
    return _lib.Tree(**{**dict(seen=P, stride=1, words=1), **kw})


def _draft(**kw):
    return _lib.Draft(**{**dict(logits=P, logits_stride=100, tokens=P, parents=P, cu_q=P, uniform=P, accepted=2 * P, path=3 * P, emitted=4 * P, rows=8, batch=2, vocab=100),
                         **kw})


def _keep(**kw):
    return _lib.Keep(**{**dict(page_table=P, page_table_stride=4, seq_lens=P, cu_q=P, path=P, accepted=P, kept_lens=2 * P, tokens=8, batch=2, table_pages=4, max_q=4), **kw})


@pytest.mark.parametrize("bad,text", BAD_CACHES, ids=str)
def test_caches_that_are_refused(bad, text):
    lib, c = _lib.load(), _cache(**bad)
    _refused(lib.ave_fp4_tree_attention_mxfp4(_ref(_attention()), _ref(_tree()), _ref(c), None, 0, None), text)
    assert lib.ave_fp4_tree_attention_mxfp4_workspace_bytes(_ref(_attention()), _ref(_tree()), _ref(c)) == 0
    _refused(lib.ave_fp4_keep_kv_mxfp4((_lib.KVCache * 1)(c), 1, _ref(_keep()), None), text)


@pytest.mark.parametrize("bad,text", [
    (dict(heads=3), "multiple of the cache's 2"), (dict(tokens=-1), "non-negative"), (dict(max_q=-1), "max_q"), (dict(window=-1), "window must"),
    (dict(cu_q=0), "without cu_q"), (dict(q=0), "null device pointer"), (dict(out=P + 2), "4-byte"), (dict(q=P + 1), "2-byte")], ids=str)
def test_attention_calls_that_are_refused(bad, text):
    _refused(_lib.load().ave_fp4_tree_attention_mxfp4(_ref(_attention(**bad)), _ref(_tree()), _ref(_cache()), None, 0, None), text)


@pytest.mark.parametrize("bad,text", [(dict(words=0), "between 1 and"), (dict(words=(1 << 25) + 1, stride=1 << 26), "2^25"), (dict(words=2), "overlap"),
                                      (dict(stride=-1), "overlap"), (dict(seen=0), "null device pointer"), (dict(seen=P + 4), "8-byte")], ids=str)
def test_trees_that_are_refused(bad, text):
    lib = _lib.load()
    _refused(lib.ave_fp4_tree_attention_mxfp4(_ref(_attention()), _ref(_tree(**bad)), _ref(_cache()), None, 0, None), text)
    _refused(lib.ave_fp4_tree_attention_mxfp4(_ref(_attention()), None, _ref(_cache()), None, 0, None), "null arguments")


def test_workspaces_and_empty_calls():
    lib, c = _lib.load(), _cache()
    assert lib.ave_fp4_tree_attention_mxfp4(_ref(_attention(tokens=0, batch=0)), _ref(_tree()), _ref(c), None, 0, None) == 0
    for extra in ({}, {"draft_probs": P}):
        d = _draft(**extra)
        need = lib.ave_fp4_verify_draft_workspace_bytes(_ref(d))
        assert need > 0
        _refused(lib.ave_fp4_verify_draft(_ref(d), None, need, None), f"must have {need} bytes")
        _refused(lib.ave_fp4_verify_draft(_ref(d), P, need - 1, None), f"must have {need} bytes")
        _refused(lib.ave_fp4_verify_draft(_ref(d), P + 8, need, None), "16-byte")
    assert lib.ave_fp4_verify_draft(_ref(_draft(rows=0, batch=0)), None, 0, None) == 0
    assert lib.ave_fp4_draft_tree(P, P, P, 0, 0, P, 1, P, None) == 0
    assert lib.ave_fp4_keep_kv_mxfp4((_lib.KVCache * 1)(c), 1, _ref(_keep(batch=0)), None) == 0


@pytest.mark.parametrize("bad,text", [
    (dict(rows=-1), "non-negative"), (dict(batch=-1), "non-negative"), (dict(vocab=0), "vocab must be"), (dict(vocab=(1 << 30) + 1), "vocab must be"),
    (dict(rows=1 << 22), "below 2^22"), (dict(batch=1 << 22), "below 2^22"), (dict(rows=1 << 12, vocab=1 << 23), "below 2^22"), (dict(cu_q=0), "null device pointer"), (dict(logits=0), "null device"),
    (dict(uniform=0), "null device pointer"), (dict(emitted=0), "null device pointer"), (dict(logits=P + 1), "aligned"),
    (dict(logits=P + 2, logits_f32=1), "aligned"), (dict(draft_probs=P + 2), "aligned"), (dict(emitted=P), "overlap"), (dict(path=P + 28), "overlap"),
    (dict(accepted=P + 8), "overlap"), (dict(path=4 * P - 28), "overlap"), (dict(accepted=3 * P + 28), "overlap")], ids=str)
def test_drafts_that_are_refused(bad, text):
    lib = _lib.load()
    _refused(lib.ave_fp4_verify_draft(_ref(_draft(**bad)), P, 1 << 40, None), text)
    _refused(lib.ave_fp4_verify_draft(None, P, 1 << 40, None), "null arguments")


def test_parents_that_are_refused():
    lib = _lib.load()
    _refused(lib.ave_fp4_draft_tree(P, P, P, -1, 1, P, 1, P, None), "non-negative")
    _refused(lib.ave_fp4_draft_tree(P, P, P, 4, 1, P, 0, P, None), "between 1 and 2^25")
    _refused(lib.ave_fp4_draft_tree(None, P, P, 4, 1, P, 1, P, None), "null device pointer")
    _refused(lib.ave_fp4_draft_tree(P, P, None, 4, 1, P, 1, P, None), "null device pointer")
    _refused(lib.ave_fp4_draft_tree(P, P, P, 4, 1, P + 4, 1, P, None), "8-byte")
    _refused(lib.ave_fp4_draft_tree(P, P, P, 4, 1, 2 * P, 1, P, None), "overlap")
    _refused(lib.ave_fp4_draft_tree(P, P, P, 4, 1, P - 24, 1, 3 * P, None), "overlap")
    _refused(lib.ave_fp4_draft_tree(P, P, P, 4, 1, 2 * P, 1, 2 * P + 28, None), "overlap")


@pytest.mark.parametrize("bad,text", [
    (dict(tokens=-1), "non-negative"), (dict(batch=-1), "non-negative"), (dict(max_q=-1), "non-negative"), (dict(table_pages=1 << 28), "2^31 - 1"),
    (dict(seq_lens=0), "null device pointer"), (dict(path=0), "null device pointer"), (dict(page_table=0), "null device pointer"), (dict(kept_lens=P), "overlap"),
    (dict(kept_lens=P + 4, seq_lens=4 * P, accepted=4 * P, path=4 * P), "overlap"), (dict(kept_lens=P - 4, seq_lens=4 * P, accepted=4 * P, cu_q=4 * P), "overlap")], ids=str)
def test_moves_that_are_refused(bad, text):
    lib = _lib.load()
    _refused(lib.ave_fp4_keep_kv_mxfp4((_lib.KVCache * 1)(_cache()), 1, _ref(_keep(**bad)), None), text)


def test_layers_that_are_refused():
    lib = _lib.load()
    keep = lambda n, *caches: lib.ave_fp4_keep_kv_mxfp4((_lib.KVCache * len(caches))(*caches), n, _ref(_keep()), None)   # noqa: E731
    other = _cache(k=2 * P, v=2 * P, k_scale=2 * P, v_scale=2 * P)
    _refused(keep(0, other), "there must be layers")
    _refused(keep(2, _cache(), _cache(k=2 * P, v=2 * P, pages=4)), "layer 1 differs")
    _refused(keep(2, _cache(), _cache()), "layers 0 and 1 have the same cache")
    _refused(keep(3, _cache(), other, _cache(k=3 * P, v=2 * P)), "layers 1 and 2 have the same cache")
    _refused(lib.ave_fp4_keep_kv_mxfp4(None, 1, _ref(_keep()), None), "null arguments")


def test_wrappers_say_what_is_wrong():
    x, i = torch.zeros(2, 2, 64, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    cache = ave.kv_cache_mxfp4(1, 2, 16, 64, "cpu")
    with pytest.raises(ValueError, match="ROCm GPU"):
        ave.tree_attention_mxfp4(x, cache, i[:, None], i, None, torch.zeros(2, 1, dtype=torch.int64))
    with pytest.raises(ValueError, match="seen is required"):
        ave.tree_attention_mxfp4(x, cache, i[:, None], i, None, None)
    with pytest.raises(ValueError, match="parents must be on a ROCm GPU"):
        ave.draft_tree(i, i, i, max_q=1)
    with pytest.raises(ValueError, match="parents must be a 1-D"):
        ave.draft_tree(i[None], i, i, max_q=1)
    with pytest.raises(ValueError, match="2-D tensor"):
        ave.verify_draft(x, i, i, i, x)
    with pytest.raises(ValueError, match="cu_q must be a 1-D"):
        ave.verify_draft(x[:, 0], i, i, None, x)
    with pytest.raises(ValueError, match="a ROCm GPU"):
        ave.verify_draft(x[:, 0], i, i, i, x)
    with pytest.raises(TypeError, match="a cache or a list of caches"):
        ave.keep_kv_mxfp4([], i[:, None], i, i, i, i)
    with pytest.raises(ValueError, match="ROCm GPU"):
        ave.keep_kv_mxfp4([cache], i[:, None], i, i, i, i)


def test_structures_match_the_header():
    assert ctypes.sizeof(_lib.Tree) == 24 and ctypes.sizeof(_lib.Draft) == 112 and ctypes.sizeof(_lib.Keep) == 72


def test_the_plain_walk_by_hand():
    """A root with two children and a grandchild; p = softmax of logs, so that the numbers can be followed."""
    p = np.array([[0.5, 0.25, 0.125, 0.125], [0.1, 0.2, 0.3, 0.4], [0.7, 0.1, 0.1, 0.1], [0.25, 0.25, 0.25, 0.25]])
    tokens, parents = np.array([9, 0, 1, 3]), np.array([-1, 0, 0, 2])
    walk = lambda u, t=1.0: D.verify_one(np.log(p).astype(np.float32), tokens, parents, np.array(u, np.float32), t)   # noqa: E731
    assert walk([0.95, 0.4, 0.9, 0.9]) == ([0, 1], [0, 3])                 # the first child, then a draw from its row
    assert walk([0.0, 0.6, 0.49, 0.05]) == ([0, 2, 3], [1, 3, 0])          # the second one: 0.25 of what 0.5 leaves
    assert walk([0.49, 0.6, 0.51, 0.9]) == ([0], [2])                      # neither: 2 and 3 are left, half each
    assert walk([0.6, 0.6, 0.51, 0.9]) == ([0], [3])
    assert walk([0.0] * 4, 0.0) == ([0, 1], [0, 3])
    q = np.tile(np.array([0.25, 0.25, 0.25, 0.25]), (4, 1))
    with_q = lambda u: D.verify_one(np.log(p).astype(np.float32), tokens, parents, np.array(u, np.float32), 1.0, q)   # noqa: E731
    assert with_q([0.5, 0.99, 0.9, 0.9])[0] == [0, 1]                      # p >= q: always
    tokens[1] = 2
    assert with_q([0.5, 0.51, 0.9, 0.9]) == ([0], [0])                     # p / q = 1/2; what is left is all on token 0
    above = D.ancestors(np.array([-1, 0, 0, 1, 7, 4]))
    assert above.tolist() == [[1, 0, 0, 0, 0, 0], [1, 1, 0, 0, 0, 0], [1, 0, 1, 0, 0, 0], [1, 1, 0, 1, 0, 0], [0, 0, 0, 0, 1, 0], [0, 0, 0, 0, 1, 1]]
    assert D.words_of(above, 1)[:, 0].tolist() == [1, 3, 5, 11, 16, 48]
