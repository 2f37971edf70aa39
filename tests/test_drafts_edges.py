"""What the entry points for drafted trees say, on the host, instead of a launch."""
import subprocess
import sys

import pytest
import torch

from avelang_amd import _lib
from tests.test_attention_api import P, _cache, _ref, _refused
from tests.test_drafts_api import _draft, _keep

FAR = 64 * P   # beyond all of the other addresses

CALLS = {
    "draft_tree": "lib.ave_fp4_draft_tree(P, P, P, 4, 1, 2 * P, 1, 3 * P, None)",
    "tree_attention": "lib.ave_fp4_tree_attention_mxfp4(_ref(_attention()), _ref(_tree()), _ref(_cache()), P, 1 << 40, None)",
    "tree_attention, many rows": "lib.ave_fp4_tree_attention_mxfp4(_ref(_attention(max_q=100)), _ref(_tree()), _ref(_cache()), P, 1 << 40, None)",
    "verify_draft": "lib.ave_fp4_verify_draft(_ref(_draft(logits=64 * P)), P, 1 << 40, None)",
    "keep_kv": "lib.ave_fp4_keep_kv_mxfp4((_lib.KVCache * 1)(_cache()), 1, _ref(_keep()), None)",
    "keep_kv, many tokens": "lib.ave_fp4_keep_kv_mxfp4((_lib.KVCache * 1)(_cache()), 1, _ref(_keep(max_q=1000)), None)",
}


@pytest.mark.skipif(torch.cuda.device_count() > 0, reason="the addresses are none: with a device the calls would launch")
@pytest.mark.parametrize("call", CALLS)
def test_no_device(call):
    """Without a device a call returns an error and leaves the process alone (a division by the number of compute units ended it)."""
    program = ("from avelang_amd import _lib\nfrom tests.test_attention_api import P, _cache, _ref\nfrom tests.test_drafts_api import _attention, _draft, _keep, _tree\n"
               f"lib = _lib.load()\nrc = {CALLS[call]}\nassert rc > 0 and 'HIP' in _lib.last_error(), (rc, _lib.last_error())")
    done = subprocess.run([sys.executable, "-c", program], capture_output=True, text=True)
    assert done.returncode == 0, done.stderr


@pytest.mark.parametrize("out", ["accepted", "path", "emitted"])
@pytest.mark.parametrize("where", [
    dict(logits=FAR, logits_stride=100, at=FAR),
    dict(logits=FAR, logits_stride=100, at=FAR + 8 * 200 - 4),                              # the last element of eight rows of 100
    dict(logits=FAR, logits_stride=1000, at=FAR + 7 * 2000 + 196),                          # rows apart
    dict(logits=FAR, logits_stride=1000, at=FAR + 3 * 2000 - 4),                            # ends in one
    dict(logits=FAR, logits_stride=1000, logits_f32=1, at=FAR + 7 * 4000 + 396),
    dict(logits=FAR, logits_stride=-1000, at=FAR - 7 * 2000),                               # rows backwards
    dict(logits=FAR, logits_stride=0, at=FAR + 196),                                        # one row for all
    dict(draft_probs=FAR, draft_probs_stride=100, at=FAR),
    dict(draft_probs=FAR, draft_probs_stride=1 << 40, at=FAR + 5 * (1 << 42) + 396)], ids=str)
def test_outputs_in_rows_of_an_input(where, out):
    where = dict(where)
    d = _draft(**{out: where.pop("at")}, **where)
    _refused(_lib.load().ave_fp4_verify_draft(_ref(d), P, 1 << 40, None), "must not overlap")


@pytest.mark.parametrize("bad", [
    dict(page_table=FAR, kept_lens=FAR), dict(page_table=FAR, kept_lens=FAR + 28), dict(page_table=FAR, page_table_stride=1000, kept_lens=FAR + 4000 + 12),
    dict(page_table=FAR, page_table_stride=1000, kept_lens=FAR + 4000 - 4)], ids=str)
def test_lengths_in_the_page_table(bad):
    lib, cache = _lib.load(), _cache()
    _refused(lib.ave_fp4_keep_kv_mxfp4((_lib.KVCache * 1)(cache), 1, _ref(_keep(**bad)), None), "must not overlap")


@pytest.mark.parametrize("part", ["k", "k_scale", "v", "v_scale"])
def test_lengths_in_a_cache(part):
    lib, cache = _lib.load(), _cache()
    last = getattr(cache, part + "_page_stride") * (cache.pages - 1)
    other = _cache(**{n: FAR * (i + 2) for i, n in enumerate(("k", "k_scale", "v", "v_scale"))})
    for at in (0, last):
        keep = _keep(kept_lens=getattr(other, part) + at)
        _refused(lib.ave_fp4_keep_kv_mxfp4((_lib.KVCache * 2)(cache, other), 2, _ref(keep), None), "must not overlap")
