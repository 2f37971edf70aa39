"""What the entry points for drafted trees say, on the host, instead of a launch."""
import subprocess
import sys

import pytest
import torch

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
