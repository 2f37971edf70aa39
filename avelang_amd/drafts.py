"""Host entry points for checking a tree of drafted tokens: what its nodes see of each other, and which of them the target model keeps.
Same conventions as :mod:`avelang_amd.attention`; attention over a tree (:func:`tree_attention_mxfp4`) and the move of the kept tokens in the caches
(:func:`keep_kv_mxfp4`) are there.  The reference has no counterpart; these are additions.

A sequence's nodes are rows ``cu_q[b]:cu_q[b+1]`` of all nodes and its last tokens in the cache, parents before children; node 0 is the last token that
was already decided on.  A step of a draft, with no word to the host::

    seen, positions = draft_tree(parents, cu_q, seq_lens, max_q=n)
    ... append_kv_mxfp4(..., positions=positions), tree_attention_mxfp4(..., seen), a layer after the other ...
    accepted, path, emitted = verify_draft(logits, tokens, parents, cu_q, uniform)
    kept_lens = keep_kv_mxfp4(caches, page_table, seq_lens, cu_q, path, accepted)
"""
from __future__ import annotations

import torch

from . import _lib
from ._lib import native as _native
from .amdgpu_gemm_fp4 import _stream_ptr
from .attention import _sizes, _vector


def _rows(t, name, dtypes, rows, columns, device):
    """``[rows, columns]`` with consecutive elements in a row, any stride between rows."""
    if not isinstance(t, torch.Tensor) or t.dtype not in dtypes or t.dim() != 2:
        raise ValueError(f"{name} must be a 2-D tensor of {' or '.join(map(str, dtypes))}.")
    _sizes(t, name)
    if (rows is not None and t.shape[0] != rows) or (columns is not None and t.shape[1] != columns):
        raise ValueError(f"{name} must have shape {(rows, columns)}, got {tuple(t.shape)}.")
    if t.device != device or device.type != "cuda":
        raise ValueError(f"{name} must be on device {device} (a ROCm GPU), got {t.device}.")
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"{name} must have consecutive elements in a row.")
    return t.data_ptr(), t.stride(0)


def _bounds(cu_q, name="cu_q"):
    if not isinstance(cu_q, torch.Tensor) or cu_q.dim() != 1 or cu_q.shape[0] < 1:
        raise ValueError(f"{name} must be a 1-D torch.int32 tensor with an entry more than there are sequences.")
    return _sizes(cu_q, name).shape[0] - 1


def draft_tree(parents, cu_q, seq_lens, seen=None, positions=None, *, max_q):
    """Ancestors and positions of the nodes of ``B`` drafts.  Returns ``(seen, positions)``.

    ``parents`` int32 ``[T]``: the index within its sequence of the node that a node follows; one that is not below the node's own, or negative, means
    none.  ``cu_q`` int32 ``[B+1]``; ``seq_lens`` int32 ``[B]``: tokens in the cache, the nodes among them.  ``seen`` int64 ``[T, ceil(max_q / 64)]``: bit
    ``j % 64`` of word ``j // 64`` is set where node ``j`` of the sequence is the node itself or above it (``max_q``: a bound on the nodes of a sequence;
    later nodes have no bit).  ``positions`` int32 ``[T]``: ``seq_lens - n`` and the number of nodes above."""
    done = _native.draft_tree(parents, cu_q, seq_lens, seen, positions, max_q)
    if done is not None:
        return done
    if not isinstance(parents, torch.Tensor) or parents.dim() != 1:
        raise ValueError("parents must be a 1-D torch.int32 tensor.")
    dev, t = parents.device, parents.shape[0]
    if dev.type != "cuda":
        raise ValueError(f"parents must be on a ROCm GPU device, got {dev}.")
    if int(max_q) < 1:
        raise ValueError(f"max_q must be positive, got {max_q}.")
    words = -(-int(max_q) // 64)
    b = _bounds(cu_q)
    args = [_vector(parents, "parents", torch.int32, t, dev), _vector(cu_q, "cu_q", torch.int32, b + 1, dev),
            _vector(seq_lens, "seq_lens", torch.int32, b, dev)]
    if words > 1 << 25:
        raise ValueError(f"seen must have at most 2^25 words a row, got {words}.")
    if seen is None:
        seen = torch.empty((t, words), dtype=torch.int64, device=dev)
    _rows(seen, "seen", (torch.int64,), t, words, dev)
    if not seen.is_contiguous():
        raise ValueError("seen must be contiguous.")
    if positions is None:
        positions = torch.empty(t, dtype=torch.int32, device=dev)
    _vector(positions, "positions", torch.int32, t, dev)
    lib = _lib.load()
    with torch.cuda.device(dev):
        rc = lib.ave_fp4_draft_tree(*args, t, b, seen.data_ptr(), words, positions.data_ptr(), _stream_ptr(dev))
    _lib.check(rc)
    return seen, positions


def verify_draft(logits, tokens, parents, cu_q, uniform, temperature=None, draft_probs=None, accepted=None, path=None, emitted=None):
    """Which nodes of ``B`` drafts are kept, and the token behind them, distributed as the target model's own (or, at temperature 0, the ones that it
    would choose).  Returns int32 ``(accepted [B], path [T], emitted [T])``.

    ``logits`` ``[T, vocab]`` bf16 or fp32, consecutive in a row: the target's behind each node.  ``tokens``, ``parents`` int32 ``[T]``, ``cu_q`` int32
    ``[B+1]``.  ``uniform`` fp32 ``[T]``: independent random numbers in [0, 1), that of a node for its acceptance, of node 0 for the token at
    the end.  ``temperature`` fp32 ``[B]`` (``None``: 1).  ``draft_probs`` fp32 ``[T, vocab]``: row ``t`` the distribution that the children of node ``t``
    were drawn from, independently; ``None``: children were chosen, not drawn.

    From node 0 on, a node's children are tried in order.  Without ``draft_probs`` child ``c`` is accepted if ``uniform[c] < r[token]``, where ``r`` is the
    softmax without the tokens of rejected siblings, over its sum; with them if ``uniform[c] * q[token] < r[token]``, where a rejection turns
    ``r`` into ``max(r - q, 0)`` over its sum.  At temperature 0 the child with the largest logit's token is.  Where no child is, the next token is the
    first index where the running sum of ``r`` is above ``uniform[node 0]`` of the whole (temperature 0: the largest logit's, the lowest of equal ones).
    ``accepted`` counts the kept nodes, node 0 among them; ``path[cu_q[b]:][:accepted[b]]`` are their indices in the sequence, and ``emitted`` as many
    tokens: the kept nodes' from the second on, then the new one; the rest of a sequence's rows is -1, and rows of no sequence are left alone.
    What is chosen is what softmax and sums in fp64 choose (fp32 sums decide an acceptance only where they are exact enough to say).  A NaN logit counts as -inf; a
    logit 708 temperatures and more below the row's largest hides its token, too."""
    done = _native.verify_draft(logits, tokens, parents, cu_q, uniform, temperature, draft_probs, accepted, path, emitted)
    if done is not None:
        return done
    if not isinstance(logits, torch.Tensor) or logits.dim() != 2:
        raise ValueError("logits must be a 2-D tensor [nodes, vocab].")
    dev, t = logits.device, logits.shape[0]
    b = _bounds(cu_q)
    d = _lib.Draft(rows=t, batch=b, vocab=_sizes(logits, "logits").shape[1], logits_f32=int(logits.dtype == torch.float32))
    d.logits, d.logits_stride = _rows(logits, "logits", (torch.bfloat16, torch.float32), t, None, dev)
    d.tokens, d.parents = (_vector(x, n, torch.int32, t, dev) for x, n in ((tokens, "tokens"), (parents, "parents")))
    d.cu_q = _vector(cu_q, "cu_q", torch.int32, b + 1, dev)
    d.uniform = _vector(uniform, "uniform", torch.float32, t, dev)
    if temperature is not None:
        d.temperature = _vector(temperature, "temperature", torch.float32, b, dev)
    if draft_probs is not None:
        d.draft_probs, d.draft_probs_stride = _rows(draft_probs, "draft_probs", (torch.float32,), t, logits.shape[1], dev)
    outs = []
    for out, name, n in ((accepted, "accepted", b), (path, "path", t), (emitted, "emitted", t)):
        if out is None:
            out = torch.empty(n, dtype=torch.int32, device=dev)
        setattr(d, name, _vector(out, name, torch.int32, n, dev))
        outs.append(out)
    lib = _lib.load()
    with torch.cuda.device(dev):
        bytes_ = lib.ave_fp4_verify_draft_workspace_bytes(d)
        workspace = torch.empty(bytes_, dtype=torch.uint8, device=dev) if bytes_ else None
        rc = lib.ave_fp4_verify_draft(d, workspace.data_ptr() if bytes_ else None, bytes_, _stream_ptr(dev))
    _lib.check(rc)
    return tuple(outs)
