"""Host entry points of what stands between the qkv projection and the output projection of a decoder layer: norms and
rotation of query and key heads, a paged key/value cache held in MXFP4, and attention over it.  Same conventions as
:mod:`avelang_amd.amdgpu_gemm_fp4` (reference ``python/avelang_kernels/amdgpu_gemm.py:458-494``): ``ValueError`` before anything
is launched, asynchronous launch on torch's current stream, optional preallocated outputs, no synchronisation -- lengths, slots,
positions and page tables are device tensors that the host never reads, so a decode step can be captured once and replayed.
The reference has no attention code; these are additions.

A ``cache`` is the tuple ``(k, k_scale, v, v_scale)`` that :func:`kv_cache_mxfp4` makes: packed E2M1 codes ``[pages, kv_heads,
page_size, head_dim/2]`` and E8M0 scales ``[pages, kv_heads, page_size, head_dim/32]``.  A token's place is its *slot*,
``page * page_size + offset``."""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from ._lib import native as _native
from .amdgpu_gemm_fp4 import _as_bytes, _stream_ptr

HEAD_DIMS = (64, 128, 256)


def kv_cache_mxfp4(pages, kv_heads, page_size, head_dim, device="cuda"):
    """An empty cache of one layer: ``(k, k_scale, v, v_scale)``, uint8, zero-filled (34 bytes for 32 channels of a token's key
    and value).  ``head_dim`` 64, 128 or 256, ``page_size`` a power of two from 16 to 4096."""
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"head_dim must be 64, 128 or 256, got {head_dim}.")
    if page_size < 16 or page_size > 4096 or page_size & (page_size - 1):
        raise ValueError(f"page_size must be a power of two from 16 to 4096, got {page_size}.")
    if pages <= 0 or kv_heads <= 0:
        raise ValueError(f"pages and kv_heads must be positive, got {pages} and {kv_heads}.")
    make = lambda last: torch.zeros((pages, kv_heads, page_size, last), dtype=torch.uint8, device=device)   # noqa: E731
    return make(head_dim // 2), make(head_dim // 32), make(head_dim // 2), make(head_dim // 32)


def _sizes(t, name):
    """``t``, whose sizes the C ABI takes as 32-bit numbers."""
    if any(n > 2 ** 31 - 1 for n in t.shape):
        raise ValueError(f"{name} must have sizes below 2^31, got {tuple(t.shape)}.")
    return t


def _cache(cache):
    """The C ABI's view of a cache; also its device.  (The library itself checks sizes and alignment.)"""
    if not isinstance(cache, (tuple, list)) or len(cache) != 4:
        raise TypeError("cache must be the tuple (k, k_scale, v, v_scale) of kv_cache_mxfp4.")
    names = ("k_cache", "k_scale", "v_cache", "v_scale")
    parts = [_sizes(_as_bytes(t, n), n) for t, n in zip(cache, names)]
    k = parts[0]
    if k.dim() != 4:
        raise ValueError(f"k_cache must be 4-D [pages, kv_heads, page_size, head_dim/2], got {k.dim()}-D.")
    if k.device.type != "cuda":
        raise ValueError(f"the cache must be on a ROCm GPU device, got {k.device}.")
    pages, heads, page, half = k.shape
    if 2 * half not in HEAD_DIMS:
        raise ValueError(f"head_dim must be 64, 128 or 256, got {2 * half}.")
    for t, n, last in zip(parts, names, (half, half // 16, half, half // 16)):
        if tuple(t.shape) != (pages, heads, page, last):
            raise ValueError(f"{n} must have shape {(pages, heads, page, last)}, got {tuple(t.shape)}.")
        if t.device != k.device:
            raise ValueError(f"{n} must be on device {k.device}, got {t.device}.")
        if pages and not t[0].is_contiguous():
            raise ValueError(f"{n} must be contiguous inside a page.")
    c = _lib.KVCache(*(t.data_ptr() for t in parts), *(t.stride(0) for t in parts), pages, heads, page, 2 * half)
    return c, k.device


def _heads(t, name, heads, head_dim, tokens, device, dtypes=(torch.bfloat16, torch.float32)):
    """``[tokens, heads, head_dim]`` with consecutive channels, any strides otherwise."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}.")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must have dtype {' or '.join(map(str, dtypes))}, got {t.dtype}.")
    if t.dim() != 3:
        raise ValueError(f"{name} must be 3-D [tokens, heads, head_dim], got {t.dim()}-D.")
    _sizes(t, name)
    want = (t.shape[0] if tokens is None else tokens, t.shape[1] if heads is None else heads, head_dim)
    if tuple(t.shape) != want:
        raise ValueError(f"{name} must have shape {want}, got {tuple(t.shape)}.")
    if t.device != device or t.device.type != "cuda":
        raise ValueError(f"{name} must be on device {device} (a ROCm GPU), got {t.device}.")
    if head_dim > 1 and t.stride(2) != 1:
        raise ValueError(f"{name} must have consecutive channels.")
    return _lib.Heads(t.data_ptr(), t.stride(0), t.stride(1), t.shape[1], int(t.dtype == torch.float32))


def _vector(t, name, dtype, length, device):
    if not isinstance(t, torch.Tensor) or t.dtype != dtype:
        raise ValueError(f"{name} must be a {dtype} tensor.")
    if tuple(_sizes(t, name).shape) != (length,):
        raise ValueError(f"{name} must have shape {(length,)}, got {tuple(t.shape)}.")
    if t.device != device:
        raise ValueError(f"{name} must be on device {device}, got {t.device}.")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous.")
    return t.data_ptr()


def _how(cos, sin, positions, q_weight, k_weight, eps, neighbours, tokens, head_dim, device):
    how = _lib.NormRope(eps=eps, neighbours=int(bool(neighbours)))
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together.")
    if cos is not None:
        for t, name in ((cos, "cos"), (sin, "sin")):
            if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.dim() != 2:
                raise ValueError(f"{name} must be a 2-D torch.float32 tensor [positions, rotary_dim/2].")
            _sizes(t, name)
            if t.shape != cos.shape or t.device != device or not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous, on device {device} and of cos's shape {tuple(cos.shape)}.")
        if positions is None:
            raise ValueError("rotation needs positions.")
        how.cos, how.sin, how.table_rows, how.rotary_dim = cos.data_ptr(), sin.data_ptr(), cos.shape[0], 2 * cos.shape[1]
        how.positions = _vector(positions, "positions", torch.int32, tokens, device)
    given = [(w, n) for w, n in ((q_weight, "q_weight"), (k_weight, "k_weight")) if w is not None]
    for w, name in given:
        if not isinstance(w, torch.Tensor) or w.dtype not in (torch.bfloat16, torch.float32) or w.dtype != given[0][0].dtype:
            raise ValueError(f"{name} must be a torch.bfloat16 or torch.float32 tensor (both weights of one type).")
        setattr(how, name, _vector(w, name, w.dtype, head_dim, device))
        how.weight_is_f32 = int(w.dtype == torch.float32)
    return how


def _bf16_out(t, name, like, head_dim, device):
    if t is None:
        t = torch.empty(like.shape, dtype=torch.bfloat16, device=device)
    return t, _heads(t, name, like.shape[1], head_dim, like.shape[0], device, (torch.bfloat16,))


def _ref(x):
    return ctypes.byref(x) if x is not None else None


def _int32(x):
    """``x``, or the nearest number of 32 bits: no length comes near, and ctypes would drop the bits above."""
    return max(-2 ** 31, min(int(x), 2 ** 31 - 1))


def qk_norm_rope(q, k, cos=None, sin=None, positions=None, q_weight=None, k_weight=None, q_out=None, k_out=None, *, eps=1e-6,
                 neighbours=False):
    """Norm and rotation of query and key heads in one launch.

    ``q`` ``[T, heads, head_dim]`` and ``k`` ``[T, kv_heads, head_dim]`` bf16 or fp32 (one type) with consecutive channels and any
    other strides, so that they may be slices of a packed projection; either may be ``None``.  With a weight ``[head_dim]`` (bf16 or
    fp32) a head is normed: ``x / sqrt(mean(x^2) + eps) * weight``.  With ``cos``, ``sin`` (fp32 ``[positions, rotary_dim/2]``) its first
    ``rotary_dim`` channels (a multiple of 16) are rotated by row ``positions[t]`` (int32 ``[T]``) as pairs ``(i, i + rotary_dim/2)``, with
    ``neighbours`` as pairs ``(2i, 2i+1)``; a position outside the table gives NaN.  All in fp32 with one rounding at the end.
    Returns bf16 ``(q_out, k_out)``; an output may be its input."""
    done = _native.qk_norm_rope(q, k, cos, sin, positions, q_weight, k_weight, q_out, k_out, eps, neighbours)
    if done is not None:
        return done
    x = q if q is not None else k
    if x is None:
        raise ValueError("q, k or both are required.")
    if not isinstance(x, torch.Tensor) or x.dim() != 3:
        raise ValueError("q and k must be 3-D tensors [tokens, heads, head_dim].")
    t, _, d = x.shape
    if d not in HEAD_DIMS:
        raise ValueError(f"head_dim must be 64, 128 or 256, got {d}.")
    dev = x.device
    qh = _heads(q, "q", None, d, t, dev) if q is not None else None
    kh = _heads(k, "k", None, d, t, dev) if k is not None else None
    if qh and kh and q.dtype != k.dtype:
        raise ValueError(f"q and k must have one dtype, got {q.dtype} and {k.dtype}.")
    how = _how(cos, sin, positions, q_weight, k_weight, eps, neighbours, t, d, dev)
    q_out, qo = _bf16_out(q_out, "q_out", q, d, dev) if qh else (None, None)
    k_out, ko = _bf16_out(k_out, "k_out", k, d, dev) if kh else (None, None)
    lib = _lib.load()
    with torch.cuda.device(dev):
        rc = lib.ave_fp4_qk_norm_rope(_ref(qh), _ref(kh), t, d, _ref(how), _ref(qo), _ref(ko), _stream_ptr(dev))
    _lib.check(rc)
    return q_out, k_out


def append_kv_mxfp4(k, v, cache, slots, cos=None, sin=None, positions=None, k_weight=None, *, q=None, q_weight=None, q_out=None,
                    eps=1e-6, neighbours=False):
    """Append keys and values of ``T`` tokens to a cache, with the keys' norm and rotation on the way.

    ``k``, ``v`` ``[T, kv_heads, head_dim]`` bf16 or fp32; ``slots`` int32 ``[T]``: a slot outside the cache (-1) stores nothing;
    those inside it must differ (what two tokens of a call share is undefined: a mix of both).
    ``cos``, ``sin``, ``positions``, ``k_weight``, ``eps``, ``neighbours`` as in :func:`qk_norm_rope` (all ``None``: the keys as they are).
    Codes and scales are those that :func:`quantize_mxfp4` gives for the fp32 values of the normed and rotated keys, and for the values.
    With ``q`` ``[T, heads, head_dim]`` the same launch norms (``q_weight``) and rotates the queries and returns them as bf16;
    otherwise returns ``None``."""
    done = _native.append_kv_mxfp4(k, v, cache, slots, cos, sin, positions, k_weight, q, q_weight, q_out, eps, neighbours)
    if done is not None:
        return done[0]
    c, dev = _cache(cache)
    d = c.head_dim
    kh = _heads(k, "k", c.kv_heads, d, None, dev)
    t = k.shape[0]
    vh = _heads(v, "v", c.kv_heads, d, t, dev, (k.dtype,))
    slots_ptr = _vector(slots, "slots", torch.int32, t, dev)
    qh = _heads(q, "q", None, d, t, dev, (k.dtype,)) if q is not None else None
    how = _how(cos, sin, positions, q_weight, k_weight, eps, neighbours, t, d, dev)
    q_out, qo = _bf16_out(q_out, "q_out", q, d, dev) if qh else (None, None)
    lib = _lib.load()
    with torch.cuda.device(dev):
        rc = lib.ave_fp4_append_kv_mxfp4(_ref(kh), _ref(vh), t, slots_ptr, _ref(how), _ref(c), _ref(qh), _ref(qo), _stream_ptr(dev))
    _lib.check(rc)
    return q_out


def gather_kv_mxfp4(cache, slots, k_out=None, v_out=None):
    """Cached tokens back as bf16 ``(k, v)``, each ``[T, kv_heads, head_dim]`` (exact): to move or fork a sequence, to offload it, to look
    at it.  ``slots`` int32 ``[T]``; a slot outside the cache gives zeros, a scale byte 0xFF NaN."""
    done = _native.gather_kv_mxfp4(cache, slots, k_out, v_out)
    if done is not None:
        return done
    c, dev = _cache(cache)
    if not isinstance(slots, torch.Tensor) or slots.dim() != 1:
        raise ValueError("slots must be a 1-D torch.int32 tensor.")
    t = slots.shape[0]
    slots_ptr = _vector(slots, "slots", torch.int32, t, dev)
    outs = []
    for out, name in ((k_out, "k_out"), (v_out, "v_out")):
        if out is None:
            out = torch.empty((t, c.kv_heads, c.head_dim), dtype=torch.bfloat16, device=dev)
        _heads(out, name, c.kv_heads, c.head_dim, t, dev, (torch.bfloat16,))
        if not out.is_contiguous():
            raise ValueError(f"{name} must be contiguous.")
        outs.append(out)
    lib = _lib.load()
    with torch.cuda.device(dev):
        rc = lib.ave_fp4_gather_kv_mxfp4(_ref(c), slots_ptr, t, outs[0].data_ptr(), outs[1].data_ptr(), _stream_ptr(dev))
    _lib.check(rc)
    return tuple(outs)


def attention_mxfp4(q, cache, page_table, seq_lens, cu_q=None, out=None, lse=None, *, max_q=None, scale=None, window=0, sinks=None,
                    causal=True):
    """Attention of the new tokens of ``B`` sequences over their cached keys and values.  Returns bf16 ``[T, heads, head_dim]``.

    ``q`` bf16 ``[T, heads, head_dim]`` (normed and rotated), consecutive channels, any other strides; ``heads`` a multiple of the cache's,
    consecutive query heads share a key head.  ``page_table`` int32 ``[B, pages]`` (rows may be strided), ``seq_lens`` int32 ``[B]``: tokens
    in the cache, the new ones among them.  ``cu_q`` int32 ``[B+1]``: sequence ``b`` has rows ``cu_q[b]:cu_q[b+1]`` of ``q``, its last tokens
    (``None``: one row each).  ``max_q``: a bound on the new tokens of a sequence, if the host knows one; it helps to choose the kernel.
    ``scale`` defaults to ``head_dim ** -0.5``.  ``causal``: a token sees itself and what is before it, with ``window`` only the last
    ``window`` of these.  ``sinks`` fp32 ``[heads]``: a logit beside the keys' in the softmax's denominator.  ``lse`` (fp32 ``[T, heads]``,
    optional) is filled with the log of the denominator.  A row that sees no key gives zeros (lse -inf, or its sink).
    Scores, softmax and sums are fp32, queries count to 2^-19 of their row's largest; probabilities enter the product with the values as bf16, each off by up to 2^-8 of
    itself, as the result is (measured against fp64: 0.0023 of the output's norm, where the result's rounding alone gives 0.0017).
    Partial results of sequences that several workgroups share go through a workspace from torch's allocator (stream-ordered)."""
    if max_q is None:
        max_q = 1 if cu_q is None else q.shape[0] if isinstance(q, torch.Tensor) and q.dim() == 3 else 0
    done = _native.attention_mxfp4(q, cache, page_table, seq_lens, cu_q, out, lse, max_q, scale, window, sinks, causal)
    if done is not None:
        return done
    return _attention(q, cache, page_table, seq_lens, cu_q, out, lse, max_q, scale, window, sinks, causal)


def tree_attention_mxfp4(q, cache, page_table, seq_lens, cu_q, seen, out=None, lse=None, *, max_q=None, scale=None, window=0, sinks=None):
    """:func:`attention_mxfp4` of drafted tokens that are not a chain: with ``n`` new tokens (nodes) in a sequence, each sees the tokens before all
    of them and, of the nodes, those whose bit is set in its row of ``seen`` (int64 ``[T, words]``, as :func:`draft_tree` makes it; rows may be strided;
    bit ``j % 64`` of word ``j // 64``: node ``j`` of the sequence).  ``window``: the last ``window`` of what a node sees (nodes are seen as the bits
    say, and ``window`` less their number of the tokens before them).  The rest, and what is returned, as there."""
    if max_q is None:
        max_q = 1 if cu_q is None else q.shape[0] if isinstance(q, torch.Tensor) and q.dim() == 3 else 0
    done = _native.tree_attention_mxfp4(q, cache, page_table, seq_lens, cu_q, seen, out, lse, max_q, scale, window, sinks)
    if done is not None:
        return done
    if seen is None:
        raise ValueError("seen is required.")
    return _attention(q, cache, page_table, seq_lens, cu_q, out, lse, max_q, scale, window, sinks, True, seen)


def _tree(seen, tokens, device):
    if not isinstance(seen, torch.Tensor) or seen.dtype != torch.int64 or seen.dim() != 2:
        raise ValueError("seen must be a 2-D torch.int64 tensor [nodes, words].")
    if _sizes(seen, "seen").shape[0] != tokens or seen.shape[1] < 1:
        raise ValueError(f"seen must have {tokens} rows of at least one word, got {tuple(seen.shape)}.")
    if seen.device != device:
        raise ValueError(f"seen must be on device {device}, got {seen.device}.")
    if seen.shape[1] > 1 and seen.stride(1) != 1:
        raise ValueError("seen must have consecutive words in a row.")
    return _lib.Tree(seen.data_ptr(), seen.stride(0) if tokens > 1 else seen.shape[1], seen.shape[1])


def _attention(q, cache, page_table, seq_lens, cu_q, out, lse, max_q, scale, window, sinks, causal, seen=None):
    c, dev = _cache(cache)
    d = c.head_dim
    _heads(q, "q", None, d, None, dev, (torch.bfloat16,))
    t, heads, _ = q.shape
    if not isinstance(page_table, torch.Tensor) or page_table.dtype != torch.int32 or page_table.dim() != 2:
        raise ValueError("page_table must be a 2-D torch.int32 tensor [sequences, pages].")
    b, width = _sizes(page_table, "page_table").shape
    if page_table.device != dev:
        raise ValueError(f"page_table must be on device {dev}, got {page_table.device}.")
    if width > 1 and page_table.stride(1) != 1:
        raise ValueError("page_table must have consecutive entries in a row.")
    a = _lib.Attention(q=q.data_ptr(), q_token_stride=q.stride(0), q_head_stride=q.stride(1), page_table=page_table.data_ptr(),
                       page_table_stride=page_table.stride(0), tokens=t, batch=b, heads=heads, table_pages=width, max_q=_int32(max_q),
                       window=_int32(window or 0), causal=int(bool(causal)), scale=d ** -0.5 if scale is None else scale)
    if not math.isfinite(a.scale):
        raise ValueError(f"scale must be finite, got {scale}.")
    a.seq_lens = _vector(seq_lens, "seq_lens", torch.int32, b, dev)
    if cu_q is not None:
        a.cu_q = _vector(cu_q, "cu_q", torch.int32, b + 1, dev)
    if sinks is not None:
        a.sinks = _vector(sinks, "sinks", torch.float32, heads, dev)
    if out is None:
        out = torch.empty((t, heads, d), dtype=torch.bfloat16, device=dev)
    _heads(out, "out", heads, d, t, dev, (torch.bfloat16,))
    if not out.is_contiguous():
        raise ValueError("out must be contiguous.")
    a.out = out.data_ptr()
    if lse is not None:
        if not isinstance(lse, torch.Tensor) or lse.dtype != torch.float32 or tuple(lse.shape) != (t, heads) or lse.device != dev or not lse.is_contiguous():
            raise ValueError(f"lse must be a contiguous torch.float32 tensor of shape {(t, heads)} on device {dev}.")
        a.lse = lse.data_ptr()
    lib = _lib.load()
    given = (_ref(a), _ref(c)) if seen is None else (_ref(a), _ref(_tree(seen, t, dev)), _ref(c))
    name = "ave_fp4_attention_mxfp4" if seen is None else "ave_fp4_tree_attention_mxfp4"
    with torch.cuda.device(dev):
        bytes_ = getattr(lib, name + "_workspace_bytes")(*given)
        workspace = torch.empty(bytes_, dtype=torch.uint8, device=dev) if bytes_ else None
        rc = getattr(lib, name)(*given, workspace.data_ptr() if bytes_ else None, bytes_, _stream_ptr(dev))
    _lib.check(rc)
    return out


def keep_kv_mxfp4(caches, page_table, seq_lens, cu_q, path, accepted, kept_lens=None, *, max_q=None):
    """Move the kept ones of each sequence's last tokens together, in the caches of all layers at once.  Returns int32 ``kept_lens`` ``[B]``.

    ``caches``: one cache, or a list of them of one shape.  Of the last ``n = cu_q[b+1] - cu_q[b]`` tokens of sequence ``b``, those at ``path[cu_q[b] + i]``,
    ``i < accepted[b]`` (int32 ``[T]`` and ``[B]``; rising), go to places ``seq_lens[b] - n + i``, keys, values and scales as they are; ``kept_lens`` is
    ``seq_lens - n + accepted``, the lengths that are left (it must not be one of the inputs).  With what :func:`verify_draft` returns a checked draft
    becomes part of its sequence; with ``n`` the whole sequence, tokens that a policy gives up leave the cache.  What stands behind the kept
    tokens stays as it was.  Pages that hold moved tokens must belong to one sequence only.  ``max_q``: a bound on ``n``, if the host knows one (without, the mean is
    taken); it helps to choose the kernel."""
    done = _native.keep_kv_mxfp4(caches, page_table, seq_lens, cu_q, path, accepted, kept_lens, max_q)
    if done is not None:
        return done
    if isinstance(caches, (tuple, list)) and len(caches) == 4 and all(isinstance(t, torch.Tensor) for t in caches):
        caches = [caches]
    if not isinstance(caches, (tuple, list)) or not caches:
        raise TypeError("caches must be a cache or a list of caches.")
    views = [_cache(c) for c in caches]
    dev = views[0][1]
    if any(d != dev for _, d in views):
        raise ValueError(f"all caches must be on device {dev}.")
    if not isinstance(path, torch.Tensor) or path.dim() != 1 or not isinstance(page_table, torch.Tensor) or page_table.dtype != torch.int32 or page_table.dim() != 2:
        raise ValueError("path must be a 1-D and page_table a 2-D torch.int32 tensor.")
    b, width = _sizes(page_table, "page_table").shape
    if page_table.device != dev:
        raise ValueError(f"page_table must be on device {dev}, got {page_table.device}.")
    if width > 1 and page_table.stride(1) != 1:
        raise ValueError("page_table must have consecutive entries in a row.")
    t = path.shape[0]
    k = _lib.Keep(page_table=page_table.data_ptr(), page_table_stride=page_table.stride(0), tokens=t, batch=b, table_pages=width,
                  max_q=_int32(-(-t // max(b, 1)) if max_q is None else max_q))
    k.seq_lens, k.cu_q = _vector(seq_lens, "seq_lens", torch.int32, b, dev), _vector(cu_q, "cu_q", torch.int32, b + 1, dev)
    k.path, k.accepted = _vector(path, "path", torch.int32, t, dev), _vector(accepted, "accepted", torch.int32, b, dev)
    if kept_lens is None:
        kept_lens = torch.empty(b, dtype=torch.int32, device=dev)
    k.kept_lens = _vector(kept_lens, "kept_lens", torch.int32, b, dev)
    lib = _lib.load()
    with torch.cuda.device(dev):
        rc = lib.ave_fp4_keep_kv_mxfp4((_lib.KVCache * len(views))(*(c for c, _ in views)), len(views), _ref(k), _stream_ptr(dev))
    _lib.check(rc)
    return kept_lens
