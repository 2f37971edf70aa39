"""Plain implementations, in numpy, of what the attention entry points compute: the norm and rotation in single fp32 operations in
the documented order (bit for bit), and attention in fp64 with a bound on how far a result may be from it."""
from __future__ import annotations

import numpy as np
import torch

from oracle import fp4_oracle as orc

EPS = 1e-6


def bf16(x):
    """fp32 array rounded to bf16 values."""
    return orc.bf16_bits_to_f32(orc.f32_to_bf16_bits(np.asarray(x, np.float32)))


def norm_rope_f32(x, weight, cos, sin, positions, neighbours, eps=EPS):
    """``x`` fp32 ``[T, H, D]``; every product and sum rounded to fp32 by itself, squares added up neighbours first."""
    x = np.asarray(x, np.float32)
    d = x.shape[-1]
    with np.errstate(all="ignore"):
        if weight is not None:
            s = x * x
            while s.shape[-1] > 1:
                s = s[..., 0::2] + s[..., 1::2]
            r = np.float32(1) / np.sqrt(s / np.float32(d) + np.float32(eps))
            x = (x * r) * np.asarray(weight, np.float32)
        if cos is None:
            return x
        half = cos.shape[1]
        ok = (positions >= 0) & (positions < cos.shape[0])
        at = np.where(ok, positions, 0)
        c, n = (np.where(ok[:, None], t[at], np.float32(np.nan))[:, None].astype(np.float32) for t in (cos, sin))
        y = x.copy()
        a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if neighbours else (slice(0, half), slice(half, 2 * half))
        y[..., a] = x[..., a] * c - x[..., b] * n
        y[..., b] = x[..., b] * c + x[..., a] * n
    return y


def tables(rows, rot, seed=0):
    angle = np.arange(rows)[:, None] * 10000.0 ** (-np.arange(0, rot, 2) / rot)
    return np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)


class Batch:
    """Sequences ``[(new tokens, keys)]`` in a paged cache whose pages are in random order; what no token occupies -- the rest of last
    pages, pages of nobody -- holds 0xFF in codes and scales, and the page table's unused entries point outside the cache."""

    def __init__(self, rows, hq, hkv, d, page, seed, *, q_std=1.0, k_gain=1.0, spare=2):
        self.rows, self.hq, self.hkv, self.d, self.page = rows, hq, hkv, d, page
        rng = np.random.default_rng(seed)
        need = [-(-k // page) for _, k in rows]
        pages = sum(need) + spare
        order = rng.permutation(pages)
        self.table = np.full((len(rows), max(need + [1]) + 1), 1 << 30, np.int32)
        self.cache = [np.full((pages, hkv, page, n), 0xFF, np.uint8) for n in (d // 2, d // 32, d // 2, d // 32)]
        self.k, self.v, at = [], [], 0
        for b, (_, keys) in enumerate(rows):
            self.table[b, :need[b]] = order[at:at + need[b]]
            at += need[b]
            x = rng.standard_normal((2, keys, hkv, d)).astype(np.float32)
            x[0] *= k_gain * np.where(rng.random((hkv, d)) < 1 / 16, 4, 1).astype(np.float32)
            for i in range(2):
                codes, scale = orc.quantize_mxfp4(x[i].reshape(keys * hkv, d)) if keys else (np.zeros((0, d // 2), np.uint8), np.zeros((0, d // 32), np.uint8))
                codes, scale = codes.reshape(keys, hkv, d // 2), scale.reshape(keys, hkv, d // 32)
                for j in range(keys):
                    p = self.table[b, j // page]
                    self.cache[2 * i][p, :, j % page] = codes[j]
                    self.cache[2 * i + 1][p, :, j % page] = scale[j]
                values = orc.dequantize_mxfp4(codes.reshape(keys * hkv, d // 2), scale.reshape(keys * hkv, d // 32), np.float64) if keys else np.zeros((0, d))
                (self.k, self.v)[i].append(values.reshape(keys, hkv, d))
        new = [n for n, _ in rows]
        self.cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.q = bf16(q_std * rng.standard_normal((int(self.cu[-1]), hq, d)))
        self.sinks = rng.standard_normal(hq).astype(np.float32)

    def place(self, b, j):
        """Page and offset of token j of sequence b."""
        return self.table[b, j // self.page], j % self.page

    def tensors(self, device):
        t = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(device)   # noqa: E731
        return {"q": t(self.q).bfloat16(), "cache": tuple(t(c) for c in self.cache), "page_table": t(self.table),
                "seq_lens": t(np.array([k for _, k in self.rows], np.int32)), "cu_q": t(self.cu)}

    def reference(self, *, scale=None, window=0, sinks=None, causal=True):
        """``(out, lse, out_bound, lse_bound)`` in fp64.

        A score is off by at most ``SCORE`` of the sum of its products' magnitudes; e^score and what follows by twice that, and by
        the bf16 rounding of a probability (2^-8); the result is rounded to bf16 (2^-8).  fp32 sums and exponentials: 2^-16."""
        scale = self.d ** -0.5 if scale is None else scale
        out = np.zeros(self.q.shape)
        lse = np.full(self.q.shape[:2], -np.inf)
        tol, lse_tol = np.zeros(self.q.shape), np.zeros(self.q.shape[:2])
        group = self.hq // self.hkv
        for b, (new, keys) in enumerate(self.rows):
            pos = keys - new + np.arange(new)[:, None]
            j = np.arange(keys)
            seen = (j <= pos) if causal else np.ones((new, keys), bool)
            if window:
                seen = seen & (j > pos - window)
            for h in range(self.hq):
                rows = slice(self.cu[b], self.cu[b + 1])
                q, k, v = self.q[rows, h].astype(np.float64), self.k[b][:, h // group], self.v[b][:, h // group]
                s = np.where(seen, scale * (q @ k.T), -np.inf)
                delta = abs(scale) * SCORE * np.where(seen, np.abs(q) @ np.abs(k).T, 0)
                m = s.max(1, initial=-np.inf)
                if sinks is not None:
                    m = np.maximum(m, sinks[h])
                m0 = np.where(np.isfinite(m), m, 0)
                p = np.where(seen, np.exp(s - m0[:, None]), 0)
                total = p.sum(1) + (np.exp(sinks[h] - m0) if sinks is not None else 0)
                some = seen.any(1)
                with np.errstate(all="ignore"):
                    out[rows, h] = np.where(some[:, None], p @ v / total[:, None], 0)
                    weight = np.where(some[:, None], p @ np.abs(v) / total[:, None], 0)
                    lse[rows, h] = m0 + np.log(total)
                worst = delta.max(1, initial=0)
                tol[rows, h] = 2.0 ** -8 * np.abs(out[rows, h]) + (2.0 ** -8 + 2.0 ** -16 + 2 * worst[:, None]) * weight * (1 + 2.0 ** -7)
                lse_tol[rows, h] = worst + 2.0 ** -16 * (1 + np.abs(np.where(np.isfinite(lse[rows, h]), lse[rows, h], 0)))
        return out, lse, tol + 1e-30, lse_tol


#: how far a score may be off, in units of the sum of the magnitudes of its products: the queries' two 8-bit parts keep 2^-19 of the
#: row's largest element, and the matrix cores align the products of a step before they add them up
SCORE = 2.0 ** -14
