"""Plain implementations, in numpy and 64 bits, of what the entry points for drafted trees compute: ancestors, attention under any mask, the walk that
accepts nodes, the move of the kept tokens."""
from __future__ import annotations

import numpy as np
import torch

from tests.attention_helpers import SCORE


def random_parents(rng, n, chain=False):
    """Parents of n nodes; now and then a node hangs at none but the first."""
    return np.array([-1 if j == 0 else j - 1 if chain else int(rng.integers(max(0, j - 6), j)) for j in range(n)], np.int32)


def lines_of(parents):
    """For each node the nodes from the top down to it; a parent that is not below the node means none."""
    lines = []
    for i, p in enumerate(parents):
        lines.append((lines[p] if 0 <= p < i else []) + [i])
    return lines


def ancestors(parents):
    above = np.zeros((len(parents), len(parents)), bool)
    for i, line in enumerate(lines_of(parents)):
        above[i, line] = True
    return above


def words_of(above, words):
    """bool [rows, nodes] as int64 [rows, words], bit j % 64 of word j / 64."""
    out = np.zeros((above.shape[0], words), np.uint64)
    for i, j in np.argwhere(above[:, :64 * words]):
        out[i, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    return out.view(np.int64)


def visible(above, keys, window=0):
    """bool [nodes, keys] of one sequence: what each of its nodes, its last tokens, sees."""
    n = above.shape[0]
    seen = np.zeros((n, keys), bool)
    for i in range(n):
        for j in range(keys):
            node = j - (keys - n)
            seen[i, j] = above[i, node] if node >= 0 else not window or j >= keys - n + above[i].sum() - window
    return seen


def masked_reference(batch, masks, *, scale=None, sinks=None):
    """``(out, lse, out_bound, lse_bound)`` of a Batch whose sequence b has rows that see keys masks[b] (bool [rows, keys]); the bounds
    are those of Batch.reference: SCORE on a score, twice that on what follows it, 2^-8 for a probability rounded to bf16 and
    2^-8 for the result, 2^-16 for fp32 sums and exponentials."""
    scale = batch.d ** -0.5 if scale is None else scale
    out, lse = np.zeros(batch.q.shape), np.full(batch.q.shape[:2], -np.inf)
    tol, lse_tol = np.zeros(batch.q.shape), np.zeros(batch.q.shape[:2])
    group = batch.hq // batch.hkv
    for b, seen in enumerate(masks):
        for h in range(batch.hq):
            rows = slice(batch.cu[b], batch.cu[b + 1])
            q, k, v = batch.q[rows, h].astype(np.float64), batch.k[b][:, h // group], batch.v[b][:, h // group]
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


def softmax(x, temperature):
    x = np.where(np.isnan(x), -np.inf, np.minimum(x.astype(np.float64), np.finfo(np.float32).max))
    if x.max() == -np.inf:
        return np.zeros_like(x)
    e = np.exp((x - x.max()) / min(temperature, np.finfo(np.float32).max))
    return e / e.sum()


def verify_one(logits, tokens, parents, uniform, temperature, probs=None):
    """``(path, emitted)`` of one sequence, as the operator is described, a distribution after the other."""
    n, v = logits.shape
    if n == 0:
        return [], []
    u = np.where(uniform > 0, np.minimum(uniform, 1), 0).astype(np.float64)
    path, emitted = [0], []
    while True:
        node = path[-1]
        x = np.where(np.isnan(logits[node]), -np.inf, logits[node])
        best = int(np.argmax(x)) if x.max() > -np.inf else -1
        target = softmax(logits[node], temperature) if temperature > 0 else None
        r, accepted = target, None
        for c in (c for c in range(node + 1, n) if parents[c] == node):
            there = 0 <= tokens[c] < v
            if not temperature > 0:
                accepted = c if there and tokens[c] == best else None
            elif probs is None:
                if there and u[c] < r[tokens[c]]:
                    accepted = c
                elif there:
                    r = r.copy()
                    r[tokens[c]] = 0
                    r = r / r.sum() if r.sum() > 0 else r
            else:
                q = np.where(probs[node] > 0, probs[node], 0).astype(np.float64)
                if there and u[c] * q[tokens[c]] < r[tokens[c]]:
                    accepted = c
                else:
                    r = np.maximum(r - q, 0)
                    r = r / r.sum() if r.sum() > 0 else r
            if accepted is not None:
                break
        if accepted is None:
            break
        path.append(accepted)
        emitted.append(int(tokens[accepted]))
    if not temperature > 0:
        return path, emitted + [best]
    r = r if r.sum() > 0 else target
    if not r.sum() > 0:
        return path, emitted + [-1]
    above = np.flatnonzero(r.cumsum() > u[0] * r.sum())
    return path, emitted + [int(above[0]) if len(above) else int(np.flatnonzero(r)[-1])]


def verify_all(logits, tokens, parents, cu, uniform, temps, probs=None, fill=-7):
    """As the entry point returns it; rows of no sequence hold `fill`."""
    accepted, path, emitted = [], np.full(len(tokens), fill, np.int32), np.full(len(tokens), fill, np.int32)
    for b in range(len(cu) - 1):
        rows = slice(cu[b], cu[b + 1])
        p, e = verify_one(logits[rows], tokens[rows], parents[rows], uniform[rows], temps[b], None if probs is None else probs[rows])
        rest = [-1] * (cu[b + 1] - cu[b] - len(p))
        accepted.append(len(p))
        path[rows], emitted[rows] = p + rest, e + rest
    return np.array(accepted, np.int32), path, emitted


def keep_tokens(cache, table, lens, cu, path, accepted):
    """The four arrays of a cache ``[pages, heads, page, bytes]`` with the kept tokens moved, and the lengths that are left."""
    page = cache[0].shape[2]
    new, kept = [c.copy() for c in cache], []
    for b in range(len(lens)):
        n = int(cu[b + 1] - cu[b])
        base, many = int(lens[b]) - n, min(max(int(accepted[b]), 0), n)
        kept.append(base + many)
        for i in range(many):
            j = int(path[cu[b] + i])
            if not 0 <= j < n or min(base + i, base + j) < 0 or max(base + i, base + j) // page >= table.shape[1]:
                continue
            src, dst = table[b, (base + j) // page], table[b, (base + i) // page]
            if 0 <= src < cache[0].shape[0] and 0 <= dst < cache[0].shape[0]:
                for c, old in zip(new, cache):
                    c[dst, :, (base + i) % page] = old[src, :, (base + j) % page]
    return new, np.array(kept, np.int32)


def tensor(x, device):
    return torch.from_numpy(np.ascontiguousarray(x)).to(device)
