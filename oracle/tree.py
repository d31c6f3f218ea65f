"""CPU oracle for draft trees and eviction (numpy, float64).

TEST INFRASTRUCTURE ONLY: plain restatements, straight from the definitions, of
what the draft-tree attention, the acceptance of a tree, the commit of its
cache rows and the eviction by accumulated weight compute. The product path
(``asrback_b200``) never imports them.
"""

from __future__ import annotations

import numpy as np

from .attention import bf16_round

__all__ = ["plan", "norm_rotate", "tree_attention", "accept", "commit", "evict"]


def plan(parents, counts):
    """``(ancestors, depths)``: boolean ``(B, N, N)``, ``[b, i, j]`` true if
    node ``j`` is live node ``i`` or above it, and int ``(B, N)``."""
    batch, nodes = parents.shape
    above = np.zeros((batch, nodes, nodes), bool)
    depths = np.zeros((batch, nodes), np.int64)
    for b in range(batch):
        for i in range(counts[b]):
            j = i
            while j >= 0:
                above[b, i, j] = True
                j = parents[b, j]
            depths[b, i] = above[b, i].sum() - 1
    return above, depths


def norm_rotate(x, weight, cos, sin, eps):
    """Per-head RMSNorm then rotate-half RoPE; ``x`` (..., D), ``cos``/``sin``
    broadcast against it."""
    x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * weight
    half = x.shape[-1] // 2
    return x * cos + np.concatenate((-x[..., half:], x[..., :half]), -1) * sin


def tree_attention(q, k, v, keys, values, lengths, above, counts, scale, weights=None,
                   rotary=None, bf16=False):
    """``q`` (B, N, H, D), ``k``/``v`` (B, N, KVH, D), caches (B, L, KVH, D):
    returns ``out`` (B, N, H, D), the caches and weights after the call, and for
    tolerances ``mass`` (the outputs' sums of |p v|) and ``reach`` (each row's
    largest scale * sum |q k| and scale * max |q k|)."""
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    keys, values = np.array(keys, np.float64), np.array(values, np.float64)
    weights = None if weights is None else np.array(weights, np.float64)
    batch, nodes, heads, dim = q.shape
    kv_heads = k.shape[2]
    group = heads // kv_heads
    out, mass = np.zeros_like(q), np.zeros_like(q)
    reach = np.zeros((batch, nodes, heads, 2))
    for b in range(batch):
        n, m = int(counts[b]), int(lengths[b])
        if n == 0:
            continue
        qb, kb = q[b, :n], k[b, :n]
        if rotary is not None:
            wq, wk, eps, cos, sin, positions, depths = rotary
            at = positions[b] + depths[b, :n]
            qb = norm_rotate(qb, wq, cos[at][:, None], sin[at][:, None], eps)
            kb = norm_rotate(kb, wk, cos[at][:, None], sin[at][:, None], eps)
        if bf16:
            kb = bf16_round(kb.astype(np.float32)).astype(np.float64)
        keys[b, m:m + n], values[b, m:m + n] = kb, v[b, :n]
        if weights is not None:
            weights[b, :, m:m + n] = 0
        for i in range(n):
            seen = np.flatnonzero(np.concatenate((np.ones(m, bool), above[b, i, :n])))
            if seen.size == m:
                continue
            for h in range(heads):
                kh, vh = keys[b, seen, h // group], values[b, seen, h // group]
                s = kh @ qb[i, h] * scale
                p = np.exp(s - s.max())
                p /= p.sum()
                out[b, i, h] = p @ vh
                mass[b, i, h] = p @ np.abs(vh)
                terms = np.abs(kh * qb[i, h]) * scale
                reach[b, i, h] = terms.sum(1).max(), terms.max()
                if weights is not None:
                    weights[b, h // group, seen] += p
    return dict(out=out, keys=keys, values=values, weights=weights, mass=mass, reach=reach)


def accept(parents, counts, drafts, chosen, logprob, state, eos_ids, lengths=None):
    """The walk of every row and the state after it (``state`` as in
    :func:`oracle.step.update_state`): returns ``path``, ``counts``, ``start``,
    the state and the lengths."""
    batch, nodes = parents.shape
    state = {name: np.array(x, copy=True) for name, x in state.items()}
    lengths = None if lengths is None else np.array(lengths, copy=True)
    path = np.full((batch, nodes), -1, np.int64)
    taken = np.zeros(batch, np.int64)
    start = np.array(state["position"] if lengths is None else lengths, copy=True)
    for b in range(batch):
        at = 0 if counts[b] and not state["finished"][b] else None
        while at is not None:
            path[b, taken[b]] = at
            taken[b] += 1
            token = chosen[b, at]
            state["position"][b] += 1
            if lengths is not None:
                lengths[b] += 1
            state["tokens"][b] = token
            state["generated"][b, state["position"][b]] = token
            state["sum_logprobs"][b] += np.float32(logprob[b, at])
            if token in eos_ids or state["position"][b] >= state["end"][b]:
                state["finished"][b] = True
                break
            at = next((i for i in range(at + 1, counts[b])
                       if parents[b, i] == at and drafts[b, i] == token), None)
    return path, taken, start, state, lengths


def commit(cache, path, counts, start):
    """``cache`` (layers, B, L, ...) after the moves."""
    cache = np.array(cache, copy=True)
    for b in range(cache.shape[1]):
        source = start[b] + path[b, :counts[b]]
        cache[:, b, start[b]:start[b] + counts[b]] = cache[:, b, source]
    return cache


def evict(weights, lengths, budget, sink, recent):
    """``kept`` (layers, B, H, budget) old slots, -1 behind, of ``weights``
    (layers, B, H, L)."""
    layers, batch, heads, _ = weights.shape
    kept = np.full((layers, batch, heads, budget), -1, np.int64)
    for b in range(batch):
        n = int(lengths[b])
        if n <= budget:
            kept[:, b, :, :n] = np.arange(n)
            continue
        middle = np.arange(sink, n - recent)
        for layer in range(layers):
            for h in range(heads):
                w = np.array(weights[layer, b, h, middle], np.float64)
                w[np.isnan(w)] = -np.inf
                best = sorted(middle, key=lambda j, w=w: (-w[j - sink], j))[:budget - sink - recent]
                kept[layer, b, h] = sorted([*range(sink), *best, *range(n - recent, n)])
    return kept
