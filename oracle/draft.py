"""CPU restatement (numpy, 64 bits) of decoding with drafted tokens: the attention of a tree of drafted tokens over a
cache and over their ancestors, and the verification of drafted tokens against the target's logits.

TEST INFRASTRUCTURE ONLY: no product code imports it. The reference decodes one token per forward, so there are no
reference lines to cite; the pins are in tests/test_oracle_draft.py (a chain against the causal sink attention of
oracle/attn.py, a tree against a chain per leaf, verified tokens against the target's distribution by enumeration).
"""
from __future__ import annotations

import math

import numpy as np


def lineage(parents) -> tuple[np.ndarray, np.ndarray]:
    """(depth of each node, [i, j]: j is i or an ancestor of i); a parent that is no earlier node is none."""
    n = len(parents)
    depth, anc = np.zeros(n, dtype=np.int64), np.eye(n, dtype=bool)
    for i, p in enumerate(parents):
        if 0 <= p < i:
            depth[i] = depth[p] + 1
            anc[i] |= anc[p]
    return depth, anc


def tree_attention(q, k, v, node_k, node_v, parents, sinks=None, window: int = 0, scale: float | None = None):
    """q (n, n_head, d); cache rows k, v (n_kv, pos, d); the nodes' rows (n_kv, n, d) -> (n, n_head, d).

    Node i, at position pos + depth(i), sees the cache's rows, its ancestors and itself, of these the last `window`
    positions when window > 0; softmax over [scores, sink] with the sink's column dropped."""
    q, k, v, node_k, node_v = (np.asarray(x, np.float64) for x in (q, k, v, node_k, node_v))
    n, n_head, d = q.shape
    n_kv, pos = k.shape[:2]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    depth, anc = lineage(parents)
    out = np.zeros_like(q)
    for i in range(n):
        first = max(0, pos + depth[i] + 1 - window) if window else 0
        own = [j for j in range(n) if anc[i, j] and (not window or depth[i] - depth[j] < window)]
        for h in range(n_head):
            g = h // (n_head // n_kv)
            keys = np.concatenate([k[g, first:], node_k[g, own]])
            vals = np.concatenate([v[g, first:], node_v[g, own]])
            s = keys @ q[i, h] * scale
            z = -math.inf if sinks is None else float(sinks[h])
            top = max(s.max(), z)
            w = np.exp(s - top)
            out[i, h] = w @ vals / (w.sum() + math.exp(z - top))
    return out


def target_probs(row, temperature: float) -> np.ndarray:
    """softmax(row / temperature); one at the largest, the lowest index of equals, at temperature 0. NaN counts as
    -infinity, infinities share the weight; all zero where the row has none."""
    row = np.where(np.isnan(row), -np.inf, np.asarray(row, np.float64))
    p = np.zeros(row.size)
    top = row.max()
    if top == -np.inf:
        return p
    if temperature == 0.0:
        p[int(np.argmax(row))] = 1.0
        return p
    p[row == top] = 1.0
    rest = row < top
    p[rest] = np.exp((row[rest] - top) / temperature)
    return p / p.sum()


def verify_one(logits, tokens, parents, uniforms, temperature: float, draft_probs=None, length: int | None = None):
    """One sequence: (accepted nodes, the token behind them or -1)."""
    n, vocab = len(tokens), np.asarray(logits).shape[1]
    length = n if length is None else min(length, n)
    if length <= 0:
        return [], -1
    path = [0]
    while True:
        cur = path[-1]
        p = target_probs(logits[cur], temperature)
        mass = p.copy()
        for c in range(cur + 1, length):
            if parents[c] != cur:
                continue
            x = int(tokens[c])
            have = mass[x] if 0 <= x < vocab else 0.0
            u = 0.0 if temperature == 0.0 else float(uniforms[c])
            if draft_probs is not None and temperature > 0.0:
                ok = u * float(draft_probs[cur][x]) < have if 0 <= x < vocab else False
                if not ok:
                    mass = np.maximum(p - np.asarray(draft_probs[cur], np.float64), 0.0)
            else:
                ok = u * mass.sum() < have
                if not ok and temperature > 0.0 and 0 <= x < vocab:
                    mass[x] = 0.0
            if ok:
                path.append(c)
                break
        else:
            break
    if not mass.sum() > 0.0:
        mass = p
    if not mass.sum() > 0.0:
        return path, -1
    run = np.cumsum(mass)
    u = 0.0 if temperature == 0.0 else float(uniforms[0])
    at = int(np.searchsorted(run, u * run[-1], side="right"))
    return path, min(at, int(np.nonzero(mass)[0][-1]))
