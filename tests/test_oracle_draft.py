"""The 64-bit restatement of drafted decoding (oracle/draft.py) against what it must equal."""
from __future__ import annotations

import numpy as np
import pytest

from oracle import attn as OA
from oracle import draft as OD


def _rows(seed, n_head=4, n_kv=2, pos=9, n=7):
    r = np.random.default_rng(seed)
    f = lambda *s: r.standard_normal(s)  # noqa: E731
    return f(n, n_head, 64), f(n_kv, pos, 64), f(n_kv, pos, 64), f(n_kv, n, 64), f(n_kv, n, 64), f(n_head)


@pytest.mark.parametrize("window", [0, 1, 4, 11])
def test_chain_is_causal_attention(window):
    """A chain is the causal sink attention's last rows over the cache and the chain."""
    q, k, v, nk, nv, sinks = _rows(1)
    n, H, _ = q.shape
    got = OD.tree_attention(q, k, v, nk, nv, list(range(-1, n - 1)), sinks, window)
    rep = H // k.shape[0]
    keys, vals = (OA.repeat_kv(np.concatenate(x, 1), rep) for x in ((k, nk), (v, nv)))
    pad = np.zeros((H, k.shape[1], 64))
    want = OA.sink_attention(np.concatenate([pad, q.transpose(1, 0, 2)], 1), keys, vals, sinks, window)
    np.testing.assert_allclose(got, want[:, -n:].transpose(1, 0, 2), rtol=0, atol=1e-12)


@pytest.mark.parametrize("window", [0, 2])
def test_tree_is_a_chain_per_leaf(window):
    q, k, v, nk, nv, sinks = _rows(2)
    parents = [-1, 0, 0, 1, 2, 2, 5]
    got = OD.tree_attention(q, k, v, nk, nv, parents, sinks, window)
    _, anc = OD.lineage(parents)
    for i in range(7):
        line = np.nonzero(anc[i])[0]
        one = OD.tree_attention(q[line], k, v, nk[:, line], nv[:, line], list(range(-1, len(line) - 1)), sinks, window)
        np.testing.assert_allclose(got[i], one[-1], rtol=0, atol=1e-12)


def test_no_parent_among_earlier_nodes_is_a_first_node():
    q, k, v, nk, nv, sinks = _rows(3)
    a = OD.tree_attention(q, k, v, nk, nv, [-1, -1, 0, 3, 99, -7, 4], sinks)
    b = OD.tree_attention(q, k, v, nk, nv, [-1, -1, 0, -1, -1, -1, 4], sinks)
    np.testing.assert_array_equal(a, b)


def _next_token_law(logits, tokens, parents, T, q, grid):
    """The law of the token behind node 0, by enumeration of uniforms at the grid's midpoints."""
    u = (np.arange(grid) + 0.5) / grid
    n, law = len(tokens), np.zeros(logits.shape[1])
    kids = [c for c in range(1, n) if parents[c] == 0]
    mesh = np.stack(np.meshgrid(*[u] * (1 + len(kids)), indexing="ij"), -1).reshape(-1, 1 + len(kids))
    for row in mesh:
        uni = np.zeros(n)
        uni[0], uni[kids] = row[0], row[1:]
        path, tok = OD.verify_one(logits, tokens, parents, uni, T, q)
        law[tokens[path[1]] if len(path) > 1 else tok] += 1.0 / len(mesh)
    return law


def test_accepted_tokens_follow_the_target():
    """Looked-up drafts (two siblings and the same token twice among three): whatever they are, the next token has the
    target's law. Each cell of the grid that a boundary crosses misplaces at most its own mass: the error is at most
    the boundaries (one per vocabulary entry and child) times 1 / grid."""
    r = np.random.default_rng(5)
    logits, T, grid = r.standard_normal((4, 5)), 0.7, 36
    p = OD.target_probs(logits[0], T)
    for tokens, parents in (([0, 3, 1], [-1, 0, 0]), ([0, 2, 2], [-1, 0, 0]), ([0, 9, 4], [-1, 0, 0]), ([0, 1], [-1, 0])):
        law = _next_token_law(logits, tokens, parents, T, None, grid)
        assert np.abs(law - p).max() <= (logits.shape[1] + 2) / grid, tokens


def test_drafts_from_q_follow_the_target():
    """A draft drawn from q: the law averaged over the draft is the target's, to the grid's resolution as above."""
    r = np.random.default_rng(6)
    logits, T, grid = r.standard_normal((2, 5)), 1.3, 120
    p, q = OD.target_probs(logits[0], T), OD.target_probs(r.standard_normal(5), 1.0)
    law = sum(q[x] * _next_token_law(logits, [0, x], [-1, 0], T, q[None], grid) for x in range(5))
    assert np.abs(law - p).max() <= (5 + 2) / grid


def test_greedy_and_edges():
    lg = np.array([[0.0, 3.0, 3.0], [1.0, 0.0, 2.0], [5.0, 0.0, 0.0]])
    assert OD.verify_one(lg, [0, 1, 2], [-1, 0, 1], None, 0.0) == ([0, 1, 2], 0)  # the lower of two equals
    assert OD.verify_one(lg, [0, 2, 2], [-1, 0, 1], None, 0.0) == ([0], 1)
    assert OD.verify_one(lg, [0, 2, 1, 2], [-1, 0, 0, 2], None, 0.0, length=3) == ([0, 2], 0)
    assert OD.verify_one(lg, [0, 1, 2], [-1, 0, 1], None, 0.0, length=0) == ([], -1)
    lg[0] = -np.inf
    assert OD.verify_one(lg, [0, 1], [-1, 0], [0.5, 0.0], 1.0) == ([0], -1)
    lg[0] = [np.nan, -np.inf, 1.0]
    assert OD.verify_one(lg, [0, 0], [-1, 0], [0.5, 0.0], 1.0) == ([0], 2)
    lg[0] = [np.inf, 0.0, np.inf]
    np.testing.assert_array_equal(OD.target_probs(lg[0], 1.0), [0.5, 0.0, 0.5])
