"""Drafted decoding next to its borders: acceptance that differs in late bits, and what a call meets at its ends."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from test_gpu_draft import TYPES, _cfg, _ids, _parents, _state, _step_inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1.0, 0.7])
def test_verify_accepts_to_the_late_bits(dev, T):
    """Drafts whose random number lies 2^-47 to 2^-41 of their probability beside it, two tokens each, T included: accepted
    where it is below and refused where it is not. (A weight of 64 bits is off by 2^-51 of itself and 6 / T steps of its
    exponent: 2^-49; the sum and the quotient add 2^-52.)"""
    from nurostream_amd.model.draft import verify
    r = np.random.default_rng(4)
    x = r.uniform(-6, 6, 8000000).astype(np.float32)
    p = 1 / (1 + np.exp(-x.astype(np.longdouble) / np.longdouble(T)))
    u = p.astype(np.float32)
    gap = ((p - u) / p).astype(np.float64)
    pick = np.flatnonzero((np.abs(gap) < 2.0 ** -41) & (np.abs(gap) > 2.0 ** -47) & (u < 1))
    assert len(pick) > 100
    B = len(pick)
    logits = torch.zeros(B, 2, 2)
    logits[:, :, 1] = torch.from_numpy(x[pick])[:, None]
    us = torch.full((B, 2), 0.5)
    us[:, 1] = torch.from_numpy(u[pick])
    count, _, _ = verify(logits.to(dev), _ids([[0, 1]] * B, dev), us.to(dev), temperature=T)
    assert (count.cpu().numpy() - 1 == (gap[pick] > 0)).all()


def test_attention_over_replaced_layers(dev):
    """A layer that the caller put in place of a view is read if it has the view's layout, and refused otherwise; commit
    refuses it either way."""
    from nurostream_amd.model.draft import commit, tree_attn
    c, kv, draft, q, sinks = _state(dev, 16, 2, 4, 50, "f32", seed=1)
    want = tree_attn(q, c, draft, 0, sinks, 0).clone()
    rows = kv.k[0]
    kv.k[0] = rows.clone()
    assert torch.equal(tree_attn(q, c, draft, 0, sinks, 0), want)
    with pytest.raises(ValueError):
        commit(draft, _ids([0], dev), _ids([1], dev))
    for bad, error in ((rows[:, :60].contiguous(), ValueError), (rows.half(), TypeError), (rows.cpu(), ValueError),
                       (rows.transpose(0, 1).contiguous().transpose(0, 1), ValueError)):
        kv.k[0] = bad
        with pytest.raises(error):
            tree_attn(q, c, draft, 0, sinks, 0)
    assert int(kv.pos) == 50


@pytest.mark.parametrize("kw", [dict(drafts=4), dict(drafts=0, kv_dtype=torch.bfloat16),
                                dict(drafts=4, temperature=0.8, top_p=1.0)])
def test_generate_without_a_number(dev, tmp_path, monkeypatch, kw):
    """Logits that are all NaN end the generation with an error, behind the tokens before them: of the prompt's last pass,
    or of a later one."""
    from test_gpu_decode import _tiny_model
    ns, _ = _tiny_model(tmp_path, dev)
    whole = ns.model.forward_tree
    for good in (0, 3):
        calls = []

        def pass_(*args, **kwargs):
            calls.append(0)
            x = whole(*args, **kwargs)
            return x if len(calls) <= good else torch.full_like(x, float("nan"))

        monkeypatch.setattr(ns.model, "forward_tree", pass_)
        got = []
        with pytest.raises(FloatingPointError):
            for piece in ns.generate([11, 200, 37], max_tokens=30, **kw):
                got.append(piece)
        assert len(got) >= good and len(calls) == good + 1


@pytest.mark.parametrize("ctx", [None, 50])
def test_generate_with_drafts_that_are_accepted(dev, tmp_path, monkeypatch, ctx):
    """Drafts that hold the tokens to come, each level a wrong one beside the right one: paths of several nodes are
    accepted, pass after pass, also up to the context's end; the tokens are those without drafts."""
    import dataclasses
    from test_gpu_decode import _tiny_model
    import nurostream_amd.model.draft as draft_calls
    ns, _ = _tiny_model(tmp_path, dev)
    if ctx:
        small = dataclasses.replace(ns.model.attn_config(), context_length=ctx)
        monkeypatch.setattr(ns.model, "attn_config", lambda: small)
    prompt = [11, 200, 37]
    want = list(ns.generate(prompt, max_tokens=60))
    known = prompt + [int(p[1:-1]) for p in want]

    class Known:
        def __init__(self, tokens):
            self.n = len(tokens)

        def extend(self, tokens):
            self.n += len(tokens)

        def propose(self, n_drafts, depth=None):
            nodes, parents, tip = [known[self.n - 1]], [-1], 0
            for level, t in enumerate(known[self.n:]):
                if level >= min(n_drafts, depth) or len(nodes) + 2 > n_drafts + 1:
                    break
                nodes += [(t + 1) % 300, t]
                parents += [tip, tip]
                tip = len(nodes) - 1
            return nodes, parents

    monkeypatch.setattr(draft_calls, "LookupDrafts", Known)
    for drafts in (2, 7, 12, 63):
        assert list(ns.generate(prompt, max_tokens=60, drafts=drafts)) == want
        s = ns.stats
        a_pass = drafts // 2 + 1  # tokens of a pass: the accepted drafts and the one that follows
        assert s.passes <= -(-(len(want) - 1) // a_pass) + 1
        assert s.accepted_tokens >= len(want) - 1 - s.passes and s.drafted_tokens <= drafts * s.passes


@pytest.mark.parametrize("T", [0.0, 0.8])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_whole_step_captured_with_accepted_paths(dev, T, dtype):
    """The captured step of test_gpu_draft.py with drafts that the target gives nearly all its weight: every replay commits
    a path of several nodes, whose rows and positions are the eager step's and are read by the next replay."""
    from nurostream_amd.model.decode import DeviceKV, yarn_inv_freq
    from nurostream_amd.model.draft import DraftKV, commit, tree_attn_qkv, verify
    H, G, V, n, L, ctx = 16, 2, 6001, 11, 2, 400
    c = _cfg(H, G)
    inv, amp = yarn_inv_freq(c, dev)
    tree = _parents(n, "tree", 4)
    parents = _ids(tree, dev)

    def inputs(seed):
        x = _step_inputs(dev, n, L, H, G, V, seed)
        g = torch.Generator().manual_seed(seed)
        for i in range(1, n):  # a child in two has the parent's heavy token
            if torch.rand(1, generator=g) < 0.5 or i == 1:
                x["logits"][tree[i], x["tokens"][0, i]] = 60.0
        return x

    def make():
        kv = DeviceKV(L, c, ctx, dev, dtype=TYPES[dtype])
        g = torch.Generator().manual_seed(1)
        for t in (kv.k_stack, kv.v_stack):
            t.copy_(torch.randn(t.shape, generator=g))
        kv.pos.fill_(300)
        return kv, DraftKV(kv, c, max_nodes=n)

    def step(x, draft):
        att = [tree_attn_qkv(x["qkv"][li], None, None, None, c, inv, amp, draft, li, None, 128 if li % 2 else 0,
                             parents=parents) for li in range(L)]
        count, path, token = verify(x["logits"], x["tokens"], x["u"], parents=parents, temperature=T)
        commit(draft, path[0], count)
        return (*att, count, path, token)

    (kv_g, dg), (kv_e, de) = make(), make()
    bufs = inputs(0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(bufs, dg)
    torch.cuda.synchronize()
    kv_g.k_stack.copy_(kv_e.k_stack), kv_g.v_stack.copy_(kv_e.v_stack), kv_g.pos.fill_(300)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        got = step(bufs, dg)
    counts = []
    for i in range(6):
        x = inputs(10 + i)
        for key in bufs:
            for a, b in zip(bufs[key], x[key]):
                a.copy_(b)
        before = int(kv_e.pos)
        graph.replay()
        want = step(x, de)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
        assert torch.equal(kv_g.k_stack, kv_e.k_stack) and torch.equal(kv_g.v_stack, kv_e.v_stack)
        counts.append(int(want[-3]))
        assert int(kv_g.pos) == int(kv_e.pos) == before + counts[-1]
        path = want[-2][0, :counts[-1]].tolist()
        for j, node in enumerate(path):
            assert torch.equal(kv_e.k_stack[:, :, before + j], de.k_stack[:, :, node])
            assert node == 0 or tree[node] == path[j - 1]
    assert min(counts) >= 2 and max(counts) >= 3
