"""Drafted decoding next to its borders: acceptance that differs in late bits, and what a call meets at its ends."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from test_gpu_draft import _ids, _state

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
