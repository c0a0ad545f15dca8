"""GPU parity of the drafted tokens' attention where a row's elements, or the softmax's weights, lie far apart: what is large
meets zeros, and what is left must keep its bits."""
from __future__ import annotations

import pytest
import torch

from helpers import rel_max, to_np
from test_gpu_draft import TOL, TYPES, _gpu_ref, _ids, _parents, _state

pytestmark = pytest.mark.gpu

# Capacities by which the kernels of 16 columns (one workgroup's keys, splits of them), 32 and 128 columns run: 40 nodes of 16
# query heads over 2 kv heads are 320 columns a kv head.
CTX = [None, 2000, 6000, 24000, 70000]


def _zero_keys(kv, draft, dims):
    for t in (kv.k[0], draft.k[0]):
        t[:, :, dims] = 0


@pytest.mark.parametrize("ctx", CTX)
@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_large_query_elements_over_zero_keys(dev, dtype, ctx):
    """A query element of 2^24 to 2^100 that every key meets with zero leaves the score to the others: they keep their
    bits. Every third node has one, in one head or all; the rest are as they were."""
    from nurostream_amd.model.draft import tree_attn
    n, pos = 40, 300
    parents = _parents(n, "tree", seed=3)
    for e in (24, 30, 40, 60, 100):
        c, kv, draft, q, sinks = _state(dev, 32, 2, n, pos, dtype, seed=e, ctx=ctx)
        _zero_keys(kv, draft, [7])
        ref = _gpu_ref(c, kv, draft, q, parents, sinks, 0, pos)  # (the element adds zero to every score)
        x = q.reshape(n, 32, 64)
        x[::3, :, 7] = 2.0 ** e
        x[1::3, 5, 7] = -(2.0 ** e)
        out = to_np(tree_attn(q, c, draft, 0, sinks, 0, parents=_ids(parents, dev)))
        assert rel_max(out, ref) < TOL, e


@pytest.mark.parametrize("ctx", CTX)
@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_small_query_elements_over_large_keys(dev, dtype, ctx):
    """The scores come from query elements 2^-16 to 2^-26 of the head's largest, over keys of 2^15, beside a large element
    over zero keys."""
    from nurostream_amd.model.draft import tree_attn
    n, pos = 40, 300
    parents = _parents(n, "tree", seed=4)
    for e in (16, 21, 26):
        c, kv, draft, q, sinks = _state(dev, 32, 2, n, pos, dtype, seed=e, ctx=ctx)
        _zero_keys(kv, draft, [0])
        for t, m in ((kv.k[0], pos), (draft.k[0], n)):
            t[:, :m] *= 2.0 ** 13  # |k| < 2^13 * 5.5 < 65504
        q *= 2.0 ** -13
        q.reshape(n, 32, 64)[..., 0] = 2.0 ** (e - 13)
        ref = _gpu_ref(c, kv, draft, q, parents, sinks, 0, pos)
        out = to_np(tree_attn(q, c, draft, 0, sinks, 0, parents=_ids(parents, dev)))
        assert rel_max(out, ref) < TOL, e


@pytest.mark.parametrize("ctx", CTX)
@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_large_projections_over_zero_keys(dev, dtype, ctx):
    """The same from raw projections: a large bias in a rotated pair of dimensions whose keys are zero, in one head."""
    from nurostream_amd.model.decode import yarn_inv_freq
    from nurostream_amd.model.draft import tree_attn_qkv
    n, pos, H, G = 40, 300, 32, 2
    parents = _parents(n, "tree", seed=5)
    c, kv, draft, _, sinks = _state(dev, H, G, n, pos, dtype, seed=2, ctx=ctx)
    inv, amp = yarn_inv_freq(c, dev)
    _zero_keys(kv, draft, [7, 39])
    qkv = torch.randn(n, (H + 2 * G) * 64, generator=torch.Generator().manual_seed(8)).to(dev)
    qkv.reshape(n, H + 2 * G, 64)[:, H:H + G, [7, 39]] = 0
    bq = torch.zeros(H * 64, device=dev)
    want = tree_attn_qkv(qkv, bq, None, None, c, inv, amp, draft, 0, sinks, 0, parents=_ids(parents, dev)).clone()
    bq.reshape(H, 64)[3, 7] = 2.0 ** 40
    got = tree_attn_qkv(qkv, bq, None, None, c, inv, amp, draft, 0, sinks, 0, parents=_ids(parents, dev))
    assert rel_max(to_np(got), to_np(want)) < 2 * TOL


@pytest.mark.parametrize("ctx", CTX)
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("at", [0, 171, 299])
def test_light_keys_under_a_heavy_one(dev, dtype, ctx, at):
    """One key has 2^20, 2^58 or 2^87 times the weight of every other and a value of zero: what the others leave is right
    beside itself."""
    from nurostream_amd.model.draft import tree_attn
    n, pos = 40, 300
    parents = _parents(n, "tree", seed=6)
    for above in (14.0, 40.0, 60.0):
        c, kv, draft, q, _ = _state(dev, 32, 2, n, pos, dtype, seed=9, ctx=ctx)
        _zero_keys(kv, draft, [7])
        q *= 0.05  # scores of deviation 0.1 beside each other
        q.reshape(n, 32, 64)[..., 7] = 8.0
        kv.k[0][:, at, 7] = above
        kv.v[0][:, at] = 0
        ref = _gpu_ref(c, kv, draft, q, parents, None, 0, pos)
        out = to_np(tree_attn(q, c, draft, 0, None, 0, parents=_ids(parents, dev)))
        assert rel_max(out, ref) < TOL, above


@pytest.mark.parametrize("ctx", CTX)
@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_infinite_queries(dev, dtype, ctx):
    """A query element of infinity whose keys all have the other sign: every score is -infinity and the sink has all the
    weight, as in the one-token attention. The other nodes and heads are as they were."""
    from nurostream_amd.model.decode import attn_decode
    from nurostream_amd.model.draft import tree_attn
    n, pos = 40, 300
    parents = _parents(n, "tree", seed=3)
    c, kv, draft, q, sinks = _state(dev, 32, 2, n, pos, dtype, seed=11, ctx=ctx)
    for t, m in ((kv.k[0], pos), (draft.k[0], n)):
        t[:, :m, 7] = t[:, :m, 7].abs() + 0.25
    ref = _gpu_ref(c, kv, draft, q, parents, sinks, 0, pos)
    x = q.reshape(n, 32, 64)
    x[5, :, 7] = -float("inf")
    x[9, 20, 7] = -float("inf")
    ref[5], ref[9, 20] = 0, 0
    out = to_np(tree_attn(q, c, draft, 0, sinks, 0, parents=_ids(parents, dev)))
    assert (out[5] == 0).all() and (out[9, 20] == 0).all()
    assert rel_max(out, ref) < TOL
    if dtype == "f32":
        kv.k[0][:, pos], kv.v[0][:, pos] = draft.k[0][:, 0], draft.v[0][:, 0]
        assert bool((attn_decode(q[5].contiguous(), kv, 0, sinks, 0, c) == 0).all())
