"""GPU parity of decoding with drafted tokens (model/draft.py): the tree attention, the verification and the commit
against their 64-bit restatements (oracle/draft.py), and a whole step of them, eager and captured."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from helpers import rel_max, to_np
from oracle import draft as OD

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# Scores are 32-bit sums of 64 products, |s| < 30: e^s is off by at most 30 * 64 * 2^-24 = 1.1e-4 where every rounding
# goes one way, by the root of that count in practice; the outputs average such errors over the keys. As for the
# one-token attention.
TOL = 2e-5


def _cfg(n_head, n_kv, window=0):
    from nurostream_amd.model.decode import AttnConfig
    return AttnConfig(n_head=n_head, n_head_kv=n_kv, head_dim=64, vocab_size=10, rope_base=150000.0,
                      context_length=131072, sliding_window=window)


def _parents(n, kind, seed=0):
    if kind == "chain":
        return [i - 1 for i in range(n)]
    if kind == "flat":
        return [-1] + [0] * (n - 1)
    if kind == "roots":
        return [-1] * n
    r = np.random.default_rng(seed)
    return [-1] + [int(r.integers(max(0, i - 5), i)) for i in range(1, n)]


def _state(dev, n_head, n_kv, n, pos, dtype="f32", seed=0, ctx=None, max_nodes=None):
    """(cfg, kv at pos, draft, q): normal rows; what no call may read holds NaN."""
    from nurostream_amd.model.decode import DeviceKV
    from nurostream_amd.model.draft import DraftKV
    c = _cfg(n_head, n_kv)
    g = torch.Generator().manual_seed(seed)
    kv = DeviceKV(1, c, max(1, pos + 40) if ctx is None else ctx, dev, dtype=TYPES[dtype])
    draft = DraftKV(kv, c, max_nodes=max_nodes or n)
    for t, m in ((kv.k[0], pos), (kv.v[0], pos), (draft.k[0], n), (draft.v[0], n)):
        t.fill_(float("nan"))
        t[:, :m] = torch.randn(n_kv, m, 64, generator=g).to(dev).to(t.dtype)
    draft.workspace.fill_(255)  # NaN: nothing there is read before it is written
    kv.pos.fill_(pos)
    q = (torch.randn(n, n_head * 64, generator=g) * 1.5).to(dev)
    sinks = torch.randn(n_head, generator=g).to(dev)
    return c, kv, draft, q, sinks


def _ref(c, kv, draft, q, parents, sinks, window, pos):
    n = q.shape[0]
    f = lambda t, m: to_np(t[0][:, :m].double())  # noqa: E731
    return OD.tree_attention(to_np(q).reshape(n, c.n_head, 64), f(kv.k, pos), f(kv.v, pos), f(draft.k, n),
                             f(draft.v, n), parents, None if sinks is None else to_np(sinks), window)


def _ids(parents, dev):
    return torch.tensor(parents, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("heads", [(16, 2), (3, 3), (5, 1), (32, 2), (64, 8)], ids=lambda h: f"{h[0]}q{h[1]}kv")
@pytest.mark.parametrize("n,kind", [(1, "chain"), (2, "tree"), (9, "tree"), (33, "tree"), (64, "chain"), (7, "roots")])
@pytest.mark.parametrize("ctx", [None, 9000])
def test_tree_attention_matches_oracle(dev, dtype, heads, n, kind, ctx):
    """One to 64 nodes over caches whose length lies on, before and behind the edges of tiles (32 keys), waves (128)
    and splits; 1 to 16 query heads per kv head. The cache's capacity, little more or 9000, chooses the kernel."""
    from nurostream_amd.model.draft import tree_attn
    for pos in (0, 1, 31, 32, 33, 127, 128, 129, 300, 1025):
        c, kv, draft, q, sinks = _state(dev, *heads, n, pos, dtype, seed=pos + n, ctx=ctx)
        parents = _parents(n, kind, seed=pos)
        s = sinks if pos % 2 else None
        out = tree_attn(q, c, draft, 0, s, 0, parents=_ids(parents, dev) if kind != "chain" else None)
        assert rel_max(to_np(out), _ref(c, kv, draft, q, parents, s, 0, pos)) < TOL, pos


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("window", [1, 2, 7, 31, 32, 33, 64, 128, 129, 1000])
def test_tree_attention_windows(dev, dtype, window):
    """Windows shorter than the tree is deep, at the tiles' edges and longer than the cache: nodes of different depths
    see different first rows; what lies outside every window holds NaN."""
    from nurostream_amd.model.draft import tree_attn
    for n, kind, pos in ((1, "chain", 400), (20, "tree", 400), (64, "chain", 400), (64, "chain", 5), (33, "tree", 130)):
        c, kv, draft, q, sinks = _state(dev, 16, 2, n, pos, dtype, seed=window + n)
        parents = _parents(n, kind, seed=window)
        ref = _ref(c, kv, draft, q, parents, sinks, window, pos)
        gone = max(0, pos + 1 - window)
        kv.k[0][:, :gone] = float("nan")
        kv.v[0][:, :gone] = float("nan")
        out = tree_attn(q, c, draft, 0, sinks, window, parents=_ids(parents, dev))
        assert rel_max(to_np(out), ref) < TOL, (n, pos)


@pytest.mark.parametrize("heads,n,pos", [((64, 8), 1, 9000), ((64, 8), 16, 9000), ((8, 8), 64, 5000), ((8, 1), 3, 20000)])
def test_tree_attention_long_cache(dev, heads, n, pos):
    """Many splits, the last one short; a cache far larger than its rows (splits without keys)."""
    from nurostream_amd.model.draft import tree_attn
    for ctx in (pos, 3 * pos):
        c, kv, draft, q, sinks = _state(dev, *heads, n, pos, "f32", seed=n, ctx=ctx)
        parents = _parents(n, "tree", seed=1)
        out = tree_attn(q, c, draft, 0, sinks, 0, parents=_ids(parents, dev))
        k = torch.cat([kv.k[0][:, :pos], draft.k[0]], 1).double()
        v = torch.cat([kv.v[0][:, :pos], draft.v[0]], 1).double()
        _, anc = OD.lineage(parents)
        seen = torch.cat([torch.ones(n, pos, dtype=torch.bool), torch.from_numpy(anc)], 1).to(dev)
        G, R = heads[1], heads[0] // heads[1]
        qd = q.double().reshape(n, G, R, 64)
        s = torch.stack([qd[:, g] @ k[g].T.contiguous() for g in range(G)], 1) / 8.0
        s = s.masked_fill(~seen[:, None, None], -math.inf)
        z = sinks.double().reshape(1, G, R, 1).expand(n, G, R, 1)
        w = torch.softmax(torch.cat([s, z], -1), -1)[..., :-1]
        ref = torch.stack([w[:, g] @ v[g] for g in range(G)], 1).reshape(n, -1, 64)
        assert rel_max(to_np(out), to_np(ref)) < TOL, ctx


WIDE = dict(ctx=70000)  # a capacity from which many columns go to the kernel of 128 columns, however few the rows


def _gpu_ref(c, kv, draft, q, parents, sinks, window, pos):
    """oracle.draft.tree_attention in float64 on the device (tests/test_oracle_draft.py pins the restatement)."""
    n, G, R = q.shape[0], c.n_head_kv, c.n_head // c.n_head_kv
    k = torch.cat([kv.k[0][:, :pos], draft.k[0][:, :n]], 1).double()
    v = torch.cat([kv.v[0][:, :pos], draft.v[0][:, :n]], 1).double()
    depth, anc = OD.lineage(parents)
    at = torch.cat([torch.arange(pos), pos + torch.from_numpy(depth)])
    seen = torch.cat([torch.ones(n, pos, dtype=torch.bool), torch.from_numpy(anc)], 1)
    if window:
        seen &= (pos + torch.from_numpy(depth))[:, None] - at[None] < window
    seen = seen.to(q.device)
    qd = q.double().reshape(n, G, R, 64)
    s = torch.stack([qd[:, g].reshape(n * R, 64) @ k[g].T.contiguous() for g in range(G)], 1) / 8.0
    s = s.reshape(n, R, G, -1).transpose(1, 2).masked_fill(~seen[:, None, None], -math.inf)
    z = sinks.double().reshape(1, G, R, 1).expand(n, G, R, 1) if sinks is not None else torch.full_like(s[..., :1], -math.inf)
    w = torch.softmax(torch.cat([s, z], -1), -1)[..., :-1]
    return to_np(torch.stack([w[:, g].reshape(n * R, -1) @ v[g] for g in range(G)], 1).reshape(n, R, G, 64).transpose(1, 2)
                 .reshape(n, -1, 64))


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("heads,n,kind", [((32, 2), 64, "tree"), ((16, 1), 33, "chain"), ((24, 8), 50, "tree"),
                                          ((64, 8), 17, "roots"), ((15, 3), 64, "tree")])
def test_many_columns(dev, dtype, heads, n, kind):
    """More columns than 64 over caches whose length lies around the tiles (32 and 64 keys), pairs of them and splits;
    blocks of 128 columns that end inside."""
    from nurostream_amd.model.draft import tree_attn
    for pos in (0, 1, 31, 32, 33, 63, 64, 65, 127, 128, 129, 191, 255, 257, 1000, 5003):
        c, kv, draft, q, sinks = _state(dev, *heads, n, pos, dtype, seed=pos + n, **WIDE)
        parents = _parents(n, kind, seed=pos)
        s = sinks if pos % 2 else None
        out = tree_attn(q, c, draft, 0, s, 0, parents=_ids(parents, dev) if kind != "chain" else None)
        assert rel_max(to_np(out), _gpu_ref(c, kv, draft, q, parents, s, 0, pos)) < TOL, pos


@pytest.mark.parametrize("heads", [(16, 1), (32, 2)], ids=lambda h: f"{h[0]}q{h[1]}kv")
@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_many_columns_in_a_window(dev, dtype, heads):
    """Windows that end inside the cache, the nodes' first rows a few apart; rows before every window hold NaN."""
    from nurostream_amd.model.draft import tree_attn
    for window, pos, n, kind in ((33000, 33500, 64, "chain"), (33001, 33010, 40, "tree"), (40000, 39990, 64, "chain")):
        c, kv, draft, q, sinks = _state(dev, *heads, n, pos, dtype, seed=n, **WIDE)
        parents = _parents(n, kind, seed=window)
        ref = _gpu_ref(c, kv, draft, q, parents, sinks, window, pos)
        gone = max(0, pos + 1 - window)
        kv.k[0][:, :gone] = float("nan")
        kv.v[0][:, :gone] = float("nan")
        out = tree_attn(q, c, draft, 0, sinks, window, parents=_ids(parents, dev))
        assert rel_max(to_np(out), ref) < TOL, (window, pos)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_many_columns_beside_rows_of_anything(dev, bad, dtype):
    """As test_masked_rows_may_hold_anything, in the kernel of 128 columns; and a visible value row of infinities is
    infinite in its dimensions' outputs and leaves the others as they were."""
    from nurostream_amd.model.draft import tree_attn
    n, pos = 64, 700
    parents = _parents(n, "tree", seed=5)
    _, anc = OD.lineage(parents)
    leaf = [j for j in range(1, n) if anc[:, j].sum() == 1][:3]
    c, kv, draft, q, sinks = _state(dev, 32, 2, n, pos, dtype, seed=9, **WIDE)
    ref = _gpu_ref(c, kv, draft, q, parents, sinks, 0, pos)
    for j in leaf:
        draft.k[0][:, j] = bad
        draft.v[0][:, j] = bad
    others = [i for i in range(n) if i not in leaf]
    out = to_np(tree_attn(q, c, draft, 0, sinks, 0, parents=_ids(parents, dev)))
    assert rel_max(out[others], ref[others]) < TOL
    kv.v[0][:, 55, 3::7] = bad
    out = to_np(tree_attn(q, c, draft, 0, sinks, 0, parents=_ids(parents, dev)))
    hit = np.zeros(64, bool)
    hit[3::7] = True
    assert rel_max(out[others][..., ~hit], ref[others][..., ~hit]) < TOL
    if math.isnan(bad):
        assert np.isnan(out[others][..., hit]).all()
    else:
        assert (out[others][..., hit] == bad).all()


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_many_columns_keys_of_minus_infinity(dev, dtype):
    """Keys whose scores overflow to -infinity, whole tiles, pairs of tiles and splits of them (bf16 and fp32; fp16
    holds keys of -infinity themselves)."""
    from nurostream_amd.model.draft import tree_attn
    n = 64
    parents = _parents(n, "tree", seed=6)
    for pos, dead in ((64, range(0, 64)), (700, range(0, 640)), (700, range(3, 700, 2))):
        c, kv, draft, q, sinks = _state(dev, 16, 1, n, pos, dtype, seed=pos, **WIDE)
        q.reshape(n, 16, 64)[:, :, 0] = 1e20 if dtype != "f16" else 1.0
        kv.k[0][:, :pos, 0] = 0
        draft.k[0][:, :n, 0] = 0
        live = [r for r in range(pos) if r not in set(dead)]
        ref = OD.tree_attention(to_np(q).reshape(n, 16, 64), to_np(kv.k[0][:, live].double()),
                                to_np(kv.v[0][:, live].double()), to_np(draft.k[0].double()),
                                to_np(draft.v[0].double()), parents, to_np(sinks))
        kv.k[0][:, list(dead), 0] = -1e20 if dtype != "f16" else -math.inf
        out = tree_attn(q, c, draft, 0, sinks, 0, parents=_ids(parents, dev))
        assert rel_max(to_np(out), ref) < TOL, pos


def test_tree_attention_one_node_is_the_decode_attention(dev):
    """A tree of one node equals the one-token attention with that token's row already in the cache."""
    from nurostream_amd.model.decode import attn_decode
    from nurostream_amd.model.draft import tree_attn
    for pos, window in ((0, 0), (50, 0), (700, 0), (700, 128)):
        c, kv, draft, q, sinks = _state(dev, 16, 2, 1, pos, seed=pos)
        out = tree_attn(q, c, draft, 0, sinks, window)
        kv.k[0][:, pos], kv.v[0][:, pos] = draft.k[0][:, 0], draft.v[0][:, 0]
        one = attn_decode(q.reshape(-1), kv, 0, sinks, window, c)
        assert rel_max(to_np(out[0]), to_np(one)) < 2 * TOL, pos


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("ctx,pos,window", [(None, 200, 40), (6000, 2000, 1500)])
def test_masked_rows_may_hold_anything(dev, bad, dtype, ctx, pos, window):
    """NaN or infinite key and value rows of nodes that are nobody's ancestors, and of cache rows that only the
    shallower nodes' windows reach: the nodes that do not see them are as without them."""
    from nurostream_amd.model.draft import tree_attn
    n = 24
    parents = _parents(n, "tree", seed=3)
    parents[1:4] = [0, 0, 0]
    _, anc = OD.lineage(parents)
    leaf = [j for j in range(1, n) if anc[:, j].sum() == 1][:3]  # leaves: only they see themselves
    c, kv, draft, q, sinks = _state(dev, 16, 2, n, pos, dtype, seed=9, ctx=ctx)
    ref = _ref(c, kv, draft, q, parents, sinks, window, pos)
    for j in leaf:
        draft.k[0][:, j] = bad
        draft.v[0][:, j] = bad
    others = [i for i in range(n) if i not in leaf]
    out = to_np(tree_attn(q, c, draft, 0, sinks, window, parents=_ids(parents, dev)))
    assert np.isfinite(out[others]).all()
    assert rel_max(out[others], ref[others]) < TOL
    # the first row that node 0 alone sees (it is the shallowest)
    kv.k[0][:, pos + 1 - window] = bad
    kv.v[0][:, pos + 1 - window] = bad
    out = to_np(tree_attn(q, c, draft, 0, sinks, window, parents=_ids(parents, dev)))
    deeper = [i for i in others if i != 0]
    assert rel_max(out[deeper], ref[deeper]) < TOL


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("ctx", [None, 6000])
def test_keys_of_minus_infinity_have_no_weight(dev, dtype, ctx):
    """Keys whose scores overflow to -infinity, single ones and whole tiles and splits of them, beside others."""
    from nurostream_amd.model.draft import tree_attn
    n = 5
    parents = [-1, 0, 0, 1, 2]
    for pos, dead in ((10, range(10)), (64, range(0, 32)), (700, range(0, 640)), (700, range(3, 700, 2))):
        c, kv, draft, q, sinks = _state(dev, 8, 2, n, pos, dtype, seed=pos, ctx=ctx)
        qr = q.reshape(n, 8, 64)
        qr[:, :, 0] = 1e20
        kv.k[0][:, :pos, 0] = 0
        draft.k[0][:, :n, 0] = 0
        live = [r for r in range(pos) if r not in set(dead)]
        ref = OD.tree_attention(to_np(qr), to_np(kv.k[0][:, live].double()), to_np(kv.v[0][:, live].double()),
                                to_np(draft.k[0].double()), to_np(draft.v[0].double()), parents, to_np(sinks))
        kv.k[0][:, list(dead), 0] = -1e20
        out = tree_attn(q, c, draft, 0, sinks, 0, parents=_ids(parents, dev))
        assert rel_max(to_np(out), ref) < TOL, pos


@pytest.mark.parametrize("ctx", [None, 6000, 70000])
@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_queries_of_any_size(dev, dtype, ctx):
    """Small queries over large keys, large ones over small keys (subnormal ones in fp16), a node's queries of zeros, of
    differing sizes by head, and values of any size: each output beside its own largest value."""
    from nurostream_amd.model.draft import tree_attn
    n, pos, heads = 40, 150, (32, 2)
    for up in (-20, 18):
        c, kv, draft, q, sinks = _state(dev, *heads, n, pos, dtype, seed=up + 50, ctx=ctx)
        parents = _parents(n, "tree", seed=2)
        size = 2.0 ** torch.arange(32, device=dev).remainder(7).neg()  # heads by 2^0 .. 2^-6
        q = (q.reshape(n, 32, 64) * size[:, None] * 2.0 ** up).reshape(n, -1).contiguous()
        q[3] = 0
        for t, m in ((kv.k[0], pos), (draft.k[0], n)):
            t[:, :m] = (t[:, :m].float() * 2.0 ** (-18 if up > 0 else 12)).to(t.dtype)
        for t, m in ((kv.v[0], pos), (draft.v[0], n)):
            t[:, :m] = (t[:, :m].float() * 2.0 ** (-up // 2)).to(t.dtype)
        ref = _ref(c, kv, draft, q, parents, sinks, 0, pos)
        out = to_np(tree_attn(q, c, draft, 0, sinks, 0, parents=_ids(parents, dev)))
        for h in range(32):
            assert rel_max(out[:, h], ref[:, h]) < TOL, (up, h)


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_wide_ranges_in_one_row(dev, dtype):
    """Value rows with elements 2^20 times their others (2^10 in fp16) and keys whose large element meets a query's
    zero: the small ones keep their bits. Column by column, each against its own largest value."""
    from nurostream_amd.model.draft import tree_attn
    big = 2.0 ** (10 if dtype == "f16" else 20)
    n, pos = 6, 333
    parents = _parents(n, "tree", seed=2)
    c, kv, draft, q, sinks = _state(dev, 16, 2, n, pos, dtype, seed=4)
    q.reshape(n, 16, 64)[:, :, 7] = 0
    for t, m in ((kv.k[0], pos), (draft.k[0], n)):
        t[:, :m, 7] *= big
    for t, m in ((kv.v[0], pos), (draft.v[0], n)):
        t[:, :m, ::5] *= big
    ref = _ref(c, kv, draft, q, parents, sinks, 0, pos)
    out = to_np(tree_attn(q, c, draft, 0, sinks, 0, parents=_ids(parents, dev)))
    for d in range(64):
        assert rel_max(out[..., d], ref[..., d]) < TOL, d


@pytest.mark.parametrize("heads,window", [((16, 2), 0), ((6, 2), 50), ((64, 8), 128)])
@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_tree_attention_qkv(dev, heads, window, dtype):
    """From raw projections: the nodes' rows are the bits that the one-token call appends at their positions (rounded
    to the cache's type), the output is tree_attn's of those rows, the projections are unchanged and rows past the
    nodes stay as they were."""
    from nurostream_amd.model.decode import DeviceKV, rope_kv_append, yarn_inv_freq
    from nurostream_amd.model.draft import tree_attn, tree_attn_qkv
    n, pos, (H, G) = 13, 201, heads
    for kind, bias in (("tree", True), ("chain", False)):
        parents = _parents(n, kind, seed=8)
        depth, _ = OD.lineage(parents)
        c, kv, draft, _, sinks = _state(dev, H, G, n, pos, dtype, seed=1, max_nodes=n + 3)
        inv, amp = yarn_inv_freq(c, dev)
        g = torch.Generator().manual_seed(6)
        qkv = torch.randn(n, (H + 2 * G) * 64, generator=g).to(dev)
        b = [torch.randn(m * 64, generator=g).to(dev) if bias else None for m in (H, G, G)]
        keep = qkv.clone()
        draft.k[0].fill_(float("nan")), draft.v[0].fill_(float("nan"))
        par = None if kind == "chain" else _ids(parents, dev)
        out = tree_attn_qkv(qkv, *b, c, inv, amp, draft, 0, sinks, window, parents=par)
        assert torch.equal(qkv, keep)
        one = DeviceKV(1, c, pos + n + 1, dev)
        q = torch.empty(n, H * 64, device=dev)
        for i in range(n):
            one.pos.fill_(pos + int(depth[i]))
            row = qkv[i].clone()
            rope_kv_append(row, *b, c, inv, amp, one, 0)
            q[i] = row[:H * 64]
            at = pos + int(depth[i])
            assert torch.equal(draft.k[0][:, i], one.k[0][:, at].to(kv.dtype)), i
            assert torch.equal(draft.v[0][:, i], one.v[0][:, at].to(kv.dtype)), i
        assert bool(draft.k[0][:, n:].isnan().all()) and bool(draft.v[0][:, n:].isnan().all())
        assert torch.equal(out, tree_attn(q, c, draft, 0, sinks, window, parents=par))
        assert rel_max(to_np(out), _ref(c, kv, draft, q, parents, sinks, window, pos)) < TOL


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("heads,n,kind,ctx", [((16, 2), 64, "tree", None), ((8, 8), 33, "chain", None),
                                              ((3, 1), 1, "chain", None), ((64, 8), 40, "tree", 9000),
                                              ((32, 2), 64, "tree", 70000), ((16, 16), 7, "roots", 70000)])
def test_tree_attention_qkv_equals_rotated_rows(dev, dtype, heads, n, kind, ctx):
    """From raw projections and from what it left of them (queries rotated on the host's orders, rows beside the
    cache): the same bits, over positions around tiles and splits, in every kernel (the capacity chooses it)."""
    from nurostream_amd.model.decode import DeviceKV, rope_kv_append, yarn_inv_freq
    from nurostream_amd.model.draft import tree_attn, tree_attn_qkv
    H, G = heads
    for pos, window in ((0, 0), (1, 0), (31, 0), (32, 9), (33, 0), (127, 70), (128, 0), (500, 0), (500, 128), (1500, 0),
                        *(((33500, 33001),) if ctx == 70000 else ())):
        c, kv, draft, _, sinks = _state(dev, H, G, n, pos, dtype, seed=pos, ctx=ctx)
        inv, amp = yarn_inv_freq(c, dev)
        g = torch.Generator().manual_seed(pos)
        qkv = torch.randn(n, (H + 2 * G) * 64, generator=g).to(dev)
        b = [torch.randn(m * 64, generator=g).to(dev) for m in (H, G, G)]
        draft.k[0].fill_(float("nan")), draft.v[0].fill_(float("nan"))
        parents = _parents(n, kind, seed=pos)
        par = None if kind == "chain" else _ids(parents, dev)
        out = tree_attn_qkv(qkv, *b, c, inv, amp, draft, 0, sinks, window, parents=par)
        depth, _ = OD.lineage(parents)
        one = DeviceKV(1, c, pos + 65, dev)
        q = qkv.clone()
        for i in range(n):
            one.pos.fill_(pos + int(depth[i]))
            rope_kv_append(q[i], *b, c, inv, amp, one, 0)
            at = pos + int(depth[i])
            assert torch.equal(draft.k[0][:, i], one.k[0][:, at].to(kv.dtype)), (pos, i)
            assert torch.equal(draft.v[0][:, i], one.v[0][:, at].to(kv.dtype)), (pos, i)
        again = tree_attn(q[:, :H * 64].contiguous(), c, draft, 0, sinks, window, parents=par)
        assert torch.equal(out, again), pos


def test_position_outside_the_cache_writes_nothing(dev):
    from nurostream_amd.model.decode import yarn_inv_freq
    from nurostream_amd.model.draft import commit, tree_attn, tree_attn_qkv
    for at in (-1, 9):
        c, kv, draft, q, sinks = _state(dev, 8, 2, 4, 8, ctx=8)
        kv.pos.fill_(at)
        rows = [t.clone() for t in (draft.k[0], draft.v[0], kv.k[0], kv.v[0])]
        out = torch.full((4, 8, 64), 7.0, device=dev)
        tree_attn(q, c, draft, 0, sinks, 0, out=out)
        inv, amp = yarn_inv_freq(c, dev)
        tree_attn_qkv(torch.ones(4, 12 * 64, device=dev), None, None, None, c, inv, amp, draft, 0, sinks, 0, out=out)
        commit(draft, _ids([0, 1, 2, 3], dev), _ids([3], dev))
        assert bool((out == 7.0).all()) and int(kv.pos) == at
        for t, r in zip((draft.k[0], draft.v[0], kv.k[0], kv.v[0]), rows):
            assert torch.equal(t.nan_to_num(5.0), r.nan_to_num(5.0))


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("layers,n_kv,n", [(1, 1, 1), (3, 2, 7), (5, 8, 64), (36, 8, 16)])
def test_commit_moves_the_accepted_rows(dev, dtype, layers, n_kv, n):
    """Every layer's accepted rows to the position, all other rows as they were; twice in a row; to the cache's end."""
    from nurostream_amd.model.decode import DeviceKV
    from nurostream_amd.model.draft import DraftKV, commit
    c = _cfg(n_kv, n_kv)
    g = torch.Generator().manual_seed(n)
    ctx = 3 * n + 5
    kv = DeviceKV(layers, c, ctx, dev, dtype=TYPES[dtype])
    draft = DraftKV(kv, c, max_nodes=min(64, n + 2))
    for t in (kv.k_stack, kv.v_stack, draft.k_stack, draft.v_stack):
        t.copy_(torch.randn(t.shape, generator=g))
    r = np.random.default_rng(n)
    pos = 2
    for _ in range(4):
        kv.pos.fill_(pos)
        count = int(r.integers(0, n + 1))
        path = np.sort(r.choice(n, count, replace=False))
        k, v = kv.k_stack.clone(), kv.v_stack.clone()
        for j, src in enumerate(path):
            if pos + j < ctx:
                k[:, :, pos + j], v[:, :, pos + j] = draft.k_stack[:, :, src], draft.v_stack[:, :, src]
        commit(draft, _ids(list(path) + [-1] * (n - count), dev), _ids([count], dev))
        pos = min(pos + count, ctx)
        assert torch.equal(kv.k_stack, k) and torch.equal(kv.v_stack, v) and int(kv.pos) == pos
        pos = min(ctx, pos + n // 2)


def test_commit_skips_bad_entries(dev):
    """Entries outside the nodes copy nothing; a count past the path is the path's length, one below zero none."""
    from nurostream_amd.model.draft import commit
    c, kv, draft, _, _ = _state(dev, 2, 2, 4, 3, ctx=20)
    k = kv.k[0].clone()
    commit(draft, _ids([0, -1, 99, 3], dev), _ids([9], dev))
    k[:, 3], k[:, 6] = draft.k[0][:, 0], draft.k[0][:, 3]
    assert torch.equal(kv.k[0].nan_to_num(5.0), k.nan_to_num(5.0)) and int(kv.pos) == 7
    commit(draft, _ids([0, 1], dev), _ids([-3], dev))
    assert torch.equal(kv.k[0].nan_to_num(5.0), k.nan_to_num(5.0)) and int(kv.pos) == 7


def test_refusals_of_tensors(dev):
    """Wrong types, sizes, layouts and another model's heads are refused before any launch."""
    from nurostream_amd.model.decode import yarn_inv_freq
    from nurostream_amd.model.draft import commit, tree_attn, tree_attn_qkv, verify
    n, H, G = 4, 8, 2
    c, kv, draft, q, sinks = _state(dev, H, G, n, 5, ctx=20)
    inv, amp = yarn_inv_freq(c, dev)
    par, qkv = _ids([-1, 0, 0, 1], dev), torch.zeros(n, (H + 2 * G) * 64, device=dev)
    attn = lambda **kw: tree_attn(**{**dict(q=q, cfg=c, draft=draft, layer=0, sinks=sinks, window=0, parents=par), **kw})  # noqa: E731
    raw = lambda **kw: tree_attn_qkv(**{**dict(qkv=qkv, bq=None, bk=None, bv=None, cfg=c, inv_freq=inv, amp=amp,  # noqa: E731
                                               draft=draft, layer=0, sinks=sinks, window=0, parents=par), **kw})
    wide = torch.zeros(n, 2 * H * 64, device=dev)
    z = lambda *s: torch.zeros(*s, device=dev)  # noqa: E731
    for kw in (dict(cfg=_cfg(H, 4)), dict(cfg=_cfg(H, 1)), dict(cfg=_cfg(16, G), q=z(n, 16 * 64)), dict(q=z(5, H * 64)),
               dict(q=wide[:, ::2]), dict(q=z(n, H * 64 - 1)), dict(sinks=z(H + 1)), dict(parents=par[:3]),
               dict(out=z(n, H, 63)), dict(window=-1), dict(q=z(0, H * 64)), dict(sinks=sinks.cpu())):
        with pytest.raises(ValueError):
            attn(**kw)
    for kw in (dict(q=q.half()), dict(parents=par.long()), dict(sinks=sinks.double()), dict(out=z(n, H, 64).half())):
        with pytest.raises(TypeError):
            attn(**kw)
    for layer in (-1, 1):
        with pytest.raises(IndexError):
            attn(layer=layer)
    for kw in (dict(qkv=q), dict(bq=z(H * 64 - 64)), dict(bk=z(H * 64)), dict(bv=z(1)), dict(inv_freq=z(64)),
               dict(cfg=_cfg(H, 4), qkv=z(n, 16 * 64))):
        with pytest.raises(ValueError):
            raw(**kw)
    path, count = _ids([0, 1], dev), _ids([2], dev)
    for args in ((path.long(), count), (path, count.long())):
        with pytest.raises(TypeError):
            commit(draft, *args)
    for args in ((_ids([0] * 5, dev), count), (path, path), (_ids([0] * 4, dev)[::2], count)):
        with pytest.raises(ValueError):
            commit(draft, *args)
    x, tok, u = z(2, 3, 50), _ids([[0, 1, 2]] * 2, dev), z(2, 3)
    ver = lambda **kw: verify(**{**dict(logits=x, tokens=tok, uniforms=u, temperature=1.0), **kw})  # noqa: E731
    for kw in (dict(tokens=tok[:1]), dict(uniforms=None), dict(uniforms=u[:1]), dict(parents=_ids([-1, 0], dev)),
               dict(parents=_ids([-1, 0, 0], dev), draft_probs=z(2, 2, 50)), dict(draft_probs=z(2, 3, 50)),
               dict(lengths=_ids([1], dev)), dict(temperature=-1.0), dict(temperature=float("nan")), dict(logits=z(50)),
               dict(logits=z(1, 65, 50), tokens=_ids([0] * 65, dev), uniforms=z(65)), dict(logits=z(2, 3, 0))):
        with pytest.raises(ValueError):
            ver(**kw)
    for kw in (dict(logits=x.double()), dict(tokens=tok.long()), dict(uniforms=u.double()), dict(draft_probs=z(2, 2, 50).half())):
        with pytest.raises(TypeError):
            ver(**kw)
    assert int(kv.pos) == 5 and ver(logits=z(0, 3, 50), tokens=tok[:0], uniforms=u[:0])[0].shape == (0,)


# -- verification ---------------------------------------------------------------


def _verify_case(seed, B, n, V, kind, q, dtype, T, dev):
    """Logits with a few large ones, drafts that are mostly likely, and uniforms of which none lies within 1e-9 of a
    decision (the restatement and the kernel may round differently there)."""
    r = np.random.default_rng(seed)
    lg = r.standard_normal((B, n, V)) * 2
    for b in range(B):
        for i in range(n):
            lg[b, i, r.integers(0, V, 3)] += r.uniform(3, 9, 3)
    logits = torch.from_numpy(lg.astype(np.float32)).to(TYPES[dtype])
    lg = logits.double().numpy()
    parents = _parents(n, kind, seed)
    tokens = r.integers(0, V, (B, n))
    probs = None
    if q:
        probs = np.stack([[OD.target_probs(lg[b, i] + r.standard_normal(V), T or 1.0) for i in range(n - 1)]
                          for b in range(B)]).astype(np.float32) if n > 1 else np.zeros((B, 0, V), np.float32)
        for b in range(B):
            for i in range(n - 1):
                tokens[b, i + 1] = r.choice(V, p=probs[b, i].astype(np.float64) / probs[b, i].astype(np.float64).sum())
    else:
        for b in range(B):
            for i in range(1, n):
                p = parents[i]
                if p >= 0 and r.random() < 0.8:
                    tokens[b, i] = np.argsort(-lg[b, p])[r.integers(0, min(3, V))]
    return logits, tokens, parents, r.random((B, n)).astype(np.float32), probs


def _check_verify(dev, logits, tokens, parents, u, probs, T, lengths=None, par="shared"):
    from nurostream_amd.model.draft import verify
    B, n, V = logits.shape
    lg = logits.double().cpu().numpy()
    want = [OD.verify_one(lg[b], tokens[b], parents, u[b], T, None if probs is None else probs[b],
                          None if lengths is None else lengths[b]) for b in range(B)]
    i32 = lambda a: torch.as_tensor(np.asarray(a), dtype=torch.int32, device=dev)  # noqa: E731
    pt = None if par is None else i32(parents) if par == "shared" else i32([parents] * B)
    count, path, token = verify(logits.to(dev), i32(tokens), torch.from_numpy(u).to(dev), parents=pt,
                                draft_probs=None if probs is None else torch.from_numpy(probs).to(dev),
                                temperature=T, lengths=None if lengths is None else i32(lengths))
    for b, (p, t) in enumerate(want):
        assert (int(count[b]), path[b].tolist(), int(token[b])) == (len(p), p + [-1] * (n - len(p)), t), b


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("V", [1, 2, 63, 4095, 4096, 4097, 20001])
@pytest.mark.parametrize("T", [0.0, 1.0, 0.6])
def test_verify_trees(dev, dtype, V, T):
    for seed, (B, n, kind) in enumerate([(1, 1, "chain"), (3, 2, "chain"), (2, 12, "tree"), (1, 64, "tree"), (2, 9, "flat")]):
        logits, tokens, parents, u, _ = _verify_case(seed + V, B, n, V, kind, False, dtype, T, dev)
        _check_verify(dev, logits, tokens, parents, u, None, T, par=("shared", "each")[seed % 2])


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("V", [2, 100, 4097, 20001])
def test_verify_drafts_from_q(dev, dtype, V):
    for seed, (B, n, T) in enumerate([(1, 1, 1.0), (4, 2, 1.0), (3, 6, 0.7), (2, 4, 1.4), (2, 5, 0.0)]):
        logits, tokens, parents, u, probs = _verify_case(seed + 7 * V, B, n, V, "chain", True, dtype, T, dev)
        _check_verify(dev, logits, tokens, parents, u, probs, T, par=None)


def test_verify_lengths(dev):
    for q, T in ((False, 0.0), (False, 0.8), (True, 0.8)):
        logits, tokens, parents, u, probs = _verify_case(3, 6, 5, 900, "chain", q, "f32", T, dev)
        u[:, 1:] = 0  # every draft of some probability is accepted: the lengths end the walks
        _check_verify(dev, logits, tokens, parents, u, probs, T, lengths=[5, 0, 1, 3, 9, -2], par=None)


def test_verify_reads_no_row_behind_a_length(dev):
    """Rows, probabilities and uniforms behind the lengths hold NaN: the same answers as with numbers there."""
    from nurostream_amd.model.draft import verify
    lengths = [5, 0, 1, 3, 9, -2]
    for q, T in ((False, 0.0), (False, 0.8), (True, 0.8)):
        logits, tokens, _, u, probs = _verify_case(5, 6, 5, 9001, "chain", q, "f32", T, dev)
        i32 = lambda a: torch.as_tensor(np.asarray(a), dtype=torch.int32, device=dev)  # noqa: E731
        run = lambda: verify(logits.to(dev), i32(tokens), torch.from_numpy(u).to(dev), temperature=T,  # noqa: E731
                             lengths=i32(lengths), draft_probs=None if probs is None else torch.from_numpy(probs).to(dev))
        want = run()
        for b, k in enumerate(lengths):
            k = max(0, min(k, 5))
            logits[b, k:], u[b, max(k, 1):] = math.nan, math.nan
            if probs is not None:
                probs[b, max(k - 1, 0):] = math.nan
        assert all(torch.equal(x, y) for x, y in zip(run(), want))


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_verify_residuals_captured(dev, dtype):
    """Drafts that q made too likely, refused over many chunks and sequences at once: each replay of a captured call,
    with eager calls between, gives the oracle's answers."""
    from nurostream_amd.model.draft import verify
    B, n, V, T = 9, 4, 50021, 0.9
    cases = [_verify_case(40 + i, B, n, V, "chain", True, dtype, T, dev) for i in range(3)]
    for logits, tokens, _, u, probs in cases:
        for b in range(B):
            for i in range(n - 1):  # q at the draft ten times what p has there
                if (b + i) % 2:
                    row = OD.target_probs(logits[b, i].double().numpy(), T)
                    probs[b, i, tokens[b, i + 1]] = 10 * row[tokens[b, i + 1]] + 0.01
                    u[b, i + 1] = 0.5
    dev_of = lambda c: [c[0].to(dev), torch.from_numpy(c[1]).to(torch.int32).to(dev),  # noqa: E731
                        torch.from_numpy(c[3]).to(dev), torch.from_numpy(c[4]).to(dev)]
    bufs = dev_of(cases[0])
    call = lambda x: verify(x[0], x[1], x[2], draft_probs=x[3], temperature=T)  # noqa: E731
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call(bufs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        got = call(bufs)
    refused = 0
    for i in (1, 2, 0, 1):
        for a, b in zip(bufs, dev_of(cases[i])):
            a.copy_(b)
        graph.replay()
        eager = call(bufs)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager)), i
        logits, tokens, parents, u, probs = cases[i]
        for b in range(B):
            path, t = OD.verify_one(logits[b].double().numpy(), tokens[b], parents, u[b], T, probs[b])
            assert (int(got[0][b]), got[1][b].tolist(), int(got[2][b])) == (len(path), path + [-1] * (n - len(path)), t), b
            refused += len(path) < n
    assert refused >= 12


def test_verify_nothing_left_of_p(dev):
    """q twice p everywhere: what is refused leaves no residual, and the token is drawn from p."""
    V, T = 9001, 1.0
    logits, tokens, parents, u, _ = _verify_case(8, 3, 2, V, "chain", False, "f32", T, dev)
    probs = np.stack([[OD.target_probs(logits[b, 0].double().numpy(), T) * 2] for b in range(3)]).astype(np.float32)
    u[:, 1] = 0.75
    _check_verify(dev, logits, tokens, parents, u, probs, T, par=None)


def test_verify_refused_and_repeated_siblings(dev):
    """Uniforms near one refuse every child; the same token twice under a node, tokens outside the vocabulary, and a
    row whose mass the drafts hold between them."""
    V = 5000
    r = np.random.default_rng(1)
    logits = torch.from_numpy(r.standard_normal((1, 6, V)).astype(np.float32))
    parents = [-1, 0, 0, 0, 0, 1]
    for tokens in ([0, 7, 7, 9, 9, 1], [0, -1, V, 4999, 0, 1], [0, 1, 2, 3, 4, 5]):
        for u0 in (0.0, 0.3, 0.9999):
            u = np.full((1, 6), 0.999999, np.float32)
            u[0, 0] = u0
            _check_verify(dev, logits, np.array([tokens]), parents, u, None, 1.0)
    two = torch.full((1, 6, V), -math.inf)
    two[..., 11], two[..., 4500] = 1.0, 1.5
    for u in (0.1, 0.5, 0.99):
        _check_verify(dev, two, np.array([[0, 11, 4500, 3, 3, 11]]), parents, np.full((1, 6), u, np.float32), None, 1.0)


def test_verify_rows_of_infinities_and_nan(dev):
    """-infinity almost everywhere, everywhere, +infinity in places, NaN: the token has a weight, or is -1."""
    V = 9000
    lg = torch.full((5, 2, V), -math.inf)
    lg[0, :, 8999] = -3.0
    lg[2, :, 5], lg[2, :, 8000] = math.inf, math.inf
    lg[3] = 0.0
    lg[3, :, ::2] = float("nan")
    lg[4] = float("nan")
    tokens = np.array([[0, 8999], [0, 1], [0, 5], [0, 1], [0, 2]])
    for T in (0.0, 1.0):
        for u in (0.0, 0.49, 0.51, 0.99):
            _check_verify(dev, lg, tokens, [-1, 0], np.full((5, 2), u, np.float32), None, T)


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_verify_rows_apart(dev, dtype):
    """Logits as a slice of a padded vocabulary, starting at odd elements: no copy's difference to the answers."""
    from nurostream_amd.model.draft import verify
    V = 5003
    for T in (0.0, 0.9):
        logits, tokens, parents, u, _ = _verify_case(2, 2, 5, V, "tree", False, dtype, T, dev)
        wide = torch.full((2, 5, V + 14), 77.0, dtype=logits.dtype, device=dev)
        i32 = lambda a: torch.as_tensor(np.asarray(a), dtype=torch.int32, device=dev)  # noqa: E731
        args = (i32(tokens), torch.from_numpy(u).to(dev))
        want = verify(logits.to(dev), *args, parents=i32(parents), temperature=T)
        for off in (0, 1, 3, 7, 13):
            view = wide[:, :, off:off + V]
            view.copy_(logits)
            got = verify(view, *args, parents=i32(parents), temperature=T)
            assert all(torch.equal(a, b) for a, b in zip(got, want)), off
            got = verify(view[1], args[0][1:].contiguous(), args[1][1:].contiguous(), parents=i32(parents), temperature=T)
            assert all(torch.equal(a, b[1:]) for a, b in zip(got, want)), off


def test_verify_sampled_tokens_follow_the_target(dev):
    """20000 sequences of one row, drafts in place: the next tokens' frequencies against the target's law. A count of
    n trials at probability p is off by more than 6 sqrt(n p (1 - p)) + 6 once in 10^8."""
    from nurostream_amd.model.draft import verify
    B, V, T = 20000, 40, 0.9
    g = torch.Generator().manual_seed(2)
    row = torch.randn(V, generator=g) * 1.5
    logits = row.to(dev).expand(B, 2, V).contiguous()
    p = OD.target_probs(row.double().numpy(), T)
    u = torch.rand(B, 2, generator=g).to(dev)
    tokens = torch.randint(0, V, (B, 2), generator=g).to(torch.int32).to(dev)
    q = torch.softmax(torch.randn(V, generator=g), -1)
    drawn = torch.multinomial(q, B, replacement=True, generator=g).to(torch.int32).to(dev)
    for probs, tok in ((None, tokens), (q.to(dev).expand(B, 1, V).contiguous(), torch.stack([tokens[:, 0], drawn], 1))):
        count, _, token = verify(logits, tok.contiguous(), u, draft_probs=probs, temperature=T)
        nxt = torch.where(count == 2, tok[:, 1], token).cpu().numpy()
        seen = np.bincount(nxt, minlength=V)
        assert (np.abs(seen - B * p) <= 6 * np.sqrt(B * p * (1 - p)) + 6).all()


# -- a step of them together ----------------------------------------------------


def _step_inputs(dev, n, n_layer, H, G, V, seed):
    g = torch.Generator().manual_seed(seed)
    f = lambda *s: torch.randn(*s, generator=g).to(dev)  # noqa: E731
    return {"qkv": [f(n, (H + 2 * G) * 64) for _ in range(n_layer)], "logits": f(n, V) * 3,
            "tokens": torch.randint(0, V, (1, n), generator=g).to(torch.int32).to(dev),
            "u": torch.rand(1, n, generator=g).to(dev)}


@pytest.mark.parametrize("T", [0.0, 0.8])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_whole_step_captured(dev, T, dtype):
    """Attention of every layer, verification and commit as one graph: each replay, with eager work between, leaves
    the outputs, caches and positions of the eager step. On a side stream, the buffers of the default one."""
    from nurostream_amd.model.decode import DeviceKV, yarn_inv_freq
    from nurostream_amd.model.draft import DraftKV, commit, tree_attn_qkv, verify
    H, G, V, n, L, ctx = 16, 2, 6001, 11, 3, 400
    c = _cfg(H, G)
    inv, amp = yarn_inv_freq(c, dev)
    parents = _ids(_parents(n, "tree", 4), dev)
    bufs = _step_inputs(dev, n, L, H, G, V, 0)

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
        return att, count, path, token

    (kv_g, dg), (kv_e, de) = make(), make()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(bufs, dg)
    torch.cuda.synchronize()
    kv_g.k_stack.copy_(kv_e.k_stack), kv_g.v_stack.copy_(kv_e.v_stack), kv_g.pos.fill_(300)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        got = step(bufs, dg)
    for i in range(5):
        x = _step_inputs(dev, n, L, H, G, V, 10 + i)
        for key in bufs:
            for a, b in zip(bufs[key], x[key]):
                a.copy_(b)
        graph.replay()
        want = step(x, de)
        torch.cuda.synchronize()
        for a, b in zip((*got[0], *got[1:]), (*want[0], *want[1:])):
            assert torch.equal(a, b), i
        assert torch.equal(kv_g.k_stack, kv_e.k_stack) and torch.equal(kv_g.v_stack, kv_e.v_stack)
        assert torch.equal(kv_g.pos, kv_e.pos)
        _ = torch.randn(1000, device=dev).sum().item()


def test_two_drafts_on_two_streams(dev):
    """Calls with a DraftKV each, in flight together on two streams, are as one after the other."""
    from nurostream_amd.model.draft import tree_attn
    sets = [_state(dev, 64, 8, 16, 5000, "f32", seed=s) for s in (1, 2)]
    par = _ids(_parents(16, "tree", 2), dev)
    want = [tree_attn(q, c, d, 0, z, 0, parents=par) for c, _, d, q, z in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        outs = []
        for st, (c, _, d, q, z) in zip(streams, sets):
            with torch.cuda.stream(st):
                outs.append(tree_attn(q, c, d, 0, z, 0, parents=par))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


# -- in the model ------------------------------------------------------------------


def _tiny(tmp_path, dev):
    from test_gpu_decode import _tiny_model
    return _tiny_model(tmp_path, dev)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_forward_tree_equals_forward_of_each_path(dev, tmp_path, dtype):
    """Every node's logits are those of the one-token path over the prompt and the node's line (past the sliding
    window of 4); a prompt in pieces leaves the cache that one token at a time leaves. A 16-bit cache against passes
    of one node over a cache of the same type (an fp32 cache is no reference for it: the rows' rounding can change
    which experts a token takes): a row's element may round to either side of a tie between the two."""
    from helpers import MFMA_TOL
    from nurostream_amd.model.decode import DeviceKV
    from nurostream_amd.model.draft import DraftKV, commit
    ns, _ = _tiny(tmp_path, dev)
    model, c = ns.model, ns.model.attn_config()
    prompt = [5, 17, 42, 7, 250, 3, 99, 1, 288]
    tol = 2 * MFMA_TOL if dtype == "f32" else 2.0 ** -5
    kv = DeviceKV(ns.cfg.n_layer, c, 40, dev, dtype=TYPES[dtype])
    draft = DraftKV(kv, c, max_nodes=12)
    for piece in (prompt[:5], prompt[5:]):
        got = model.forward_tree(_ids(piece, dev), draft)
        commit(draft, _ids(range(len(piece)), dev), _ids([len(piece)], dev))
    def by_one(toks):
        """(logits, cache) of one token after the other."""
        one = DeviceKV(ns.cfg.n_layer, c, 40, dev, dtype=TYPES[dtype])
        if dtype == "f32":
            return model.forward(toks, one, last_only=False), one
        d1, out = DraftKV(one, c, max_nodes=1), []
        for t in toks:
            out.append(model.forward_tree(_ids([t], dev), d1))
            commit(d1, _ids([0], dev), _ids([1], dev))
        return torch.cat(out), one

    want, one = by_one(prompt)
    assert rel_max(to_np(got), to_np(want[5:])) < tol
    assert int(kv.pos) == len(prompt)
    for a, b in ((kv.k_stack, one.k_stack), (kv.v_stack, one.v_stack)):
        assert rel_max(to_np(a.float()), to_np(b.float())) < tol
    tokens, parents = [12, 30, 31, 8, 9, 30, 77], [-1, 0, 0, 1, 1, 2, 5]
    tree = model.forward_tree(_ids(tokens, dev), draft, _ids(parents, dev))
    last = model.forward_tree(_ids(tokens, dev), draft, _ids(parents, dev), last_only=True)
    assert rel_max(to_np(last), to_np(tree[-1:])) < tol
    for i in range(len(tokens)):
        line, j = [], i
        while j >= 0:
            line.insert(0, tokens[j])
            j = parents[j]
        ref = by_one(prompt + line)[0][-1]
        assert rel_max(to_np(tree[i]), to_np(ref)) < tol, i


def test_generate_with_drafts_is_generate(dev, tmp_path):
    """Greedy: the tokens with drafts are those without, whatever the number of drafts, also where the context or
    max_tokens ends in the middle of a pass. (The tiny model repeats itself, so drafts are accepted.)"""
    ns, _ = _tiny(tmp_path, dev)
    for prompt in ([11, 200, 37], [5, 6, 7, 5, 6, 7, 5, 6] * 10):
        want = list(ns.generate(prompt, max_tokens=40))
        for drafts in (1, 4, 15, 63):
            got = list(ns.generate(prompt, max_tokens=40, drafts=drafts))
            assert got == want, drafts
            assert ns.stats.generated_tokens == 40 and ns.stats.prompt_tokens == len(prompt)
            assert ns.stats.passes <= 40
        assert list(ns.generate(prompt, max_tokens=5, drafts=8)) == want[:5]
    assert list(ns.generate([1, 2], max_tokens=0, drafts=3)) == []
    with pytest.raises(ValueError):
        list(ns.generate([1], drafts=64))


def test_generate_ends_with_the_context(dev, tmp_path, monkeypatch):
    """A context that ends before max_tokens, in the middle of a pass, at the prompt's end and before it."""
    import dataclasses
    ns, _ = _tiny(tmp_path, dev)
    small = dataclasses.replace(ns.model.attn_config(), context_length=20)
    monkeypatch.setattr(ns.model, "attn_config", lambda: small)
    for prompt in ([5, 6, 7] * 3, [5, 6] * 10, [9]):
        want = list(ns.generate(prompt, max_tokens=50))
        assert len(want) == 21 - len(prompt)
        for drafts in (1, 7, 40):
            assert list(ns.generate(prompt, max_tokens=50, drafts=drafts)) == want
    for kw in ({}, dict(drafts=3)):
        with pytest.raises(ValueError):
            list(ns.generate([5] * 21, max_tokens=2, **kw))


def test_generate_sampled_and_16_bit(dev, tmp_path):
    """Sampling with drafts and 16-bit caches runs to its end, the same for the same seed."""
    ns, _ = _tiny(tmp_path, dev)
    for kw in (dict(drafts=6, temperature=0.9, top_p=0.9), dict(drafts=0, temperature=0.9, kv_dtype=torch.bfloat16),
               dict(drafts=5, kv_dtype=torch.float16)):
        runs = []
        for _ in range(2):
            torch.manual_seed(7)
            runs.append(list(ns.generate([4, 5, 4, 5, 4], max_tokens=20, **kw)))
        assert runs[0] == runs[1] and len(runs[0]) == 20
