"""Refusals of the drafted-decoding calls (model/draft.py) that end on the host: the C ABI's checks of sizes, types,
alignment and workspaces, and the Python calls' checks of their tensors (CPU only)."""
from __future__ import annotations

import pytest
import torch

from nurostream_amd import _native as N
from nurostream_amd.model.decode import AttnConfig, DeviceKV, attn_decode, attn_decode_qkv, rope_kv_append
from nurostream_amd.model.draft import MAX_NODES, DraftKV, commit, tree_attn, tree_attn_qkv, verify


@pytest.fixture(scope="module")
def lib():
    if not N.LIB_PATH.exists():
        from nurostream_amd import build
        build.build()
    return N.load()


def _cfg(n_head=16, n_kv=2, head_dim=64):
    return AttnConfig(n_head=n_head, n_head_kv=n_kv, head_dim=head_dim, vocab_size=10, rope_base=150000.0,
                      context_length=4096)


A = 1 << 20  # an address that no check follows


def _attn(lib, **kw):
    a = dict(q=A, k=A, v=A, dt=N.DT_F32, dk=A, dv=A, parents=None, n=4, m=4, sinks=None, H=16, G=2, d=64, pos=A, ctx=100,
             window=0, scale=0.125, ws=A, wsb=1 << 30, out=A)
    a.update(kw)
    rest = (a["k"], a["v"], a["dt"], a["dk"], a["dv"], a["parents"], a["n"], a["m"], a["sinks"], a["H"], a["G"], a["d"],
            a["pos"], a["ctx"], a["window"], a["scale"], a["ws"], a["wsb"], a["out"], None)
    both = {lib.nsx_tree_attn(a["q"], *rest), lib.nsx_tree_attn_qkv(a["q"], None, None, None, A, 1.0, *rest)}
    assert len(both) == 1
    return both.pop()


@pytest.mark.parametrize("kw,code", [
    (dict(d=128), N.ENOTIMPL), (dict(n=0), N.EINVAL), (dict(n=5), N.EINVAL), (dict(n=65, m=65), N.EINVAL),
    (dict(H=15), N.EINVAL), (dict(H=34), N.EINVAL), (dict(G=0), N.EINVAL), (dict(ctx=0), N.EINVAL),
    (dict(ctx=1 << 31), N.EINVAL), (dict(window=-1), N.EINVAL), (dict(dt=7), N.ETYPE), (dict(k=None), N.EINVAL),
    (dict(dv=None), N.EINVAL), (dict(pos=None), N.EINVAL), (dict(ws=None), N.EINVAL), (dict(out=None), N.EINVAL),
    (dict(q=None), N.EINVAL), (dict(k=A + 8), N.EINVAL), (dict(dk=A + 4), N.EINVAL), (dict(out=A + 4), N.EINVAL),
    (dict(ws=A + 8), N.EINVAL), (dict(wsb=4096), N.EINVAL)])
def test_tree_attention_refusals(lib, kw, code):
    assert _attn(lib, **kw) == code


def test_tree_attention_query_alignment(lib):
    """Rotated queries are read 16 bytes at a time."""
    args = (A, A, N.DT_F32, A, A, None, 4, 4, None, 16, 2, 64, A, 100, 0, 0.125, A, 1 << 30, A, None)
    assert lib.nsx_tree_attn(A + 4, *args) == N.EINVAL


def test_tree_workspace_serves_every_call(lib):
    """The size for max_nodes serves fewer nodes and any window: one byte less than a call needs is refused."""
    need = lib.nsx_tree_workspace_bytes(16, 2, 64, 64, 5000)
    assert need > 64 * 16 * 64 * 4
    sizes = [lib.nsx_tree_workspace_bytes(16, 2, 64, m, 5000) for m in (1, 2, 8, 33, 64)]
    assert sizes == sorted(sizes) and sizes[-1] == need
    assert lib.nsx_tree_workspace_bytes(16, 2, 64, 65, 5000) == -1
    assert lib.nsx_tree_workspace_bytes(16, 2, 128, 4, 5000) == -1
    assert lib.nsx_tree_workspace_bytes(16, 2, 64, 4, 0) == -1
    assert _attn(lib, n=4, m=4, ctx=5000, wsb=0) == N.EINVAL


def _commit(lib, **kw):
    a = dict(k=A, v=A, dk=A, dv=A, dt=N.DT_F16, L=2, G=2, d=64, n=4, m=4, path=A, count=A, pos=A, ctx=10, counter=A)
    a.update(kw)
    return lib.nsx_tree_commit(a["k"], a["v"], a["dk"], a["dv"], a["dt"], a["L"], a["G"], a["d"], a["n"], a["m"],
                               a["path"], a["count"], a["pos"], a["ctx"], a["counter"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(L=0), N.EINVAL), (dict(L=1 << 23), N.EINVAL), (dict(G=0), N.EINVAL), (dict(d=32), N.ENOTIMPL),
    (dict(n=5), N.EINVAL), (dict(n=0), N.EINVAL), (dict(dt=3), N.ETYPE), (dict(path=None), N.EINVAL),
    (dict(count=None), N.EINVAL), (dict(pos=None), N.EINVAL), (dict(counter=None), N.EINVAL), (dict(k=A + 2), N.EINVAL), (dict(ctx=0), N.EINVAL)])
def test_commit_refusals(lib, kw, code):
    assert _commit(lib, **kw) == code


def _verify(lib, **kw):
    a = dict(x=A, dt=N.DT_F32, ld=100, B=2, n=4, V=100, tok=A, par=None, ps=0, lens=None, u=A, q=None, T=1.0, c=A, p=A, t=A,
             ws=A, wsb=1 << 30)
    a.update(kw)
    return lib.nsx_verify(a["x"], a["dt"], a["ld"], a["B"], a["n"], a["V"], a["tok"], a["par"], a["ps"], a["lens"],
                          a["u"], a["q"], a["T"], a["c"], a["p"], a["t"], a["ws"], a["wsb"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(dt=5), N.ETYPE), (dict(n=0), N.EINVAL), (dict(n=65), N.EINVAL), (dict(B=-1), N.EINVAL),
    (dict(B=20000), N.EINVAL), (dict(V=0), N.EINVAL), (dict(V=1 << 23, ld=1 << 23), N.EINVAL), (dict(ld=99), N.EINVAL),
    (dict(T=-1.0), N.EINVAL), (dict(T=1e-40), N.EINVAL), (dict(T=float("nan")), N.EINVAL),
    (dict(T=float("inf")), N.EINVAL), (dict(u=None), N.EINVAL), (dict(q=A, par=A), N.EINVAL), (dict(ps=3), N.EINVAL),
    (dict(tok=None), N.EINVAL), (dict(x=None), N.EINVAL), (dict(ws=None), N.EINVAL), (dict(wsb=8), N.EINVAL),
    (dict(ws=A + 8), N.EINVAL)])
def test_verify_refusals(lib, kw, code):
    assert _verify(lib, **kw) == code


def test_verify_of_no_sequences(lib):
    assert _verify(lib, B=0) == N.OK
    assert lib.nsx_verify_workspace_bytes(0, 4, 100) == -1
    assert 0 < lib.nsx_verify_workspace_bytes(1, 4, 100) < lib.nsx_verify_workspace_bytes(3, 4, 100)


def test_python_refusals(lib):
    """What the Python calls refuse before any kernel: sizes, and tensors that are not on the GPU."""
    c = _cfg()
    kv = DeviceKV(2, c, 50, "cpu")
    with pytest.raises(TypeError):
        DeviceKV(1, c, 50, "cpu", dtype=torch.float64)
    for m in (0, MAX_NODES + 1):
        with pytest.raises(ValueError):
            DraftKV(kv, c, max_nodes=m)
    with pytest.raises(ValueError):
        DraftKV(kv, _cfg(n_kv=4), max_nodes=4)
    draft = DraftKV(kv, c, max_nodes=4)
    assert [t.shape for t in draft.k] == [(2, 4, 64)] * 2 and draft.k[1].data_ptr() != draft.k[0].data_ptr()
    x = torch.zeros(4, 16 * 64)
    with pytest.raises(N.NativeError):
        tree_attn(x, c, draft, 0, None, 0)
    with pytest.raises(N.NativeError):
        tree_attn_qkv(torch.zeros(4, 20 * 64), None, None, None, c, torch.zeros(32), 1.0, draft, 0, None, 0)
    with pytest.raises(N.NativeError):
        commit(draft, torch.zeros(4, dtype=torch.int32), torch.ones(1, dtype=torch.int32))
    with pytest.raises(N.NativeError):
        verify(torch.zeros(4, 10), torch.zeros(1, 4, dtype=torch.int32))
    with pytest.raises(ValueError):
        verify(torch.zeros(10), torch.zeros(1, dtype=torch.int32))


def test_one_token_calls_refuse_16_bit_caches(lib):
    c = _cfg()
    kv = DeviceKV(1, c, 8, "cpu", dtype=torch.bfloat16)
    q = torch.zeros(20 * 64)
    inv = torch.zeros(32)
    with pytest.raises(TypeError):
        rope_kv_append(q, None, None, None, c, inv, 1.0, kv, 0)
    with pytest.raises(TypeError):
        attn_decode(q, kv, 0, None, 0, c)
    with pytest.raises(TypeError):
        attn_decode_qkv(q, None, None, None, c, inv, 1.0, kv, 0, None, 0)


def test_lookup_drafts():
    from nurostream_amd.model.draft import LookupDrafts
    d = LookupDrafts([1, 2, 3, 4, 9, 1, 2, 3, 5, 6, 1, 2, 3])
    assert d.propose(0) == ([3], [-1])
    # the latest place first (5 6 1 2 ..), the earlier one beside it (4 9 1 ..), level by level
    assert d.propose(2) == ([3, 5, 4], [-1, 0, 0])
    assert d.propose(4) == ([3, 5, 4, 6, 9], [-1, 0, 0, 1, 2])
    assert d.propose(63, depth=1) == ([3, 5, 4], [-1, 0, 0])
    tokens, parents = d.propose(63)
    assert len(tokens) <= 64 and all(p < i for i, p in enumerate(parents))
    d.extend([5, 6, 1])  # both places agree now: one line of them
    assert d.propose(3, depth=3) == ([1, 2, 3], [-1, 0, 1]) or d.propose(3, depth=3)[0][:2] == [1, 2]
    assert LookupDrafts([7]).propose(5) == ([7], [-1])
    assert LookupDrafts([7, 8, 9]).propose(5) == ([9], [-1])
    assert LookupDrafts([4, 4, 4, 4]).propose(8, depth=2)[0] == [4, 4, 4]  # the places' lines merge
    with pytest.raises(ValueError):
        LookupDrafts([1], ngram=0)


def test_lookup_drafts_follow_earlier_places():
    """Every path of a proposal is a run of the sequence behind an earlier place of its last token."""
    import random
    from nurostream_amd.model.draft import LookupDrafts
    r = random.Random(3)
    seq = [r.randrange(6) for _ in range(300)]
    d = LookupDrafts(seq[:50])
    for t in seq[50:]:
        d.extend([t])
        tokens, parents = d.propose(r.randrange(1, 20))
        for i in range(1, len(tokens)):
            line, j = [], i
            while j >= 0:
                line.append(tokens[j])
                j = parents[j]
            line.reverse()
            runs = [d.tokens[k:k + len(line)] for k in range(len(d.tokens) - 1)]
            assert line in runs


@pytest.mark.parametrize("top_p", [0.1, 0.5, 0.9, 0.999, 1.0, 0.0])
def test_nucleus_keeps_what_sample_draws(top_p):
    """The rows' kept tokens are those that the one-token path draws from."""
    from nurostream_amd.api import NeuroStream
    lg = torch.randn(5, 40, generator=torch.Generator().manual_seed(1)) * 2
    kept = NeuroStream._nucleus(lg, 0.8, top_p) > float("-inf")
    for row, keep in zip(lg, kept):
        p, order = torch.sort(torch.softmax(row / 0.8, -1), descending=True)
        n = 40
        if 0 < top_p < 1:
            n = min(int(torch.searchsorted(torch.cumsum(p, 0), torch.tensor([top_p]))) + 1, 40)
        assert set(torch.nonzero(keep).flatten().tolist()) == set(order[:n].tolist())
    assert NeuroStream._nucleus(lg, 0.0, 0.5) is lg
