"""Drafted decoding on the host (CPU only): what its calls refuse beyond their tensors' types and sizes, the workspace's
size against every call's need, drafts looked up."""
from __future__ import annotations

import random
import re

import pytest
import torch

from nurostream_amd import _native as N
from nurostream_amd.model.decode import DeviceKV
from nurostream_amd.model.draft import DraftKV, LookupDrafts, commit
from test_draft import A, _cfg, lib  # noqa: F401  (a fixture)


def test_replaced_layers(lib):  # noqa: F811
    """commit moves rows from stack to stack: with a layer of the caller's in place of a view it is refused (the attention
    would have read that one)."""
    import copy
    import pickle
    c = _cfg()
    path, count = torch.zeros(4, dtype=torch.int32), torch.ones(1, dtype=torch.int32)

    def make():
        kv = DeviceKV(3, c, 50, "cpu")
        return kv, DraftKV(kv, c, max_nodes=4)

    def replace(lst):
        lst[1] = lst[1].clone()

    changes = [lambda kv, d: replace(kv.k), lambda kv, d: replace(kv.v), lambda kv, d: replace(d.k),
               lambda kv, d: replace(d.v), lambda kv, d: kv.k.reverse(), lambda kv, d: d.v.append(d.v.pop()),
               lambda kv, d: setattr(kv, "k", list(kv.k)), lambda kv, d: setattr(kv, "k", kv.v),
               lambda kv, d: setattr(kv, "v_stack", kv.v_stack.clone()), lambda kv, d: kv.v.__iadd__([kv.v[0]])]
    for change in changes:
        kv, d = make()
        change(kv, d)
        with pytest.raises(ValueError):
            commit(d, path, count)
    for kv, d in (make(), copy.deepcopy(make()), pickle.loads(pickle.dumps(make()))):
        assert kv.k[1].data_ptr() == kv.k_stack[1].data_ptr() and d.k[2].data_ptr() == d.k_stack[2].data_ptr()
        with pytest.raises(N.NativeError):  # on to the check for tensors on the GPU
            commit(d, path, count)


def test_lengths_past_the_cache(lib):  # noqa: F811
    """The host's mirror of the position says where rows would be dropped: a commit into a full cache, and attention or a
    commit behind its end, are refused before anything else."""
    from nurostream_amd.model.draft import tree_attn, tree_attn_qkv
    c = _cfg()
    kv = DeviceKV(1, c, 50, "cpu")
    d = DraftKV(kv, c, max_nodes=4)
    path, count = torch.zeros(4, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    calls = {"commit": lambda: commit(d, path, count), "attn": lambda: tree_attn(torch.zeros(4, 16 * 64), c, d, 0, None, 0),
             "qkv": lambda: tree_attn_qkv(torch.zeros(4, 20 * 64), None, None, None, c, torch.zeros(32), 1.0, d, 0, None, 0)}
    for length, refused in ((0, ()), (49, ()), (50, ("commit",)), (51, ("commit", "attn", "qkv"))):
        kv.length = length
        for name, call in calls.items():
            with pytest.raises(ValueError if name in refused else N.NativeError):
                call()


def _need(lib, H, G, n, m, ctx, window, dt):  # noqa: F811
    """The workspace that a call of n nodes asks for: from the refusal of one without bytes."""
    args = (A, A, A, dt, A, A, None, n, m, None, H, G, 64, A, ctx, window, 0.125, A)
    assert lib.nsx_tree_attn(*args, 0, A, None) == N.EINVAL
    need = int(re.search(r"workspace of 0 bytes, (\d+) needed", lib.nsx_last_error().decode()).group(1))
    assert lib.nsx_tree_attn(*args, need - 1, A, None) == N.EINVAL
    return need


@pytest.mark.parametrize("H,G", [(1, 1), (16, 1), (3, 3), (32, 2), (24, 8), (64, 8), (64, 64)])
def test_workspace_against_every_calls_need(lib, H, G):  # noqa: F811
    """The size for max_nodes covers each call of fewer nodes, any window and type, over capacities at which the kernels
    change; one call of max_nodes or fewer needs all of it, and one byte less is refused."""
    r = random.Random(H * 100 + G)
    for ctx in (1, 31, 500, 1500, 6000, 20000, 49151, 49152, 131072, 300001):
        for m in (1, 5, 17, 33, 64):
            size = lib.nsx_tree_workspace_bytes(H, G, 64, m, ctx)
            most = 0
            for n in range(1, m + 1):
                for dt in (N.DT_F32, N.DT_F16, N.DT_BF16):
                    most = max(most, _need(lib, H, G, n, m, ctx, 0, dt))
            assert most == size
            for _ in range(60):
                window = int(2 ** r.uniform(0, 18.5))
                assert _need(lib, H, G, r.randint(1, m), m, ctx, window, r.choice((N.DT_F32, N.DT_F16, N.DT_BF16))) <= size


def test_lookup_drafts_follow_the_latest_place_first():
    """Behind 1 2 3 5 6 1 the sequence went on with 2 3 5 6 1 .. (its latest place) and with 2 3 4 9 (an earlier one)."""
    d = LookupDrafts([1, 2, 3, 4, 9, 1, 2, 3, 5, 6, 1, 2, 3])
    d.extend([5, 6, 1])
    assert d.propose(3, depth=3) == ([1, 2, 3, 5], [-1, 0, 1, 2])
    assert d.propose(6, depth=3) == ([1, 2, 3, 5, 4], [-1, 0, 1, 2, 2])
