"""Drafted decoding on the host (CPU only): what its calls refuse beyond their tensors' types and sizes, the workspace's
size against every call's need, drafts looked up."""
from __future__ import annotations

import pytest
import torch

from nurostream_amd import _native as N
from nurostream_amd.model.decode import DeviceKV
from nurostream_amd.model.draft import DraftKV, commit
from test_draft import _cfg, lib  # noqa: F401  (a fixture)


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
