"""generate's filter ahead of verification (NeuroStream._nucleus): every combination of its filters, and no work for those that
are not asked for (CPU only)."""
from __future__ import annotations

import itertools

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from nurostream_amd.api import NeuroStream


def _kept(x, T, top_p, top_k, min_p):
    """Row by row, token by token, in 64 bits."""
    kept = torch.zeros_like(x, dtype=torch.bool)
    for r in range(x.shape[0]):
        w = torch.softmax(x[r].double() / T, -1).tolist()
        order = sorted(range(len(w)), key=lambda i: (-float(x[r, i]), i))
        order = order[:top_k] if top_k > 0 else order
        whole, before = sum(w[i] for i in order), 0.0
        for i in order:
            if 0 < top_p < 1 and not before < top_p * whole:
                break
            before += w[i]
            kept[r, i] = w[i] >= min_p * w[order[0]]
    return kept


@pytest.mark.parametrize("top_p,top_k,min_p", list(itertools.product((1.0, 0.35, 0.82), (0, 1, 17, 500), (0.0, 0.03, 1.0))))
def test_every_combination(top_p, top_k, min_p):
    x = 2 * torch.randn(6, 120, generator=torch.Generator().manual_seed(3))
    x[1, ::2] = -float("inf")
    x[2] = torch.round(x[2] * 4) / 4  # equal ones
    given = x.clone()
    got = NeuroStream._nucleus(x, 0.9, top_p, top_k, min_p)
    assert torch.equal(x, given)
    keep = _kept(x, 0.9, top_p, top_k, min_p)
    assert torch.equal(got, x.masked_fill(~keep, -float("inf")))


class _Ops(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.names.append(func._schema.name.split("::")[1])
        return func(*args, **(kwargs or {}))


def test_only_what_is_asked_for():
    """Top-p alone, as before there were other filters: no comparison for min-p, nothing joined."""
    x = torch.randn(2, 50)
    with _Ops() as ops:
        NeuroStream._nucleus(x, 0.9, 0.8)
    assert not {"lt", "arange", "bitwise_or", "bitwise_or_", "__or__", "__ior__", "logical_or"} & set(ops.names), ops.names
    with _Ops() as ops:
        assert NeuroStream._nucleus(x, 0.9, 1.0) is x and NeuroStream._nucleus(x, 0.0, 0.5, 3, 0.1) is x
    assert not ops.names
