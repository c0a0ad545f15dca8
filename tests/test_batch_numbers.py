"""Whole numbers past the C entries' types: windows and top-k of the calls on several sequences keep their meaning (CPU only)."""
from __future__ import annotations

import pytest
import torch

from nurostream_amd import _native as N
from nurostream_amd.model import batch, sampling
from nurostream_amd.model.decode import AttnConfig


@pytest.fixture
def calls(monkeypatch):
    """What would be handed to the library, as its argument types take it."""
    got = []

    def call(what, fn, device, *args):
        got.append([t(a).value if t in (N._i, N._i64) else a for t, a in zip(N._SIGS["nsx_" + what][1], args)])

    for module in (batch, sampling):
        monkeypatch.setattr(module, "_call", call)
    monkeypatch.setattr(N, "require_device", lambda *t: None)
    return got


@pytest.mark.parametrize("window,want", [(0, 0), (1, 1), (2 ** 31 - 1, 2 ** 31 - 1), (2 ** 31, 2 ** 31 - 1), (2 ** 32 + 1, 2 ** 31 - 1),
                                         (2 ** 70 + 5, 2 ** 31 - 1)])
def test_windows(calls, window, want):
    cfg = AttnConfig(n_head=4, n_head_kv=2, head_dim=64, vocab_size=10, rope_base=150000.0, context_length=4096)
    kv = batch.BatchKV(1, cfg, 2, 10, "cpu")
    batch.batch_attn(torch.zeros(2, 1, 4, 64), cfg, kv, 0, None, window)
    at = len(calls[0]) - 5  # (window, scale, workspace, its bytes, out)
    assert calls[0][at] == want and calls[0][at + 1] == 0.125


@pytest.mark.parametrize("top_k,want", [(0, 0), (5, 5), (9, 9), (2 ** 33 + 1, 9), (2 ** 64 + 1, 9), (-1, -1), (-2 ** 64 + 3, -1)])
def test_top_k(calls, top_k, want):
    """A top-k past the vocabulary is all of it; one below zero stays one that is refused."""
    sampling.sample(torch.zeros(2, 9), torch.zeros(2), top_k=top_k)
    assert calls[0][6]._obj.top_k == want
