"""Drafted decoding next to its borders: acceptance that differs in late bits, and what a call meets at its ends."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from test_gpu_draft import _ids

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
