"""Where several filters of sampling (model/sampling.py) end in different places of one row, against the plain 64-bit form,
token for token."""
from __future__ import annotations

import pytest
import torch

from batch_cases import FLOATS, sample_exact
from nurostream_amd.model.sampling import sample

pytestmark = pytest.mark.gpu


def _gen(dev, seed):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return g


def _check(logits, u, T, top_k, top_p, min_p):
    B = logits.shape[0]
    row = lambda x: x.tolist() if isinstance(x, torch.Tensor) else [x] * B  # noqa: E731
    got = sample(logits, u, temperature=T, top_k=top_k, top_p=top_p, min_p=min_p)
    want = sample_exact(logits, row(u), row(T), row(top_k), row(top_p), row(min_p))
    assert got.tolist() == want, [(r, g, w) for r, (g, w) in enumerate(zip(got.tolist(), want)) if g != w][:5]
    return got


@pytest.mark.parametrize("x", FLOATS)
@pytest.mark.parametrize("V,top_k,size", [(1200, 1100, 1.0), (4097, 1500, 1.0), (5600, 1025, 2.0), (9000, 3000, 2.0), (11000, 4900, 2.0),
                                          (32000, 1400, 1.0), (32000, 3200, 4.0), (50257, 1200, 3.0)])
def test_top_p_ends_ahead_of_a_large_top_k(dev, x, V, top_k, size):
    """A top-k past the tokens that a row lists whole, and a top-p that ends far ahead of it: few tokens are open between the
    ends or many, in a row of few workgroups (one launch to the token) and of many rows."""
    g = _gen(dev, V + top_k)
    for B in (5, max(8, 200000 // V)):  # (more than 160 workgroups of 4096 logits)
        B = min(B, 90)
        logits = (size * torch.randn(B, V, generator=g, device=dev)).to(x)
        u = torch.rand(B, generator=g, device=dev)
        for top_p, min_p in ((0.5, 0.0), (0.6, 0.02), (0.9, 0.0), (0.95, 0.001)):
            _check(logits, u, 0.8, top_k, top_p, min_p)


@pytest.mark.parametrize("V,top_k,top_p", [(5894, 3269, 0.6), (4097, 1500, 0.5), (9000, 3000, 0.7)])
def test_the_tokens_kept_by_both(dev, V, top_k, top_p):
    """Every draw of a row: nothing from behind top-p's end."""
    g = _gen(dev, V)
    n = 90
    logits = (2 * torch.randn(1, V, generator=g, device=dev)).expand(n, V).contiguous()
    _check(logits, (torch.arange(n, device=dev) + 0.5) / n, 0.8, top_k, top_p, 0.0)


@pytest.mark.parametrize("x", FLOATS)
@pytest.mark.parametrize("B,V", [(6, 20011), (60, 12007)])
def test_rows_of_large_top_k_of_their_own(dev, x, B, V):
    g = _gen(dev, B)
    r = lambda: torch.rand(B, generator=g, device=dev)  # noqa: E731
    logits = ((0.5 + 3 * r())[:, None] * torch.randn(B, V, generator=g, device=dev)).to(x)
    T, k = 0.3 + r(), (900 + r() * 6000).floor().to(torch.int32)
    p, m = 0.4 + 0.65 * r(), torch.where(r() < 0.5, 0.0, 0.1 * r() ** 3)
    _check(logits, r(), T, k, p, m)


@pytest.mark.parametrize("kw", [dict(top_k=3000, top_p=0.7), dict(top_k=1100, top_p=0.95, min_p=0.003)])
def test_a_row_alone_and_the_definition(dev, kw):
    """A row's token does not depend on the batch that it is in, and is the definition's."""
    g = _gen(dev, 15)
    logits = 2 * torch.randn(130, 9000, generator=g, device=dev)
    u = torch.rand(130, generator=g, device=dev)
    want = sample(logits, u, temperature=0.9, **kw)
    for rows in (slice(0, 1), slice(77, 78), slice(100, 130)):
        got = _check(logits[rows], u[rows].clone(), 0.9, kw["top_k"], kw["top_p"], kw.get("min_p", 0.0))
        assert torch.equal(got, want[rows])
