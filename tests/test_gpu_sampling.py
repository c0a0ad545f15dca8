"""Sampling (model/sampling.py) against a plain 64-bit form, decision for decision."""
from __future__ import annotations

import math

import pytest
import torch

from batch_cases import FLOATS, sample_exact
from nurostream_amd.model.draft import verify
from nurostream_amd.model.sampling import sample

pytestmark = pytest.mark.gpu


def _gen(dev, seed):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return g


def _check(logits, u, T=1.0, top_k=0, top_p=1.0, min_p=0.0):
    B = logits.shape[0]
    row = lambda x: x.tolist() if isinstance(x, torch.Tensor) else [x] * B  # noqa: E731
    got = sample(logits, u, temperature=T, top_k=top_k, top_p=top_p, min_p=min_p).tolist()
    want = sample_exact(logits, row(u), row(T), row(top_k), row(top_p), row(min_p))
    assert got == want, [(r, g, w) for r, (g, w) in enumerate(zip(got, want)) if g != w][:5]


@pytest.mark.parametrize("x", FLOATS)
@pytest.mark.parametrize("V", [1, 2, 63, 1000, 4097])
@pytest.mark.parametrize("T,top_k,top_p,min_p", [
    (1.0, 0, 1.0, 0.0), (0.7, 5, 1.0, 0.0), (1.3, 0, 0.9, 0.0), (0.8, 0, 1.0, 0.05), (0.9, 50, 0.8, 0.01), (0.0, 3, 0.5, 0.1),
    (2.5, 1, 0.1, 1.0), (1.0, 10 ** 6, 0.999, 0.0), (0.05, 2, 1.0, 0.0)])
def test_sample(dev, x, V, T, top_k, top_p, min_p):
    g = _gen(dev, V + top_k)
    logits = (3 * torch.randn(40, V, generator=g, device=dev)).to(x)
    u = torch.rand(40, generator=g, device=dev)
    u[:3] = torch.tensor([0.0, 1 - 2.0 ** -24, 0.5])
    _check(logits, u, T, top_k, top_p, min_p)


@pytest.mark.parametrize("x", FLOATS)
def test_settings_of_each_row(dev, x):
    g = _gen(dev, 5)
    B, V = 64, 777
    logits = (4 * torch.randn(B, V, generator=g, device=dev)).to(x)
    r = lambda: torch.rand(B, generator=g, device=dev)  # noqa: E731
    T = torch.where(r() < 0.2, 0.0, 0.2 + 2 * r())
    T[:2] = torch.tensor([-1.0, math.nan])
    k = (r() * 60 - 10).floor().to(torch.int32)
    p = 1.3 * r() - 0.1
    m = torch.where(r() < 0.5, 0.0, 1.2 * r() ** 3)
    _check(logits, r(), T, k, p, m)
    _check(logits, r(), 0.8, k, 0.9, m)
    p[3] = math.nan  # no number: no restriction
    m[4] = math.nan
    got = sample(logits, r(), temperature=1.0, top_p=p, min_p=m)
    assert bool(((got >= 0) & (got < V)).all())


@pytest.mark.parametrize("x", FLOATS)
def test_equal_logits(dev, x):
    """Borders that fall among equal logits: the lowest indices are kept."""
    g = _gen(dev, 6)
    V = 3001
    logits = torch.randint(0, 4, (60, V), generator=g, device=dev).to(x)
    logits[:5] = 1.5  # all equal
    logits[5, ::2] = -0.0
    logits[5, 1::2] = 0.0
    u = torch.rand(60, generator=g, device=dev)
    for top_k, top_p in ((7, 1.0), (1500, 1.0), (0, 0.3), (0, 0.77), (1000, 0.25), (2, 0.5)):
        _check(logits, u, 1.0, top_k, top_p)


def test_strange_logits(dev):
    """Infinities, NaN, rows without any weight, values far apart."""
    inf, nan = math.inf, math.nan
    rows = [[nan, nan, nan, nan], [-inf] * 4, [inf, 1.0, inf, nan], [nan, 2.0, -inf, 1.9], [1e38, -1e38, 3e38, 3e38],
            [-3e38, -3.4e38, -inf, nan], [5.0, 5.0, 5.0, 5.0], [0.0, -700.0, -800.0, -1e5], [inf, -inf, nan, inf]]
    logits = torch.tensor(rows, device=dev)
    for u in (0.0, 0.3, 0.6, 1 - 2.0 ** -24):
        for kw in (dict(), dict(top_k=1), dict(top_p=0.6), dict(min_p=0.3), dict(T=0.0)):
            _check(logits, torch.full((9,), u, device=dev), **kw)


def test_the_kept_tokens(dev):
    """Every draw of a row between two kept tokens' borders: the filters keep exactly the tokens that they should."""
    g = _gen(dev, 8)
    V, n = 50, 4000
    logits = (2 * torch.randn(1, V, generator=g, device=dev)).expand(n, V).contiguous()
    u = (torch.arange(n, device=dev) + 0.5) / n
    for kw in (dict(top_k=7), dict(top_p=0.85), dict(min_p=0.1), dict(top_k=20, top_p=0.9, min_p=0.02)):
        _check(logits, u, 1.0, **kw)


@pytest.mark.parametrize("x", FLOATS)
@pytest.mark.parametrize("B,V,kw", [(3, 201088, dict(top_k=50, top_p=0.95)), (2, 151936, dict(top_p=0.9, min_p=0.01)),
                                    (1, 32001, dict()), (5, 65537, dict(top_k=30000, top_p=0.6))])
def test_large_vocabularies(dev, x, B, V, kw):
    g = _gen(dev, V)
    logits = (2 * torch.randn(B, V, generator=g, device=dev)).to(x)
    for _ in range(3):
        _check(logits, torch.rand(B, generator=g, device=dev), 0.8, **kw)


@pytest.mark.parametrize("x", FLOATS)
def test_fewer_tokens_than_asked_for(dev, x):
    """Most tokens masked away: top-k finds fewer than it may keep, top-p fewer than its share needs."""
    g = _gen(dev, 14)
    logits = torch.full((30, 5000), -math.inf, device=dev)
    logits[:, ::617] = torch.randn(30, 9, generator=g, device=dev)
    logits[::3, 7] = -3000.0  # a weight of nothing
    u = torch.rand(30, generator=g, device=dev)
    for kw in (dict(top_k=20), dict(top_k=9), dict(top_k=3), dict(top_k=20, top_p=0.7), dict(top_k=2000, top_p=0.999), dict(top_p=0.4)):
        _check(logits.to(x), u, 0.7, **kw)


@pytest.mark.parametrize("top_k", [1023, 1024, 1025, 2049, 9000])
def test_top_k_among_many_equals(dev, top_k):
    """Borders of every way to hold the tokens of the last bin: in registers, in a list, or read again."""
    g = _gen(dev, top_k)
    for step in (1.0, 0.02, 1e-4):
        logits = torch.round(torch.randn(3, 20000, generator=g, device=dev) / step) * step
        _check(logits, torch.rand(3, generator=g, device=dev), 1.0, top_k, 0.9)
        _check(logits * 0.01, torch.rand(3, generator=g, device=dev), 1.0, top_k)


@pytest.mark.parametrize("V", [300000, 4194304])
def test_flat_row(dev, V):
    """All tokens of equal weight: whole counts tell the answer."""
    logits = torch.zeros(1, V, dtype=torch.bfloat16, device=dev)
    for u in (0.0, 0.25, 0.7):
        at = lambda keep: math.floor(float(torch.tensor(u)) * keep)  # noqa: E731
        ut = torch.tensor([u], device=dev)
        assert sample(logits, ut).item() == at(V)
        assert sample(logits, ut, top_k=V // 3).item() == at(V // 3)
        assert sample(logits, ut, top_p=0.5).item() == at(math.ceil(0.5 * V))
        assert sample(logits, ut, top_k=V // 3, top_p=0.5).item() == at(math.ceil(0.5 * (V // 3)))


def test_strides_and_padding(dev):
    """Rows of a padded vocabulary, odd offsets, another order of axes, many rows."""
    g = _gen(dev, 9)
    wide = torch.randn(300, 1037, generator=g, device=dev)
    wide[:, 1001:] = 50.0
    u = torch.rand(300, generator=g, device=dev)
    for view in (wide[:, :1001], wide[:, 1:1001], wide[::3, 3:900], wide[:, :1001].half(), wide.t()[:1001].t()):
        want = sample(view.contiguous(), u[:view.shape[0]].contiguous(), top_k=40, top_p=0.9)
        assert torch.equal(sample(view, u[:view.shape[0]].contiguous(), top_k=40, top_p=0.9), want)
        assert int(want.max()) < 1001
    turned = wide[:, :64].t().contiguous().t()
    assert torch.equal(sample(turned, u), sample(turned.contiguous(), u))
    assert sample(wide[:0], u[:0]).shape == (0,)


def test_greedy_needs_no_numbers(dev):
    logits = torch.randn(4, 5000, generator=_gen(dev, 10), device=dev)
    assert torch.equal(sample(logits, temperature=0.0).long(), logits.argmax(-1))
    with pytest.raises(ValueError):
        sample(logits)


def test_as_verification_draws(dev):
    """Without filters the token is the one that `verify` draws behind a sequence of one node."""
    g = _gen(dev, 11)
    logits = 2 * torch.randn(50, 1, 4000, generator=g, device=dev)
    u = torch.rand(50, 1, generator=g, device=dev)
    _, _, token = verify(logits, torch.zeros(50, 1, dtype=torch.int32, device=dev), u, temperature=0.9)
    assert torch.equal(sample(logits[:, 0], u[:, 0].contiguous(), temperature=0.9), token)


def test_captured(dev):
    """A captured call draws anew from what its inputs hold."""
    g = _gen(dev, 12)
    logits, u = torch.zeros(6, 3000, device=dev), torch.zeros(6, device=dev)
    p = torch.ones(6, device=dev)
    kw = dict(temperature=0.9, top_k=100, top_p=p, min_p=0.01)
    sample(logits, u, **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        token = sample(logits, u, **kw)
    for _ in range(5):
        logits.copy_(2 * torch.randn(6, 3000, generator=g, device=dev))
        u.copy_(torch.rand(6, generator=g, device=dev))
        p.copy_(torch.rand(6, generator=g, device=dev))
        want = sample(logits, u, **kw)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(token, want)


def test_extreme_temperatures_of_rows(dev):
    """Temperatures past both ends count as the ends: all tokens alike, or the largest logits alone."""
    g = _gen(dev, 13)
    logits = torch.randn(4, 5000, generator=g, device=dev)
    logits[:, 7] = -float("inf")
    logits[2, 100] = logits[2, 4000] = 9.0
    t = torch.tensor([float("inf"), 1e38, 1e-38, float("nan")], device=dev)
    u = torch.tensor([0.3, 0.75, 0.6, 0.5], device=dev)
    others = [i for i in range(5000) if i != 7]
    got = sample(logits, u, temperature=t).tolist()
    assert got == [others[int(float(u[0]) * 4999)], others[int(0.75 * 4999)], 4000, int(logits[3].argmax())]


def test_two_streams_at_once(dev):
    """Calls on two streams, each with scratch of its own, as one after the other."""
    g = _gen(dev, 14)
    kw = dict(temperature=0.8, top_k=300, top_p=0.9)
    sides = [(torch.randn(b, 50000, generator=g, device=dev), torch.rand(b, generator=g, device=dev)) for b in (1, 40)]
    want = [[sample(x + i, u, **kw) for i in range(6)] for x, u in sides]
    shifted = [[x + i for i in range(6)] for x, u in sides]
    streams, got = [torch.cuda.Stream() for _ in sides], [[], []]
    torch.cuda.synchronize()
    for i in range(6):
        for s, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[s].append(sample(shifted[s][i], sides[s][1], **kw))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("kw", [dict(top_p=0.9), dict(top_k=70), dict(top_k=3000, top_p=0.7), dict()])
def test_a_row_alone(dev, kw):
    """A row's token does not depend on the batch that it is in."""
    g = _gen(dev, 15)
    logits = 2 * torch.randn(130, 9000, generator=g, device=dev)
    u = torch.rand(130, generator=g, device=dev)
    want = sample(logits, u, temperature=0.9, **kw)
    for rows in (slice(0, 1), slice(77, 78), slice(100, 130)):
        assert torch.equal(sample(logits[rows], u[rows].clone(), temperature=0.9, **kw), want[rows])
