"""What a token sees takes part in its attention (model/batch.py), however its keys are shared out over workgroups: an infinity
or a NaN in a row that is seen shows, whatever weight the row has beside others and beside the sink."""
from __future__ import annotations

import math

import pytest
import torch

from batch_cases import FLOATS, ROWS, attn_exact, rounding
from nurostream_amd.model.batch import BatchKV, batch_attn, store_rows
from test_gpu_batch import _cfg, _close, _fill, _gen, _held

pytestmark = pytest.mark.gpu


def _batch(dev, t, P, pos, n=1, d=64, rows=60, seed=0):
    """A prefix of P rows and sequences of pos rows and n more behind it, 8 heads over 2."""
    normal = _gen(dev, 100 + seed + P)
    cfg = _cfg(8, 2, d)
    prefix = BatchKV(1, cfg, 1, P, dev, dtype=t)
    _fill(prefix, normal, [P])
    prefix.pos.fill_(P)
    kv = BatchKV(1, cfg, len(pos), rows, dev, dtype=t, prefix=prefix)
    _fill(kv, normal, [p + n for p in pos])
    kv.pos.copy_(torch.tensor(pos, dtype=torch.int32))
    return normal, cfg, prefix, kv


def _exact(q, kv, prefix, pos, P, sinks, window=0):
    return attn_exact(q, *(y[0].nan_to_num(0.0) for y in _held(prefix)), *(y.nan_to_num(0.0) for y in _held(kv)), pos, P, None, sinks,
                      window, 1 / math.sqrt(q.shape[-1]))


@pytest.mark.parametrize("x", FLOATS)
@pytest.mark.parametrize("t", ROWS)
@pytest.mark.parametrize("P", [100, 2000, 9000])
@pytest.mark.parametrize("sinks", [False, True])
def test_the_only_own_key(dev, x, t, P, sinks):
    """A NaN in the one key of a sequence's own, which a workgroup of its own takes where the prefix is long; the other
    sequence stays as it is."""
    normal, cfg, prefix, kv = _batch(dev, t, P, [0, 0])
    q = normal(2, 1, 8, 64).to(x)
    s = normal(8) if sinks else None
    want, room = _exact(q, kv, prefix, [0, 0], P, s)
    _close(batch_attn(q, cfg, kv, 0, s, 0), want, room + rounding(want, x))
    rows = normal(2, 2, 1, 64)
    rows[0] = math.nan
    store_rows(rows, rows, kv, 0, 0)
    want, room = _exact(q, kv, prefix, [0, 0], P, s)
    got = batch_attn(q, cfg, kv, 0, s, 0)
    assert torch.isnan(got[0]).all()
    _close(got[1], want[1], room[1] + rounding(want[1], x))


@pytest.mark.parametrize("x", FLOATS)
@pytest.mark.parametrize("t", ROWS)
@pytest.mark.parametrize("P", [100, 2000, 9000])
@pytest.mark.parametrize("bad", ["key", "value"])
def test_keys_of_no_weight(dev, x, t, P, bad):
    """A NaN in a prefix row beside which an own key has e^500 of the weight: weight times value is still no number."""
    normal, cfg, prefix, kv = _batch(dev, t, P, [0, 0], seed=1)
    q = torch.zeros(2, 1, 8, 64, device=dev)
    q[..., 5] = 16.0
    heavy = torch.zeros(2, 2, 1, 64, device=dev)
    heavy[..., 5] = 256.0  # a score of 16 * 256 / 8
    light = torch.zeros(1, 2, P, 64, device=dev)
    light[..., 6:] = normal(1, 2, P, 58)
    values = normal(1, 2, P, 64)
    store_rows(light, values, prefix, 0)
    store_rows(heavy, normal(2, 2, 1, 64), kv, 0)
    q = q.to(x)
    want, room = _exact(q, kv, prefix, [0, 0], P, None)
    _close(batch_attn(q, cfg, kv, 0, None, 0), want, room + rounding(want, x))
    for row in (0, P // 2, P - 1):
        k, v = light.clone(), values.clone()
        (k if bad == "key" else v)[:, :, row] = math.nan
        store_rows(k, v, prefix, 0)
        assert torch.isnan(batch_attn(q, cfg, kv, 0, None, 0)).all(), row


@pytest.mark.parametrize("x", FLOATS)
@pytest.mark.parametrize("t", ROWS)
@pytest.mark.parametrize("P", [100, 2000])
@pytest.mark.parametrize("bad", ["key", "value"])
def test_beside_a_heavy_sink(dev, x, t, P, bad):
    """The same beside a sink of e^1000 of every key's weight; a token that its sequence does not have is still zero."""
    normal, cfg, prefix, kv = _batch(dev, t, P, [0, 3], seed=2)
    q, s = normal(2, 1, 8, 64).to(x), torch.full((8,), 1000.0, device=dev)
    assert not batch_attn(q, cfg, kv, 0, s, 0).any()
    k, v = normal(1, 2, P, 64), normal(1, 2, P, 64)
    (k if bad == "key" else v)[:, :, P - 2] = math.nan
    store_rows(k, v, prefix, 0)
    assert torch.isnan(batch_attn(q, cfg, kv, 0, s, 0)).all()
    counts = torch.tensor([0, 1], dtype=torch.int32, device=dev)
    got = batch_attn(q, cfg, kv, 0, s, 0, counts=counts, out=torch.full_like(q, math.nan))
    assert not got[0].any() and torch.isnan(got[1]).all()
    # and by a window that the row lies before
    assert not batch_attn(q, cfg, kv, 0, s, 1, out=torch.full_like(q, math.nan)).any()
