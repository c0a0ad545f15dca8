"""The codes of rows of 8 bits (model/batch.py) are those of a division by the row's scale: fp32's nearest quotient, rounded to
the nearest code, between two to the even one."""
from __future__ import annotations

import pytest
import torch

from batch_cases import FLOATS, LARGEST
from nurostream_amd.model.batch import BatchKV, append_qkv, store_rows
from nurostream_amd.model.decode import yarn_inv_freq
from test_gpu_batch import _cfg, _gen

pytestmark = pytest.mark.gpu

EIGHT = (torch.int8, torch.float8_e4m3fn)


def _codes(x, t):
    """(codes as the type's values, scales) of fp32 rows on the host, by IEEE division."""
    x = x.float().cpu()
    scale = x.abs().amax(-1) / LARGEST[t]
    y = x / torch.where(scale > 0, scale, 1.0)[..., None]
    return (y.round().clamp(-127, 127) if t == torch.int8 else y.clamp(-448, 448).to(t).float()), scale


def _equal(kv, b, rows, t, want_k, want_v):
    for stack, scales, want in ((kv.k_stack, kv.k_scale, want_k), (kv.v_stack, kv.v_scale, want_v)):
        codes, scale = _codes(want, t)
        assert torch.equal(scales[0, b, :, rows].cpu(), scale)
        got = stack[0, b, :, rows].float().cpu()
        assert torch.equal(got, codes), f"{int((got != codes).sum())} of {codes.numel()} codes"


@pytest.mark.parametrize("x", FLOATS)
@pytest.mark.parametrize("t", EIGHT)
@pytest.mark.parametrize("d,n", [(64, 5), (64, 9001), (128, 301)])
def test_codes_of_stored_rows(dev, x, t, d, n):
    """Random rows (of 16 bits, one in some 30 holds half of its largest element), rows of halves and quarters of their
    largest, and rows of sizes from the least to the largest."""
    normal = _gen(dev, n + d)
    kv = BatchKV(1, _cfg(2, 2, d), 2, n, dev, dtype=t)
    k, v = normal(2, 2, n, d), normal(2, 2, n, d)
    top = k.abs().amax(-1, keepdim=True)
    k[:, 0] = (torch.round(k[:, 0] / top[:, 0] * 254) / 254 * top[:, 0])  # halves of steps
    v[0] *= torch.exp2(torch.arange(n, device=dev) % 240 - 120.0)[:, None]
    k, v = k.to(x), v.to(x)
    fine = torch.isfinite(v).all(-1, keepdim=True)
    v = torch.where(fine, v, torch.ones_like(v))
    store_rows(k, v, kv, 0)
    for b in range(2):
        _equal(kv, b, slice(0, n), t, k[b], v[b])


@pytest.mark.parametrize("x", FLOATS)
@pytest.mark.parametrize("t", EIGHT)
def test_codes_of_appended_values(dev, x, t):
    cfg, normal = _cfg(4, 2, 64), _gen(dev, 2)
    kv = BatchKV(1, cfg, 3, 700, dev, dtype=t)
    qkv = normal(3, 700, 8, 64).to(x)
    inv, amp = yarn_inv_freq(cfg, dev)
    append_qkv(qkv.reshape(3, 700, -1), None, None, None, cfg, inv, amp, kv, 0)
    for b in range(3):
        codes, scale = _codes(qkv[b, :, 6:].transpose(0, 1), t)
        assert torch.equal(kv.v_scale[0, b].cpu(), scale)
        assert torch.equal(kv.v_stack[0, b].float().cpu(), codes)
