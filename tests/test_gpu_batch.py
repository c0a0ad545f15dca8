"""Several sequences at once (model/batch.py) against plain 64-bit forms: rows into the cache and back, norms and rotation,
attention over a shared prefix and own rows."""
from __future__ import annotations

import math

import pytest
import torch

from batch_cases import FLOATS, LARGEST, ROWS, append_exact, attn_exact, row_error, rounding, values
from nurostream_amd.model.batch import BatchKV, append_qkv, batch_attn, load_rows, store_rows
from nurostream_amd.model.decode import AttnConfig, DeviceKV, yarn_inv_freq

pytestmark = pytest.mark.gpu


def _cfg(n_head=16, n_kv=2, d=64):
    return AttnConfig(n_head=n_head, n_head_kv=n_kv, head_dim=d, vocab_size=10, rope_base=150000.0, context_length=131072)


def _gen(dev, seed):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return lambda *shape: torch.randn(*shape, generator=g, device=dev)


def _poison(kv: BatchKV) -> None:
    """NaN in every row: what a kernel reads past a sequence's rows shows."""
    for t in (kv.k_stack, kv.v_stack):
        if t.dtype == torch.int8:
            t.fill_(55)
        elif t.dtype == torch.bfloat16:
            t.fill_(math.nan)
        else:
            t.view(torch.uint8).fill_(0x7f)
    for t in (kv.k_scale, kv.v_scale):
        if t is not None:
            t.fill_(math.nan)


def _held(kv: BatchKV, layer=0):
    k = values(kv.k_stack[layer], None if kv.k_scale is None else kv.k_scale[layer])
    v = values(kv.v_stack[layer], None if kv.v_scale is None else kv.v_scale[layer])
    return k, v


def _close(got, want, room, what=""):
    got = got.double()
    bad = ~((got - want).abs() <= room)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, by up to " \
        f"{float(((got - want).abs() / room.clamp(min=1e-300)).nan_to_num(1e9).max()):.3g} of what is allowed"


# -- rows ---------------------------------------------------------------------


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("t", ROWS)
@pytest.mark.parametrize("x", FLOATS)
@pytest.mark.parametrize("n_seq,n_kv,n,start", [(1, 1, 1, 0), (3, 2, 37, 5), (2, 3, 129, 1)])
def test_rows_and_back(dev, x, t, d, n_seq, n_kv, n, start):
    normal = _gen(dev, 1 + n)
    kv = BatchKV(2, _cfg(n_kv, n_kv, d), n_seq, start + n + 3, dev, dtype=t)
    _poison(kv)
    before = [s.view(torch.uint8).clone() if s.dtype != torch.float32 else s.view(torch.int32).clone()
              for s in (kv.k_stack, kv.v_stack) + ((kv.k_scale, kv.v_scale) if kv.k_scale is not None else ())]
    k, v = ((normal(n_seq, n_kv, n, d) * 3).to(x) for _ in "kv")
    store_rows(k, v, kv, 1, start)
    for got, want in zip(load_rows(kv, 1, start, n), (k, v)):
        assert got.dtype == torch.float32
        _close(got, want.double(), row_error(want.double(), t), f"{x} into {t}")
    # as the codes have it, to the bit where the type takes the value (8 bits times a scale: rounded once)
    for y in FLOATS:
        for got, held in zip(load_rows(kv, 1, start, n, dtype=y), _held(kv, 1)):
            held = held[:, :, start:start + n]
            assert torch.equal(got, held.float().to(y)), y
    # nothing else was written: other layers, rows before and behind
    for s, old in zip((kv.k_stack, kv.v_stack, kv.k_scale, kv.v_scale), before):
        new = s.view(old.dtype)
        assert torch.equal(new[0], old[0]) and torch.equal(new[1, :, :, :start], old[1, :, :, :start])
        assert torch.equal(new[1, :, :, start + n:], old[1, :, :, start + n:])


@pytest.mark.parametrize("t", ROWS)
def test_rows_from_the_device(dev, t):
    """First rows of each sequence's own; what lies outside the cache is not written, and reads as zeros."""
    normal = _gen(dev, 3)
    cfg = _cfg(2, 2, 64)
    kv = BatchKV(1, cfg, 5, 20, dev, dtype=t)
    start = torch.tensor([0, -2, 17, 30, -2 ** 31], dtype=torch.int32, device=dev)
    k, v = normal(5, 2, 6, 64), normal(5, 2, 6, 64)
    store_rows(k, v, kv, 0, start)
    got = load_rows(kv, 0, start, 6)
    for b, s in enumerate(start.tolist()):
        for j in range(6):
            for g, x in zip(got, (k, v)):
                if 0 <= s + j < 20:
                    _close(g[b, :, j], x[b, :, j].double(), row_error(x[b, :, j].double(), t))
                else:
                    assert not g[b, :, j].any()
    held = _held(kv)[0]
    assert not held[3].any() and not held[4].any() and not held[0, :, 6:].any() and not held[1, :, 4:].any()
    with pytest.raises(ValueError):
        load_rows(kv, 0, 15, 6)


@pytest.mark.parametrize("t", (torch.int8, torch.float8_e4m3fn))
def test_quantised_edges(dev, t):
    """Rows of zeros, of one element, with infinities or NaN, very large and very small ones, values between two codes."""
    d, tiny = 64, 2.0 ** -149
    rows = torch.zeros(12, d, device=dev)
    rows[1, 5] = -3.0
    rows[2, 7] = math.inf
    rows[3, 9] = math.nan
    rows[4] = 3.4e38
    rows[5, ::2] = -3.4e38
    rows[6, 3] = tiny
    rows[7] = torch.linspace(-200, 200, d, device=dev) * tiny * 1000
    rows[8] = (torch.arange(d, device=dev) - 31.5)  # halves beside a scale of one
    rows[8, 0] = LARGEST[t]
    rows[9] = -0.0
    rows[10] = torch.exp2(torch.linspace(-20, 8, d, device=dev))
    rows[11, -1] = 1e-30
    kv = BatchKV(1, _cfg(1, 1, d), 1, 12, dev, dtype=t)
    store_rows(rows[None, None], rows[None, None].flip(2).contiguous(), kv, 0)
    k, v = load_rows(kv, 0, 0, 12)
    assert torch.equal(k.flip(2).view(torch.int32), v.view(torch.int32))
    k = k[0, 0]
    assert torch.isnan(k[2]).all() and torch.isnan(k[3]).all()
    fine = [i for i in range(12) if i not in (2, 3, 6, 7)]
    _close(k[fine], rows[fine].double(), row_error(rows[fine].double(), t))
    assert not k[0].any() and not k[9].any() and k[1, 5] == -3.0
    # scales below the normal numbers round to steps of 2^-149: off by one code's worth of the largest at most
    _close(k[6:8], rows[6:8].double(), rows[6:8].double().abs().amax(-1, keepdim=True) + tiny)
    # a tie goes to the even code
    if t == torch.int8:
        assert torch.equal(k[8, 1:], torch.round(rows[8, 1:].double()).float())
    else:
        assert torch.equal(k[8, 1:], rows[8, 1:].to(t).float())


# -- append -------------------------------------------------------------------


@pytest.mark.parametrize("x", FLOATS)
@pytest.mark.parametrize("t", ROWS)
@pytest.mark.parametrize("n_head,n_kv,d,n_seq,n,norm,bias,far", [
    (2, 2, 64, 1, 1, False, False, 0), (16, 2, 64, 3, 2, False, True, 1000), (12, 4, 128, 5, 1, True, False, 130000),
    (5, 1, 64, 2, 7, True, True, 70001), (64, 8, 64, 2, 300, False, True, 0), (24, 8, 128, 1, 600, True, True, 5)])
def test_append(dev, x, t, n_head, n_kv, d, n_seq, n, norm, bias, far):
    normal = _gen(dev, n + d)
    cfg = _cfg(n_head, n_kv, d)
    H, G = n_head, n_kv
    prefix = None
    if far:
        prefix = BatchKV(1, cfg, 1, 4, dev, dtype=t)
        prefix.pos.fill_(far)  # (the kernels take the position, not the rows)
    kv = BatchKV(1, cfg, n_seq, n + 11, dev, dtype=t, prefix=prefix)
    _poison(kv)
    lens = torch.arange(n_seq, dtype=torch.int32, device=dev) * 3 % 12
    kv.pos.copy_(lens)
    counts = torch.tensor([max(0, n - 2 * b) for b in range(n_seq)], dtype=torch.int32, device=dev) if n_seq > 1 else None
    qkv = (normal(n_seq, n, (H + 2 * G) * d) * 2).to(x)
    bq, bk, bv = ((normal(h * d) if bias else None) for h in (H, G, G))
    wq, wk = (1 + 0.3 * normal(d), 1 + 0.3 * normal(d)) if norm else (None, None)
    inv, amp = yarn_inv_freq(cfg, dev)
    out = torch.full((n_seq, n, H, d), math.nan, dtype=x, device=dev)
    q = append_qkv(qkv, bq, bk, bv, cfg, inv, amp, kv, 0, counts=counts, q_norm=wq, k_norm=wk, eps=1e-5, out=out)
    assert q is out
    at = far + lens[:, None].double() + torch.arange(n, device=dev)
    eq, ek, ev, rq, rk = append_exact(qkv, bq, bk, bv, wq, wk, 1e-5, inv, amp, at, H, G, d)
    c = [n] * n_seq if counts is None else counts.tolist()
    got = load_rows(kv, 0, kv.pos, n)
    for b in range(n_seq):
        _close(q[b, :c[b]], eq[b, :c[b]], rq[b, :c[b]] + rounding(eq[b, :c[b]], x), "queries")
        assert not q[b, c[b]:].any()
        # (a row's fp32 error, of its largest element's size, moves its scale and its codes beside the rounding)
        for name, g, e, r in (("keys", got[0][b], ek[b], rk[b]), ("values", got[1][b], ev[b], ev[b].abs() * 2.0 ** -23)):
            e, r = e.transpose(0, 1)[:, :c[b]], r.transpose(0, 1)[:, :c[b]]
            _close(g[:, :c[b]], e, row_error(e, t) * (1 + 2.0 ** -10) + 2 * r.amax(-1, keepdim=True), name) if c[b] else None
        # rows outside lens .. lens + c - 1 keep what they held
        k, v = _held(kv)
        for rows in (k[b], v[b]):
            free = torch.ones(n + 11, dtype=torch.bool, device=dev)
            free[lens[b]:lens[b] + c[b]] = False
            assert torch.isnan(rows[:, free]).all()
    assert torch.equal(kv.pos, lens)


def test_append_past_the_end(dev):
    """Rows past the cache by the device's length are not written, and lengths below zero leave nothing."""
    cfg = _cfg(4, 2, 64)
    kv = BatchKV(1, cfg, 4, 10, dev)
    normal = _gen(dev, 5)
    kv.pos.copy_(torch.tensor([8, 10, -1, 2 ** 31 - 1], dtype=torch.int32))
    qkv = normal(4, 3, 8 * 64)
    inv, amp = yarn_inv_freq(cfg, dev)
    append_qkv(qkv, None, None, None, cfg, inv, amp, kv, 0)
    held = _held(kv)[1]
    v = qkv.reshape(4, 3, 8, 64)[:, :, 6:].transpose(1, 2)
    assert torch.equal(held[0, :, 8:], v[0, :, :2].to(torch.bfloat16).double()) and not held[0, :, :8].any()
    assert not held[1].any() and not held[3].any()
    assert torch.equal(held[2, :, :2], v[2, :, 1:].to(torch.bfloat16).double()) and not held[2, :, 2:].any()


# -- attention ----------------------------------------------------------------


def _fill(kv: BatchKV, normal, rows, layer=0):
    """Random rows 0 .. rows[b] - 1 in sequence b, NaN behind them."""
    _poison(kv)
    G, d = kv.heads
    for b, n in enumerate(rows):
        if n:
            one = BatchKV(1, _cfg(G, G, d), 1, n, kv.device, dtype=kv.dtype)
            store_rows(normal(1, G, n, d) * 1.5, normal(1, G, n, d), one, 0)
            for name in ("k_stack", "v_stack", "k_scale", "v_scale"):
                if getattr(kv, name) is not None:
                    getattr(kv, name)[layer, b, :, :n] = getattr(one, name)[0, 0]


def _attention(dev, x, t, n_head, n_kv, d, P, pos, n, counts, window, sinks=True, seed=0, extra=3, size=1.0):
    normal = _gen(dev, seed + 7 * n + (P or 0))
    cfg = _cfg(n_head, n_kv, d)
    B = len(pos)
    prefix = None
    if P is not None:
        prefix = BatchKV(1, cfg, 1, P + extra, dev, dtype=t)
        _fill(prefix, normal, [P])
        prefix.pos.fill_(P)
    c = [n] * B if counts is None else counts
    kv = BatchKV(1, cfg, B, max(p + n for p in pos) + extra, dev, dtype=t, prefix=prefix)
    _fill(kv, normal, [p + k for p, k in zip(pos, c)])
    kv.pos.copy_(torch.tensor(pos, dtype=torch.int32))
    q = (normal(B, n, n_head, d) * size).to(x)
    s = normal(n_head) if sinks else None
    cn = None if counts is None else torch.tensor(counts, dtype=torch.int32, device=dev)
    out = torch.full_like(q, math.nan)
    got = batch_attn(q, cfg, kv, 0, s, window, counts=cn, out=out)
    assert got is out
    k, v = _held(kv)
    pk, pv = (None, None) if prefix is None else (y[0] for y in _held(prefix))
    want, room = attn_exact(q, pk, pv, k, v, pos, P or 0, counts, s, window, 1 / math.sqrt(d))
    _close(got, want, room + rounding(want, x), f"{x} over {t}")
    return q, cfg, kv, s, cn, got


@pytest.mark.parametrize("x", FLOATS)
@pytest.mark.parametrize("t", ROWS)
@pytest.mark.parametrize("n_head,n_kv,d,P,pos,n,counts,window", [
    (1, 1, 64, None, [0], 1, None, 0),                                  # one key
    (8, 1, 64, 0, [3, 0], 1, None, 0),                                  # an empty prefix
    (16, 2, 64, 1, [0, 1, 2], 1, None, 0),
    (16, 2, 128, 77, [0, 31, 32, 33, 95], 1, None, 0),                  # around tiles
    (24, 8, 64, 200, [17, 130], 1, [1, 0], 0),                          # three heads each, a sequence that is done
    (6, 2, 128, 1000, [5, 700, 64], 1, None, 128),                      # the window inside the prefix, at its edge, past it
    (5, 1, 64, 333, [0, 3], 9, [9, 4], 0),                              # several tokens, ragged
    (32, 4, 64, 64, [0, 100], 40, [40, 33], 33),                        # a window below a step's tokens
    (16, 16, 64, 129, [1, 2], 1, None, 1),                              # a window of one: itself
    (32, 2, 128, 511, [63], 70, None, 0),
    (64, 4, 64, None, [400, 12, 0], 3, [3, 2, 0], 0),                   # no prefix, sixteen heads each
    (40, 2, 64, 2100, [0] * 20, 1, None, 0)])                           # twenty heads each, many rows behind a prefix
def test_attention(dev, x, t, n_head, n_kv, d, P, pos, n, counts, window):
    _attention(dev, x, t, n_head, n_kv, d, P, pos, n, counts, window)


@pytest.mark.parametrize("x,t,n_head,n_kv,d,P,pos,n", [
    (torch.float32, torch.int8, 64, 8, 64, 6000, [300, 0, 7, 120, 299, 33, 64, 65], 1),
    (torch.bfloat16, torch.float8_e4m3fn, 64, 8, 64, 9001, [3] * 40, 1),
    (torch.bfloat16, torch.bfloat16, 32, 4, 128, 700, [18, 0], 300),
    (torch.float16, torch.int8, 16, 2, 128, 30, [5000, 4100], 2),
    (torch.float32, torch.bfloat16, 16, 8, 64, None, [0], 500)])
def test_attention_at_length(dev, x, t, n_head, n_kv, d, P, pos, n):
    for window in (0, 128):
        _attention(dev, x, t, n_head, n_kv, d, P, pos, n, None, window)


@pytest.mark.parametrize("x", FLOATS)
@pytest.mark.parametrize("t", ROWS)
def test_attention_wide_scores(dev, x, t):
    """Scores of some hundreds: nearly all weight on a few keys, others far below; and no sinks."""
    _attention(dev, x, t, 8, 2, 64, 300, [40, 3], 1, None, 0, sinks=False, size=30.0)


@pytest.mark.parametrize("t", ROWS)
def test_attention_light_keys(dev, t):
    """A heavy key whose value is zero leaves the light ones their bits."""
    cfg = _cfg(2, 1, 64)
    kv = BatchKV(1, cfg, 1, 400, dev, dtype=t)
    normal = _gen(dev, 9)
    k, v = normal(1, 1, 400, 64) * 0.01, normal(1, 1, 400, 64)
    q = torch.zeros(1, 1, 2, 64, device=dev)
    q[..., 0] = 8.0
    k[..., 0] = 0.25
    k[0, 0, 100, 0], v[0, 0, 100] = 40.0, 0.0  # e^40 of the others' weight
    store_rows(k, v, kv, 0)
    kv.pos.fill_(399)
    got = batch_attn(q, cfg, kv, 0, None, 0)
    kk, vv = _held(kv)
    want, room = attn_exact(q, None, None, kk, vv, [399], 0, None, None, 0, 0.125)
    assert float(want.abs().max()) < 1e-14
    _close(got, want, room + want.abs() * 2.0 ** -22)


@pytest.mark.parametrize("x", FLOATS)
@pytest.mark.parametrize("t", ROWS)
@pytest.mark.parametrize("n", [1, 6, 40])
def test_attention_masked_infinities(dev, x, t, n):
    """Infinities and NaN in rows that a token does not see leave it as it is; where it sees them they show."""
    normal = _gen(dev, 11)
    cfg = _cfg(8, 2, 64)
    prefix = BatchKV(1, cfg, 1, 100, dev, dtype=t)
    _fill(prefix, normal, [100])
    prefix.pos.fill_(100)
    kv = BatchKV(1, cfg, 2, 60, dev, dtype=t, prefix=prefix)
    _fill(kv, normal, [10 + n, 4 + n])
    kv.pos.copy_(torch.tensor([10, 4], dtype=torch.int32))
    q = normal(2, n, 8, 64).to(x)
    window = 30
    # the first token sees prefix rows 100 + 10 + 1 - 30 = 81 and on (sequence 0), 75 and on (sequence 1)
    bad = torch.full((1, 2, 1, 64), math.nan, device=dev)
    store_rows(bad, bad, prefix, 0, 74)
    want, room = attn_exact(q, *(y[0].nan_to_num(0.0) for y in _held(prefix)), *(y.nan_to_num(0.0) for y in _held(kv)), [10, 4], 100, None,
                            None, window, 0.125)
    got = batch_attn(q, cfg, kv, 0, None, window)
    _close(got, want, room + rounding(want, x))
    if n > 1:  # the last token's own row: only that token sees it
        both = bad.expand(2, 2, 1, 64).contiguous()
        store_rows(both, both, kv, 0, torch.tensor([10 + n - 1, 4 + n - 1], dtype=torch.int32, device=dev))
        inf = batch_attn(q, cfg, kv, 0, None, window)
        _close(inf[:, :-1], want[:, :-1], (room + rounding(want, x))[:, :-1])
        assert torch.isnan(inf[:, -1]).all()


def test_attention_sees_nothing(dev):
    """Lengths of zero and below: no key is seen, and the answer is zero."""
    cfg = _cfg(4, 2, 64)
    kv = BatchKV(1, cfg, 2, 10, dev)
    _poison(kv)
    kv.pos.fill_(-1)
    q = torch.ones(2, 1, 4, 64, device=dev)
    for s in (None, torch.ones(4, device=dev)):
        assert not batch_attn(q, cfg, kv, 0, s, 0, out=torch.full_like(q, math.nan)).any()


def test_attention_same_bits_again(dev):
    """The same inputs give the same bits, whatever the workspace held."""
    q, cfg, kv, s, cn, first = _attention(dev, torch.float32, torch.int8, 64, 8, 64, 3000, [200, 10, 77], 1, None, 0)
    for _ in range(3):
        torch.full((1 << 22,), math.nan, device=dev)
        assert torch.equal(batch_attn(q, cfg, kv, 0, s, 0, counts=cn), first)


def test_views_and_streams(dev):
    """Queries of another shape with as many elements, tensors used on a stream of their own."""
    q, cfg, kv, s, cn, first = _attention(dev, torch.bfloat16, torch.bfloat16, 16, 2, 64, 500, [20, 10], 1, None, 0)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        again = batch_attn(q.reshape(2, -1), cfg, kv, 0, s, 0)
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(again, first)
    with pytest.raises(ValueError):
        batch_attn(torch.cat([q, q], 1)[:, ::2], cfg, kv, 0, s, 0)


# -- the two together -----------------------------------------------------------


def _pass(kv, cfg, qkv, inv, amp, sinks, counts=None, window=0):
    q = append_qkv(qkv, None, None, None, cfg, inv, amp, kv, 0, counts=counts)
    return batch_attn(q, cfg, kv, 0, sinks, window, counts=counts)


@pytest.mark.parametrize("t", ROWS)
def test_prompt_in_pieces_or_at_once(dev, t):
    """A prompt's rows are the same however it is cut, and its tokens' attention to rounding; a batch behind it sees them."""
    cfg, normal = _cfg(16, 2, 64), _gen(dev, 21)
    inv, amp = yarn_inv_freq(cfg, dev)
    qkv, sinks = normal(1, 90, 20 * 64), normal(16)
    whole = BatchKV(1, cfg, 1, 90, dev, dtype=t)
    a = _pass(whole, cfg, qkv, inv, amp, sinks)
    whole.advance(90)
    cut, outs, at = BatchKV(1, cfg, 1, 90, dev, dtype=t), [], 0
    for n in (1, 40, 3, 46):
        outs.append(_pass(cut, cfg, qkv[:, at:at + n].contiguous(), inv, amp, sinks))
        cut.advance(n)
        at += n
    for x, y in zip(load_rows(whole, 0, 0, 90), load_rows(cut, 0, 0, 90)):
        assert torch.equal(x, y)
    # (the same products in other orders; both are within the tolerance of the 64-bit form)
    assert float((torch.cat(outs, 1) - a).abs().max()) <= 2.0 ** -16 * float(a.abs().max())
    # a token behind the prompt: as its 91st, and as the first of a batch that shares it
    more = normal(1, 1, 20 * 64)
    tall = BatchKV(1, cfg, 1, 91, dev, dtype=t)
    tall.copy_from(whole)
    one = _pass(tall, cfg, more, inv, amp, sinks)
    kv = BatchKV(1, cfg, 3, 4, dev, dtype=t, prefix=whole)
    three = _pass(kv, cfg, more.expand(3, 1, -1).contiguous(), inv, amp, sinks)
    assert torch.equal(three[0], three[1]) and torch.equal(three[0], three[2])
    assert float((three[:1] - one).abs().max()) <= 2.0 ** -16 * float(one.abs().max())


@pytest.mark.parametrize("t", ROWS)
def test_steps_of_a_captured_batch(dev, t):
    """A step captured once serves every later one: lengths, prefix and counts are the device's."""
    cfg, normal = _cfg(16, 2, 64), _gen(dev, 31)
    inv, amp = yarn_inv_freq(cfg, dev)
    prefix = BatchKV(1, cfg, 1, 60, dev, dtype=t)
    _pass(prefix, cfg, normal(1, 50, 20 * 64), inv, amp, None)
    prefix.advance(50)
    eager, replayed = (BatchKV(1, cfg, 4, 12, dev, dtype=t, prefix=prefix) for _ in "ab")
    x, counts = torch.zeros(4, 1, 20 * 64, device=dev), torch.ones(4, dtype=torch.int32, device=dev)
    sinks = normal(16)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        _pass(replayed, cfg, x, inv, amp, sinks, counts)
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _pass(replayed, cfg, x, inv, amp, sinks, counts)
        replayed.advance(1, counts)
    replayed.reset()
    for step in range(6):
        rows = normal(4, 1, 20 * 64)
        c = torch.tensor([1, int(step % 2 == 0), int(step < 3), 1], dtype=torch.int32, device=dev)
        want = _pass(eager, cfg, rows, inv, amp, sinks, c)
        eager.advance(1, c)
        x.copy_(rows)
        counts.copy_(c)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(replayed.pos, eager.pos), step
    assert replayed.pos.tolist() == [6, 3, 3, 6]
    for a, b in zip(load_rows(eager, 0, 0, 12), load_rows(replayed, 0, 0, 12)):
        assert torch.equal(a[0], b[0]) and torch.equal(a[3], b[3])


@pytest.mark.parametrize("t", ROWS)
@pytest.mark.parametrize("dt", FLOATS)
def test_copies(dev, t, dt):
    """A DeviceKV's rows for every sequence of a batch, and a batch's rows in another batch and type."""
    cfg, normal = _cfg(8, 2, 64), _gen(dev, 41)
    kv = DeviceKV(3, cfg, 30, dev, dtype=dt)
    kv.k_stack.copy_(normal(3, 2, 30, 64))
    kv.v_stack.copy_(normal(3, 2, 30, 64))
    kv.pos.fill_(23)
    kv.length = 23
    b = BatchKV(3, cfg, 2, 25, dev, dtype=t)
    b.copy_from(kv)
    assert b.pos.tolist() == [23, 23] and b.length == 23
    for layer in range(3):
        for got, src in zip(load_rows(b, layer, 0, 23), (kv.k[layer], kv.v[layer])):
            want = src[None, :, :23].double().expand(2, -1, -1, -1)
            _close(got, want, row_error(want, t))
    c = BatchKV(3, cfg, 2, 40, dev, dtype=torch.bfloat16)
    c.copy_from(b)
    for x, y in zip(load_rows(c, 2, 0, 23), load_rows(b, 2, 0, 23)):
        assert torch.equal(x, y.to(torch.bfloat16).float())


def test_two_streams_at_once(dev):
    """Two batches behind one prefix, each a step at a time on a stream of its own, as one after the other."""
    cfg, normal = _cfg(32, 4, 128), _gen(dev, 51)
    inv, amp = yarn_inv_freq(cfg, dev)
    prefix = BatchKV(1, cfg, 1, 3000, dev, dtype=torch.float8_e4m3fn)
    _pass(prefix, cfg, normal(1, 2900, 40 * 128), inv, amp, None)
    prefix.advance(2900)
    sizes, steps = (5, 33), 8
    rows = [[normal(b, 1, 40 * 128) for _ in range(steps)] for b in sizes]
    sinks = normal(32)

    def make():
        return [BatchKV(1, cfg, b, steps, dev, dtype=torch.float8_e4m3fn, prefix=prefix) for b in sizes]

    want = [[], []]
    for i, kv in enumerate(make()):
        for x in rows[i]:
            want[i].append(_pass(kv, cfg, x, inv, amp, sinks))
            kv.advance()
    torch.cuda.synchronize()
    batches, streams, got = make(), [torch.cuda.Stream() for _ in sizes], [[], []]
    torch.cuda.synchronize()
    for step in range(steps):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(_pass(batches[i], cfg, rows[i][step], inv, amp, sinks))
                batches[i].advance()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("x,t,d,window", [(torch.float16, torch.bfloat16, 128, 0), (torch.bfloat16, torch.int8, 64, 20),
                                          (torch.float32, torch.float8_e4m3fn, 128, 37)])
def test_captured_steps_of_several_tokens(dev, x, t, d, window):
    """Ragged steps of several tokens, two graphs of two batches behind one prefix replayed in turn, eager work between."""
    cfg, normal = _cfg(24, 3, d), _gen(dev, 61 + window)
    inv, amp = yarn_inv_freq(cfg, dev)
    prefix = BatchKV(1, cfg, 1, 700, dev, dtype=t)
    _pass(prefix, cfg, normal(1, 650, 30 * d).to(x), inv, amp, None)
    prefix.advance(650)
    sides = []
    for B, n in ((3, 5), (2, 18)):
        eager, kept = (BatchKV(1, cfg, B, 6 * n, dev, dtype=t, prefix=prefix) for _ in "ab")
        rows, counts = torch.zeros(B, n, 30 * d, device=dev, dtype=x), torch.zeros(B, dtype=torch.int32, device=dev)
        _pass(kept, cfg, rows, inv, amp, None, counts, window)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _pass(kept, cfg, rows, inv, amp, None, counts, window)
            kept.advance(n, counts)
        kept.reset()
        sides.append((B, n, eager, kept, rows, counts, graph, out))
    for step in range(5):
        for B, n, eager, kept, rows, counts, graph, out in sides:
            fresh = normal(B, n, 30 * d).to(x)
            c = torch.tensor([(step * 3 + 2 * b) % (n + 1) for b in range(B)], dtype=torch.int32, device=dev)
            want = _pass(eager, cfg, fresh, inv, amp, None, c, window)
            eager.advance(n, c)
            rows.copy_(fresh)
            counts.copy_(c)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(kept.pos, eager.pos), (step, B)
            assert not any(want[b, int(c[b]):].any() for b in range(B))


@pytest.mark.parametrize("t", ROWS)
def test_far_rows(dev, t):
    """A cache of more than 2^31 elements: rows at its end, as those of a small one."""
    cfg, normal = _cfg(8, 2, 128), _gen(dev, 71)
    far, near = BatchKV(1, cfg, 3, 3_000_001, dev, dtype=t), BatchKV(1, cfg, 3, 101, dev, dtype=t)
    assert far.k_stack.numel() > 2 ** 31
    start = torch.tensor([0, 2, 1], dtype=torch.int32, device=dev)  # of 90 rows
    k, v, qkv = normal(3, 2, 90, 128), normal(3, 2, 90, 128), normal(3, 9, 12 * 128)
    inv = torch.zeros(64, device=dev)  # (positions differ)
    outs = []
    for kv in (far, near):
        first = start + (kv.ctx_max - 101)
        store_rows(k, v, kv, 0, first)
        kv.pos.copy_(first + 90)
        q = append_qkv(qkv, None, None, None, cfg, inv, 1.0, kv, 0)
        outs.append((q, batch_attn(q, cfg, kv, 0, None, 60), *load_rows(kv, 0, kv.pos - 90, 99)))
    for a, b in zip(outs[0][2:], outs[1][2:]):
        assert torch.equal(a, b)
    assert torch.equal(outs[0][0], outs[1][0])
    held = _held(near)
    want, room = attn_exact(outs[1][0], None, None, *held, near.pos.tolist(), 0, None, None, 60, 1 / math.sqrt(128))
    for q, out, *_ in outs:
        _close(out, want, room + rounding(want, out.dtype))


def test_empty_copies(dev):
    """Nothing copied: lengths of zero."""
    cfg = _cfg(8, 2, 64)
    b = BatchKV(2, cfg, 2, 25, dev, dtype=torch.int8)
    b.advance(3)
    b.copy_from(DeviceKV(2, cfg, 30, dev, dtype=torch.float16))
    assert b.pos.tolist() == [0, 0] and b.length == 0
    assert all(t.shape == (2, 2, 0, 64) for t in load_rows(b, 0, 5, 0))


@pytest.mark.parametrize("x,t,n_head,n_kv,d,P,pos,n,counts,window", [
    (torch.bfloat16, torch.bfloat16, 32, 4, 128, 1900, [10, 0, 300], 300, [300, 17, 0], 0),
    (torch.bfloat16, torch.int8, 32, 4, 64, 2000, [5, 40, 0, 77], 260, [131, 260, 133, 1], 0),
    (torch.float32, torch.float8_e4m3fn, 32, 4, 64, 1500, [0, 9, 2], 301, [299, 150, 200], 0),
    (torch.float16, torch.bfloat16, 32, 4, 128, 1900, [0, 1, 2], 290, [0, 0, 290], 0),
    (torch.bfloat16, torch.bfloat16, 24, 8, 128, 1500, [0] * 5, 250, [250, 200, 100, 60, 249], 700),
    (torch.bfloat16, torch.bfloat16, 8, 1, 64, None, [100] * 70, 120, [(7 * i) % 121 for i in range(70)], 0),
    (torch.bfloat16, torch.bfloat16, 32, 4, 64, 1900, [3, 4], 400, [-3, 500], 0)])
def test_attention_ragged_prompts(dev, x, t, n_head, n_kv, d, P, pos, n, counts, window):
    """Many tokens of sequences of very different numbers of them."""
    given, counts = counts, [min(max(c, 0), n) for c in counts]
    q, cfg, kv, s, cn, got = _attention(dev, x, t, n_head, n_kv, d, P, pos, n, counts, window)
    if given != counts:  # (counts below 0 and above n count as those)
        cn = torch.tensor(given, dtype=torch.int32, device=dev)
        assert torch.equal(batch_attn(q, cfg, kv, 0, s, window, counts=cn, out=torch.full_like(q, math.nan)), got)
