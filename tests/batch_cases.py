"""Plain 64-bit forms of the operators on several sequences, and how far a right kernel may be from them."""
from __future__ import annotations

import math

import torch

LARGEST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
ROWS = (torch.bfloat16, torch.int8, torch.float8_e4m3fn)
FLOATS = (torch.float32, torch.float16, torch.bfloat16)


def half_step(t: torch.dtype) -> float:
    return torch.finfo(t).eps / 2


def values(codes: torch.Tensor, scale: torch.Tensor | None) -> torch.Tensor:
    """What a cache's rows stand for, in 64 bits."""
    x = codes.float().double()
    return x if scale is None else x * scale.double()[..., None]


def row_error(x: torch.Tensor, t: torch.dtype) -> torch.Tensor:
    """How far a row's value may lie from the 64-bit row x: half a step of the type, and for 8 bits the scale's rounding
    (2^-23 of the value) and that of x / scale before it is rounded (2^-23 of x, below 2^-23 of the largest)."""
    if t == torch.bfloat16:
        return x.abs() * half_step(t) + 2.0 ** -134  # (half of bf16's least number)
    most = x.abs().amax(-1, keepdim=True)
    scale = most / LARGEST[t]
    step = scale / 2 if t == torch.int8 else torch.maximum(x.abs() * half_step(t), scale * 2.0 ** -10)
    return step + most * 2.0 ** -21


def append_exact(qkv, bq, bk, bv, wq, wk, eps, inv, amp, at, H, G, d):
    """(q, k, v, room) in 64 bits: heads (B, n, heads, d) and how far fp32 may be from the rotated ones beside rounding.
    at: (B, n) positions."""
    B, n = at.shape
    x = qkv.double().reshape(B, n, H + 2 * G, d)
    q, k, v = x[:, :, :H], x[:, :, H:H + G], x[:, :, H + G:]
    q, k, v = (y if b is None else y + b.double().reshape(-1, d) for y, b in ((q, bq), (k, bk), (v, bv)))

    def norm(y, w):
        return y if w is None else y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * w.double()

    angle = at.double()[..., None] * inv.double()
    cos, sin = torch.cos(angle)[:, :, None] * amp, torch.sin(angle)[:, :, None] * amp

    def turn(y):
        a, b = y[..., :d // 2], y[..., d // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    # Bias 2^-24; the norm's sum of d squares (d / 8 + 4 additions in a row) and its root, quotient and two products, below
    # (d / 8 + 16) 2^-24 / 2 + 4 2^-24 <= 20 2^-24; sine and cosine of a 32-bit angle below pi (2^-23 of it: 2^-22) with
    # their own 2 steps and the amplitude's, 2^-21; two products and a sum 2 2^-24. Together below 2^-18.6 of |a| + |b|.
    def room(y):
        a = y[..., :d // 2].abs() + y[..., d // 2:].abs()
        return torch.cat([a, a], -1) * amp * 2.0 ** -18

    q, k = norm(q, wq), norm(k, wk)
    return turn(q), turn(k), v, room(q), room(k)


def attn_exact(q, pk, pv, k, v, pos, P, counts, sinks, window, scale):
    """(out, room) in 64 bits. q (B, n, H, d); pk, pv (G, Pmax, d) or None; k, v (B, G, L, d) values; pos list; room: how far
    the kernel may be beside the rounding of its output."""
    B, n, H, d = q.shape
    G = k.shape[1]
    R = H // G
    out, room = torch.zeros(B, n, H, d, dtype=torch.float64, device=q.device), torch.zeros(B, n, H, d, dtype=torch.float64, device=q.device)
    # weights as `batch_attn` rounds them; every fp32 weight keeps 24 bits
    wbits = {torch.float32: 2.0 ** -23, torch.float16: 2.0 ** -16, torch.bfloat16: 2.0 ** -8}[q.dtype]
    for b in range(B):
        c = n if counts is None else counts[b]
        L = pos[b] + c
        if c < 1 or not P + L:
            continue
        kk, vv = k[b, :, :L], v[b, :, :L]
        if P:
            kk, vv = torch.cat([pk[:, :P], kk], 1), torch.cat([pv[:, :P], vv], 1)
        qq = q[b, :c].double().reshape(c, G, R, d).permute(1, 0, 2, 3).reshape(G, c * R, d)
        at = torch.arange(P + L, device=q.device)
        mine = (P + pos[b] + torch.arange(c, device=q.device)).repeat_interleave(R)[:, None]
        hidden = at > mine
        if window:
            hidden = hidden | (mine - at >= window)
        kt = kk.transpose(1, 2).contiguous()
        s = (qq @ kt * scale).masked_fill(hidden, -math.inf)
        # a score: d exact products summed in 32 bits in any order, its scales: (d + 4) 2^-24 of the sum of magnitudes
        off = ((qq.abs() @ kt.abs()) * scale).masked_fill(hidden, 0).amax(-1, keepdim=True) * (d + 4) * 2.0 ** -24
        sink = torch.full((G, c * R, 1), -math.inf, dtype=torch.float64, device=q.device)
        if sinks is not None:
            sink = sinks.double().reshape(G, 1, R).expand(G, c, R).reshape(G, c * R, 1)
        top = torch.maximum(s.amax(-1, keepdim=True), sink)
        w = torch.exp(s - top)
        z = w.sum(-1, keepdim=True) + torch.exp(sink - top)
        w = w / z
        o = torch.where(z > 0, w @ vv, 0.0)
        # a weight: its score's error in nats, the same of the largest, the exponent's rounding (its argument, a few hundred
        # at most: 2^-16 of it in 2^-24 steps of 2^8; 2^-15 for both), the exponential's and the rescalings' 8 2^-24, rounding
        # beside the queries' type; in the numerator and the denominator. Sums of P + L terms: 2^-24 each, at worst all one way.
        one = torch.expm1(2 * off) + 2.0 ** -20 + 2.0 ** -24 * (s.masked_fill(hidden, 0).abs().amax(-1, keepdim=True) * 1.5 * 2)
        rel = 2 * one + wbits + (P + L + 64) * 2.0 ** -24
        r = torch.where(z > 0, rel * (w @ vv.abs()), 0.0)
        back = lambda y: y.reshape(G, c, R, d).permute(1, 0, 2, 3).reshape(c, H, d)  # noqa: E731
        out[b, :c], room[b, :c] = back(o), back(r)
    return out, room


def rounding(want: torch.Tensor, t: torch.dtype) -> torch.Tensor:
    """Half a step of an output's type (fp16's below its normal numbers: 2^-25); fp32: the two operations that end a sum."""
    return want.abs() * (half_step(t) if t != torch.float32 else 2.0 ** -22) + (2.0 ** -25 if t == torch.float16 else 2.0 ** -30)


def sample_exact(logits, u, T, top_k, top_p, min_p) -> list[int]:
    """Row by row: weights in 64 bits, summed as whole multiples of 2^-min(51, 62 - ceil(log2 vocab)) of the
    largest."""
    got = []
    for r in range(logits.shape[0]):
        x = logits[r].double().cpu()
        x = torch.where(torch.isnan(x), -math.inf, x)
        V, top = x.numel(), float(x.max())
        if top == -math.inf:
            got.append(-1)
            continue
        if not T[r] > 0:
            got.append(int((x == top).nonzero()[0]))
            continue
        real = ((x == top).double() if top == math.inf else torch.exp((x - top) / T[r])).tolist()
        unit = 2.0 ** min(51, 62 - (V - 1).bit_length())
        w = [round(a * unit) for a in real]
        x = x.tolist()
        order = sorted(range(V), key=lambda i: (-x[i], i))
        kept = order[:top_k[r]] if 0 < top_k[r] < V else order
        if top_p[r] < 1:
            border, before, some = max(top_p[r], 0.0) * sum(w[i] for i in kept), 0, []
            for i in kept:
                if some and not before < border:
                    break
                some.append(i)
                before += w[i]
            kept = some
        kept = sorted(i for i in kept if not real[i] < min(min_p[r], 1.0))
        total, run, token = sum(w[i] for i in kept), 0, -1
        for i in kept:
            run += w[i]
            if w[i] > 0:
                token = i
            if run > u[r] * total:
                break
        got.append(token)
    return got
