"""Serving several sequences at once, operator by operator: what is computed, at which sizes, in plain torch and through
the framework's calls.

Four operators:

- "append": the raw q | k | v projections of every sequence's new tokens to rotated queries and to key and value rows in
  the cache (bias, an optional norm of each query and key head, rotation at the token's position, rows in bf16 or quantised
  to 8 bits with a scale each), and the rows just written read back.
- "rows": finished key and value rows into a cache, quantised, and the values that they then stand for.
- "attn": attention of a batch of sequences over a prefix that all of them share and over rows of their own.
- "sample": a token per row of logits by temperature, top-k, top-p and min-p from given random numbers.

`listed()` are fixed cases, `draw()` more of the same ranges. With `own` false, `run` computes the plain form.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda:0"
VOCAB_A, VOCAB_B = 201088, 151936  # the repository's two LM heads
TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16, "int8": torch.int8,
         "e4m3": torch.float8_e4m3fn}
LARGEST = {"int8": 127.0, "e4m3": 448.0}  # what a row's largest element becomes
EPS = 1e-6  # of the heads' norms


def listed() -> list[dict]:
    def append(name, n_seq, n, n_head, n_kv, d, norm, start, x, cache):
        return {"name": name, "kind": "append", "n_seq": n_seq, "n": n, "n_head": n_head, "n_kv": n_kv, "d": d, "norm": norm,
                "start": start, "x": x, "cache": cache}

    def attn(name, n_seq, n, n_head, n_kv, d, prefix, most, window, x, cache):
        return {"name": name, "kind": "attn", "n_seq": n_seq, "n": n, "n_head": n_head, "n_kv": n_kv, "d": d,
                "prefix": prefix, "most": most, "window": window, "x": x, "cache": cache}

    return [
        # one token of two sequences, 16-bit cache: the smallest call, latency
        append("append_b2_bf16", 2, 1, 64, 8, 64, False, 211, "float32", "bfloat16"),
        # a step of a batch of 64, heads with norms, far into their texts
        append("append_b64_norm_e4m3", 64, 1, 32, 4, 128, True, 70001, "bfloat16", "e4m3"),
        # a prompt's 4001 tokens in one piece
        append("append_prompt4001_int8", 1, 4001, 64, 8, 64, False, 0, "float32", "int8"),
        # a short text's finished rows into a quantised cache and back
        {"name": "rows_37_e4m3", "kind": "rows", "n_seq": 1, "n": 37, "n_kv": 4, "d": 128, "x": "float32", "cache": "e4m3"},
        # four long texts' rows
        {"name": "rows_4x16000_int8", "kind": "rows", "n_seq": 4, "n": 16000, "n_kv": 8, "d": 64, "x": "bfloat16",
         "cache": "int8"},
        # two sequences early behind a short prompt: the smallest call
        attn("attn_b2_prefix200", 2, 1, 64, 8, 64, 200, 17, 0, "float32", "bfloat16"),
        # sixteen answers to one long prompt, as the framework's model runs them (fp32 activations)
        attn("attn_b16_prefix6000_int8", 16, 1, 64, 8, 64, 6000, 300, 0, "float32", "int8"),
        # a sliding-window layer of a batch: few keys of the prefix are still seen
        attn("attn_b32_window128", 32, 1, 64, 8, 64, 3001, 99, 128, "float32", "int8"),
        # four users' own prompts of up to 512 tokens behind a shared one
        attn("attn_b4_prompt512_d128", 4, 512, 32, 4, 128, 2000, 530, 0, "bfloat16", "bfloat16"),
        # a large batch behind a very long shared prompt: the largest
        attn("attn_b64_prefix32768_e4m3", 64, 1, 64, 8, 64, 32768, 640, 0, "bfloat16", "e4m3"),
        # one sequence's next token
        {"name": "sample_b1", "kind": "sample", "n_seq": 1, "vocab": VOCAB_A, "top_k": 50, "top_p": 0.95, "min_p": 0.0,
         "each": False, "x": "float32"},
        # a batch of requests, each with settings of its own
        {"name": "sample_b48_each", "kind": "sample", "n_seq": 48, "vocab": VOCAB_B, "top_k": 400, "top_p": 0.9,
         "min_p": 0.02, "each": True, "x": "bfloat16"},
    ]


def _log_between(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(("append", "rows", "attn", "attn", "attn", "sample"))
    d, n_kv = rng.choice((64, 128)), rng.choice((1, 2, 4, 8))
    x, cache = rng.choice(("float32", "float16", "bfloat16")), rng.choice(("bfloat16", "int8", "e4m3"))
    if kind == "append":
        n_head = n_kv * rng.choice((1, 3, 4, 8))
        tokens = 4001 * 80 * 64 // ((n_head + 2 * n_kv) * d)
        n_seq = _log_between(rng, 1, 96)
        return {"kind": kind, "n_seq": n_seq, "n": 1 if rng.random() < 0.5 else _log_between(rng, 1, max(1, tokens // n_seq)),
                "n_head": n_head, "n_kv": n_kv, "d": d, "norm": rng.random() < 0.5, "start": _log_between(rng, 1, 120000) - 1,
                "x": x, "cache": cache}
    if kind == "rows":
        n_seq = _log_between(rng, 1, 16)
        return {"kind": kind, "n_seq": n_seq, "n": _log_between(rng, 1, 4 * 16000 * 8 * 64 // (n_seq * n_kv * d)),
                "n_kv": n_kv, "d": d, "x": x, "cache": cache}
    if kind == "attn":
        n_head = n_kv * rng.choice((1, 3, 4, 5, 8, 8, 16))
        n = rng.choice((1, 1, 1, _log_between(rng, 2, 512)))
        n_seq = _log_between(rng, 1, 64 if n == 1 else max(1, 2048 // n))
        n_seq = min(n_seq, 64)
        keys = 64 * 64 * 33408 * 64 // (n_head * d * n_seq * n)  # so that none costs more than the largest listed one
        most = n + _log_between(rng, 1, max(1, min(1500, keys - n)))
        prefix = 0 if rng.random() < 0.1 else _log_between(rng, 1, max(1, min(32768, keys - most)))
        return {"kind": kind, "n_seq": n_seq, "n": n, "n_head": n_head, "n_kv": n_kv, "d": d, "prefix": prefix, "most": most,
                "window": rng.choice((0, 0, 0, 128, _log_between(rng, 1, 5000))), "x": x, "cache": cache}
    vocab = _log_between(rng, 1000, VOCAB_A)
    return {"kind": kind, "n_seq": min(_log_between(rng, 1, 128), max(1, 48 * VOCAB_B // vocab)), "vocab": vocab,
            "top_k": rng.choice((0, 1, 20, _log_between(rng, 2, 5000))), "top_p": rng.choice((1.0, 0.95, round(rng.uniform(0.05, 1), 3))),
            "min_p": rng.choice((0.0, 0.0, 0.05, round(rng.uniform(0, 0.3), 3))), "each": rng.random() < 0.5, "x": x}


# -- inputs ------------------------------------------------------------------


def _gen(seed: int) -> torch.Generator:
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed) * 1000003 % (1 << 62))
    return g


def _quantised(x: torch.Tensor, cache: str) -> tuple[torch.Tensor, torch.Tensor | None]:
    """fp32 rows as a cache holds them: (elements, a scale per row)."""
    if cache == "bfloat16":
        return x.to(torch.bfloat16), None
    scale = x.abs().amax(-1) / LARGEST[cache]
    y = x / torch.where(scale > 0, scale, torch.ones_like(scale))[..., None]
    return (y.round().clamp(-127, 127).to(torch.int8) if cache == "int8" else y.clamp(-448, 448).to(torch.float8_e4m3fn)), scale


def _values(codes: torch.Tensor, scale: torch.Tensor | None) -> torch.Tensor:
    return codes.float() if scale is None else codes.float() * scale[..., None]


def _inputs(case: dict, seed: int) -> dict:
    g = _gen(seed)
    kind, B = case["kind"], case["n_seq"]
    normal = lambda *shape: torch.randn(*shape, generator=g, device=DEVICE)  # noqa: E731
    s = {"case": case}
    if kind == "append":
        H, G, d, n, t = case["n_head"], case["n_kv"], case["d"], case["n"], TYPES[case["x"]]
        # heads differ in size, and a few dimensions of the keys are far larger than the others
        qkv = normal(B, n, H + 2 * G, d) * (0.5 + torch.rand(H + 2 * G, 1, generator=g, device=DEVICE))
        qkv[:, :, H:H + G, 3::29] *= 8
        s["qkv"] = qkv.to(t).reshape(B, n, (H + 2 * G) * d)
        s["bq"], s["bk"], s["bv"] = (normal(h * d) * 0.1 for h in (H, G, G))
        s["wq"], s["wk"] = (1 + 0.2 * normal(d), 1 + 0.2 * normal(d)) if case["norm"] else (None, None)
        s["inv"], s["amp"] = 1.0 / 150000.0 ** (torch.arange(d // 2, dtype=torch.float32, device=DEVICE) / (d // 2)), 1.3465
        # a text's rows so far, of `start` positions that its sequences share and a few of their own
        s["len"] = torch.randint(0, 40, (B,), generator=g, device=DEVICE, dtype=torch.int32)
        s["rows"] = 40 + n
    elif kind == "rows":
        shape = (B, case["n_kv"], case["n"], case["d"])
        size = 0.3 + torch.rand(B, case["n_kv"], 1, case["d"], generator=g, device=DEVICE)
        s["k"], s["v"] = ((normal(*shape) * size).to(TYPES[case["x"]]) for _ in "kv")
    elif kind == "attn":
        H, G, d, n, P, L = case["n_head"], case["n_kv"], case["d"], case["n"], case["prefix"], case["most"]
        s["q"] = (normal(B, n, H, d) * 1.2).to(TYPES[case["x"]])
        s["sinks"] = normal(H)
        for name, shape, size in (("pk", (G, P, d), 1.5), ("pv", (G, P, d), 1.0), ("k", (B, G, L, d), 1.5), ("v", (B, G, L, d), 1.0)):
            s[name], s[name + "s"] = _quantised(normal(*shape) * size, case["cache"])
        # rows of their own before these tokens, and how many of the new tokens each sequence has
        s["len"] = torch.randint(0, L - n + 1, (B,), generator=g, device=DEVICE, dtype=torch.int32)
        s["counts"] = None
        if n > 1:
            s["counts"] = torch.randint((n + 1) // 2, n + 1, (B,), generator=g, device=DEVICE, dtype=torch.int32)
    else:
        V = case["vocab"]
        # an LM head's logits: a broad bulk and a few candidates far above it
        logits = 2.0 * normal(B, V)
        top = torch.randint(0, V, (B, 6), generator=g, device=DEVICE)
        logits.scatter_add_(1, top, 6 + 8 * torch.rand(B, 6, generator=g, device=DEVICE))
        s["logits"] = logits.to(TYPES[case["x"]])
        s["u"] = torch.rand(B, generator=g, device=DEVICE)
        if case["each"]:  # a row's settings around the case's, some rows greedy, some without a filter
            r = lambda: torch.rand(B, generator=g, device=DEVICE)  # noqa: E731
            s["temperature"] = torch.where(r() < 0.1, 0.0, 0.5 + r())
            s["top_k"] = torch.where(r() < 0.3, 0.0, (1 + 2 * r() * case["top_k"]).floor()).to(torch.int32)
            s["top_p"] = torch.where(r() < 0.2, 1.0, (case["top_p"] + 0.1 * (r() - 0.5)).clamp(0.01, 1.0))
            s["min_p"] = torch.where(r() < 0.5, 0.0, 2 * r() * case["min_p"])
        else:
            s["temperature"], s["top_k"], s["top_p"], s["min_p"] = 0.8, case["top_k"], case["top_p"], case["min_p"]
    return s


def prepare(case: dict, seed: int) -> dict:
    s = _inputs(case, seed)
    if own and case["kind"] != "sample":
        _own_caches(case, s)
    return s


def _own_caches(case: dict, s: dict) -> None:
    """The caches as a user's program holds them."""
    from nurostream_amd.model.batch import BatchKV
    from nurostream_amd.model.decode import AttnConfig

    kind, B, G, d = case["kind"], case["n_seq"], case["n_kv"], case["d"]
    cfg = AttnConfig(n_head=case.get("n_head", G), n_head_kv=G, head_dim=d, vocab_size=VOCAB_A, rope_base=150000.0,
                     context_length=131072, sliding_window=128)
    t = TYPES[case["cache"]]
    prefix = None
    if kind == "attn" and case["prefix"]:
        prefix = BatchKV(1, cfg, 1, case["prefix"], DEVICE, dtype=t)
        for stack, codes in ((prefix.k_stack, "pk"), (prefix.v_stack, "pv"), (prefix.k_scale, "pks"), (prefix.v_scale, "pvs")):
            if stack is not None:
                stack[0, 0].copy_(s[codes])
        prefix.advance(case["prefix"])
    elif kind == "append" and case["start"]:
        # (only the length of the shared rows counts here: few rows of storage would do, but a prefix holds what it says)
        prefix = BatchKV(1, cfg, 1, case["start"], DEVICE, dtype=t)
        prefix.advance(case["start"])
    rows = {"append": s.get("rows"), "rows": case.get("n"), "attn": case.get("most")}[kind]
    kv = BatchKV(1, cfg, B, rows, DEVICE, dtype=t, prefix=prefix)
    if kind == "attn":
        for stack, codes in ((kv.k_stack, "k"), (kv.v_stack, "v"), (kv.k_scale, "ks"), (kv.v_scale, "vs")):
            if stack is not None:
                stack[0].copy_(s[codes])
        for name in ("pk", "pv", "pks", "pvs", "k", "v", "ks", "vs"):
            s.pop(name)
    if kind != "rows":
        kv.pos.copy_(s["len"])
        kv.length = rows - case["n"]  # (the most that a sequence may hold before these tokens)
    s["cfg"], s["kv"] = cfg, kv


# -- one pass ----------------------------------------------------------------


def run(state: dict):
    kind = state["case"]["kind"]
    if own:
        return {"append": _append_own, "rows": _rows_own, "attn": _attn_own, "sample": _sample_own}[kind](state)
    return {"append": _append_plain, "rows": _rows_plain, "attn": _attn_plain, "sample": _sample_plain}[kind](state)


def _append_own(s: dict):
    from nurostream_amd.model.batch import append_qkv, load_rows

    kv = s["kv"]
    q = append_qkv(s["qkv"], s["bq"], s["bk"], s["bv"], s["cfg"], s["inv"], s["amp"], kv, 0, q_norm=s["wq"], k_norm=s["wk"],
                   eps=EPS)
    return (q, *load_rows(kv, 0, kv.pos, s["case"]["n"], dtype=torch.bfloat16))


def _append_plain(s: dict):
    case = s["case"]
    B, n, H, G, d = case["n_seq"], case["n"], case["n_head"], case["n_kv"], case["d"]
    x = s["qkv"].float().reshape(B, n, H + 2 * G, d)
    q, k, v = x[:, :, :H] + s["bq"].reshape(H, d), x[:, :, H:H + G] + s["bk"].reshape(G, d), x[:, :, H + G:] + s["bv"].reshape(G, d)
    if s["wq"] is not None:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + EPS) * s["wq"]
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + EPS) * s["wk"]
    at = case["start"] + s["len"].double()[:, None] + torch.arange(n, device=DEVICE)
    angle = (at[:, :, None] * s["inv"].double())[:, :, None]  # in 64 bits: far positions are many turns
    cos, sin = (torch.cos(angle) * s["amp"]).float(), (torch.sin(angle) * s["amp"]).float()
    turned = lambda y: torch.cat([y[..., :d // 2] * cos - y[..., d // 2:] * sin, y[..., d // 2:] * cos + y[..., :d // 2] * sin], -1)  # noqa: E731
    held = lambda y: _values(*_quantised(y, case["cache"])).transpose(1, 2).to(torch.bfloat16)  # noqa: E731
    return turned(q).to(s["qkv"].dtype), held(turned(k)).contiguous(), held(v).contiguous()


def _rows_own(s: dict):
    from nurostream_amd.model.batch import load_rows, store_rows

    store_rows(s["k"], s["v"], s["kv"], 0)
    return load_rows(s["kv"], 0, 0, s["case"]["n"], dtype=torch.bfloat16)


def _rows_plain(s: dict):
    return tuple(_values(*_quantised(s[name].float(), s["case"]["cache"])).to(torch.bfloat16) for name in "kv")


def _attn_own(s: dict):
    from nurostream_amd.model.batch import batch_attn

    return (batch_attn(s["q"], s["cfg"], s["kv"], 0, s["sinks"], s["case"]["window"], counts=s["counts"]),)


def _attn_plain(s: dict):
    case = s["case"]
    B, n, H, G, d = case["n_seq"], case["n"], case["n_head"], case["n_kv"], case["d"]
    P, L, window, R = case["prefix"], case["most"], case["window"], H // G
    first = max(0, P - window + 1) if window else 0  # prefix rows before it are seen by nobody
    q = s["q"].float().reshape(B, n, G, R, d).permute(2, 0, 1, 3, 4)  # (G, B, n, R, d)
    part = lambda x, f: None if x is None else x[:, f:]  # noqa: E731
    pk, pv = _values(s["pk"][:, first:], part(s["pks"], first)), _values(s["pv"][:, first:], part(s["pvs"], first))
    k, v = _values(s["k"], s["ks"]).transpose(0, 1), _values(s["v"], s["vs"]).transpose(0, 1)
    shared = torch.matmul(q.reshape(G, B * n * R, d), pk.transpose(1, 2).contiguous()).reshape(G, B, n, R, P - first)
    mine = torch.matmul(q.reshape(G, B, n * R, d), k.transpose(2, 3).contiguous()).reshape(G, B, n, R, L)
    score = torch.cat([shared, mine], -1).mul_(1.0 / math.sqrt(d))
    del shared, mine
    j, t = torch.arange(n, device=DEVICE), torch.arange(L, device=DEVICE)
    upto = s["len"][:, None] + j  # the row of its own that a token is
    seen = torch.cat([torch.ones(B, n, P - first, dtype=torch.bool, device=DEVICE), t <= upto[..., None]], -1)
    if window:
        at = torch.cat([torch.arange(first, P, device=DEVICE), P + t])
        seen &= P + upto[..., None] - at < window
    score.masked_fill_(~seen[None, :, :, None], -math.inf)
    sink = s["sinks"].reshape(G, 1, 1, R, 1)
    top = torch.maximum(score.amax(-1, keepdim=True), sink)
    w = torch.exp_(score.sub_(top))
    total = w.sum(-1, keepdim=True) + torch.exp(sink - top)
    out = torch.matmul(w[..., :P - first].reshape(G, B * n * R, P - first), pv).reshape(G, B, n, R, d)
    out = out + torch.matmul(w[..., P - first:].reshape(G, B, n * R, L), v).reshape(G, B, n, R, d)
    out = (out / total).permute(1, 2, 0, 3, 4).reshape(B, n, H, d)
    if s["counts"] is not None:  # nothing for the tokens that a sequence does not have
        out = out.masked_fill((j >= s["counts"][:, None])[..., None, None], 0.0)
    return (out.to(s["q"].dtype),)


def _sample_own(s: dict):
    from nurostream_amd.model.sampling import sample

    return (sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"]),)


def _sample_plain(s: dict):
    # in 64 bits: sums over the vocabulary are compared with borders and a random number
    B, V = s["logits"].shape
    column = lambda x: torch.as_tensor(x, device=DEVICE).expand(B)[:, None]  # noqa: E731
    T, k, top_p, min_p = (column(s[name]).double() for name in ("temperature", "top_k", "top_p", "min_p"))
    x = s["logits"].double()
    value, order = torch.sort(x, dim=-1, descending=True, stable=True)  # equal ones by their index
    w = torch.exp((value - value[:, :1]) / torch.where(T > 0, T, 1.0))
    rank = torch.arange(V, device=DEVICE)
    keep = rank < torch.where(k > 0, k, V)
    w = torch.where(keep, w, 0.0)
    mass = w.cumsum(-1)
    keep = (top_p >= 1) | (mass - w < top_p * mass[:, -1:])
    w = torch.where(keep & (w >= min_p), w, 0.0)
    mass = torch.zeros_like(w).scatter_(1, order, w).cumsum_(-1)
    token = (mass <= s["u"].double()[:, None] * mass[:, -1:]).sum(-1).clamp_(max=V - 1)
    return (torch.where(T[:, 0] > 0, token, order[:, 0]).to(torch.int32),)


# -- what a pass cannot do without -------------------------------------------


def work(case: dict) -> dict:
    size = {"float32": 4, "float16": 2, "bfloat16": 2}
    held = lambda d: 2 * d if case["cache"] == "bfloat16" else d + 4  # noqa: E731
    if case["kind"] == "append":
        tokens, H, G, d, e = case["n_seq"] * case["n"], case["n_head"], case["n_kv"], case["d"], size[case["x"]]
        return {"bytes": tokens * ((2 * H + 2 * G) * d * e + 2 * G * (held(d) + 2 * d)), "flops": 8 * tokens * (H + 2 * G) * d}
    if case["kind"] == "rows":
        rows, d = 2 * case["n_seq"] * case["n_kv"] * case["n"], case["d"]
        return {"bytes": rows * (d * size[case["x"]] + held(d) + 2 * d), "flops": 3 * rows * d}
    if case["kind"] == "sample":
        return {"bytes": case["n_seq"] * case["vocab"] * size[case["x"]], "flops": 2 * case["n_seq"] * case["vocab"]}
    # rows of their own: half of what there is room for, with the new tokens, on average
    B, n, H, G, d, P, window = (case[name] for name in ("n_seq", "n", "n_head", "n_kv", "d", "prefix", "window"))
    mine, new = (case["most"] - n) / 2 + n / 2, n if n == 1 else 3 * n / 4
    shared, seen = P, P + mine
    if window:
        shared, seen, mine = max(0, min(P, window - 1)), min(seen, window), min(mine + n, window + n)
    return {"bytes": 2 * G * held(d) * (shared + B * mine) + 2 * B * n * H * d * size[case["x"]], "flops": 4 * d * H * B * new * seen}


# -- the definition in 64 bits -----------------------------------------------


def exact(case: dict, seed: int):
    if case["kind"] == "sample":
        return None  # (whole numbers)
    s = _inputs(case, seed)
    return {"append": _append_exact, "rows": _rows_exact, "attn": _attn_exact}[case["kind"]](case, s)


def _held_exact(x: torch.Tensor, cache: str) -> torch.Tensor:
    """What a cache's rows stand for, given 64-bit rows: the nearest of the type's values, to even between two."""
    if cache == "bfloat16":
        step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=1e-300))) - 7)
        return torch.round(x / step) * step
    scale = x.abs().amax(-1, keepdim=True) / LARGEST[cache]
    y = torch.where(scale > 0, x / scale, 0.0)
    if cache == "int8":
        return torch.round(y) * scale
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)  # three bits, subnormal below 2^-6
    return torch.round(y / step) * step * scale


def _append_exact(case: dict, s: dict):
    B, n, H, G, d = case["n_seq"], case["n"], case["n_head"], case["n_kv"], case["d"]
    heads = s["qkv"].double().reshape(B, n, H + 2 * G, d) + torch.cat([s["bq"], s["bk"], s["bv"]]).double().reshape(H + 2 * G, d)
    qk, v = heads[:, :, :H + G], heads[:, :, H + G:]
    if case["norm"]:
        qk = qk / (qk.pow(2).sum(-1, keepdim=True) / d + EPS).sqrt()
        qk = torch.cat([qk[:, :, :H] * s["wq"].double(), qk[:, :, H:] * s["wk"].double()], 2)
    place = (s["len"].double()[:, None] + torch.arange(n, device=DEVICE).double()[None] + float(case["start"]))[..., None]
    turn = torch.polar(torch.full((B, n, d // 2), s["amp"], dtype=torch.float64, device=DEVICE), place * s["inv"].double())
    z = torch.complex(qk[..., :d // 2].contiguous(), qk[..., d // 2:].contiguous()) * turn[:, :, None]
    qk = torch.cat([z.real, z.imag], -1)
    k, v = (_held_exact(y.transpose(1, 2), case["cache"]).contiguous() for y in (qk[:, :, H:], v))
    return qk[:, :, :H].contiguous(), k, v


def _rows_exact(case: dict, s: dict):
    return tuple(_held_exact(s[name].double(), case["cache"]) for name in "kv")


def _attn_exact(case: dict, s: dict):
    """Sequence by sequence and kv head by kv head, each token over the keys that it sees."""
    B, n, H, G, d = case["n_seq"], case["n"], case["n_head"], case["n_kv"], case["d"]
    P, window, R = case["prefix"], case["window"], H // G
    whole = lambda codes, scale: codes.double() if scale is None else codes.double() * scale.double()[..., None]  # noqa: E731
    out = torch.zeros(B, n, H, d, dtype=torch.float64, device=DEVICE)
    lens = s["len"].tolist()
    counts = [n] * B if s["counts"] is None else s["counts"].tolist()
    for g in range(G):
        pk, pv = whole(s["pk"][g], None if s["pks"] is None else s["pks"][g]), whole(s["pv"][g], None if s["pvs"] is None else s["pvs"][g])
        for b in range(B):
            c = counts[b]
            rows = lens[b] + c
            k, v = (torch.cat([p, whole(s[x][b, g, :rows], None if s[x + "s"] is None else s[x + "s"][b, g, :rows])])
                    for p, x in ((pk, "k"), (pv, "v")))
            q = s["q"][b, :c, g * R:(g + 1) * R].double().reshape(c * R, d)
            at = torch.arange(P + rows, device=DEVICE)
            mine = (P + lens[b] + torch.arange(c, device=DEVICE)).repeat_interleave(R)[:, None]
            hidden = (at > mine) | ((mine - at >= window) if window else False)
            sc = (q @ k.T.contiguous() / math.sqrt(d)).masked_fill(hidden, -math.inf)
            sc = torch.cat([sc, s["sinks"][g * R:(g + 1) * R].double().repeat(c)[:, None]], 1)
            out[b, :c, g * R:(g + 1) * R] = (torch.softmax(sc, -1)[:, :-1] @ v).reshape(c, R, d)
    return (out,)
